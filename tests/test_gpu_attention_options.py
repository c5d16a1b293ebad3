"""GPU: the attention options of the token blocks (transformer_model.attention_options: qk_norm, rope,
softcap, distance_bias), a block and the hybrid encoder with them; and the ops of dmf_attention as a
program uses them: one after the other, on another stream, in a replayed graph, over caches whose offsets
pass 32 bits.

Tolerances of the blocks are those of tests/test_gpu_transformer.py (max |ours - ref| <= tol * max(1, max |ref|)):
1e-4 for the f32 parity mode, 3e-2 for bf16 blocks and their gradients."""
import copy

import pytest
import torch
import torch.nn.functional as F

import dmf_attention as A
import dmf_tokens as D
import model_module as MM
import parameters as PR
import transformer_model as TM

pytestmark = pytest.mark.gpu
DEV = "cuda"
ALL = dict(qk_norm=True, rope=True, softcap=8.0, distance_bias=True)


def _close(a, b, tol, what):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape, (what, a.shape, b.shape)
    err = (a - b).abs().max().item()
    assert err <= tol * max(1.0, b.abs().max().item()), f"{what}: {err:.3e} (ref max {b.abs().max():.3e})"


def _rms(x, w):
    return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w


def _rot(x, cos, sin):  # [b, n, h, d], pairs (p, p + rot / 2)
    r = cos.shape[1]
    a, b = x[..., :r], x[..., r:2 * r]
    c, s = cos[None, :, None], sin[None, :, None]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * r:]], -1)


def _block64(blk, x, o, rope):
    """TransformerBlock in 64 bits with the options `o`, from the block's own (double) parameters."""
    at, (b, n, e) = blk.attn, x.shape
    h = F.layer_norm(x, (e,), blk.norm1.weight, blk.norm1.bias, blk.norm1.eps)
    q, k, v = F.linear(h, at.qkv.weight, at.qkv.bias).view(b, n, 3, at.num_heads, at.head_dim).unbind(2)
    if o.get("qk_norm"):
        q, k = _rms(q, at.q_norm), _rms(k, at.k_norm)
    if o.get("rope"):
        q, k = (_rot(t, rope[0].double(), rope[1].double()) for t in (q, k))
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    s = (q @ k.transpose(-1, -2)) * at.head_dim ** -0.5
    if o.get("softcap"):
        s = o["softcap"] * torch.tanh(s / o["softcap"])
    if o.get("distance_bias"):
        i = torch.arange(n, device=x.device)
        s = s - at.slopes.double()[:, None, None] * (i[:, None] - i).abs()
    y = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(b, n, e)
    x = x + F.linear(y, at.proj.weight, at.proj.bias) * blk.gamma1
    h = F.layer_norm(x, (e,), blk.norm2.weight, blk.norm2.bias, blk.norm2.eps)
    h = F.linear(F.gelu(F.linear(h, blk.mlp.fc1.weight, blk.mlp.fc1.bias)), blk.mlp.fc2.weight, blk.mlp.fc2.bias)
    return x + h * blk.gamma2


def _block(options, seed, e=256, heads=4):
    torch.manual_seed(seed)
    blk = TM.TransformerBlock(e, heads, options=options).to(DEV).eval()
    with torch.no_grad():
        blk.gamma1.fill_(0.7)
        blk.gamma2.fill_(0.6)
        for t in (getattr(blk.attn, "q_norm", None), getattr(blk.attn, "k_norm", None)):
            if t is not None:
                t.copy_(1 + 0.2 * torch.randn_like(t))
        blk.attn.qkv.weight.mul_(3)   # scores away from zero
    return blk


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("options", [dict(qk_norm=True), dict(rope=True), dict(softcap=4.0), dict(distance_bias=True), ALL],
                         ids=lambda o: "-".join(o))
def test_block_with_options_vs_float64(options, dtype, tol):
    blk = _block(options, 1)
    blk.compute_dtype = dtype
    rope = A.rope_table_2d(6, 12, 64, device=DEV)
    torch.manual_seed(2)
    x = torch.randn(3, 72, 256, device=DEV, requires_grad=True)
    g = torch.randn(3, 72, 256, device=DEV)
    y = blk(x, rope)
    y.backward(g)
    ref = copy.deepcopy(blk).double()
    ref.zero_grad(set_to_none=True)
    x64 = x.detach().double().requires_grad_()
    y64 = _block64(ref, x64, options, rope)
    y64.backward(g.double())
    _close(y, y64, tol, "out")
    _close(x.grad, x64.grad, tol, "dx")
    for (name, p), (_, r) in zip(blk.named_parameters(), ref.named_parameters()):
        _close(p.grad, r.grad, tol, name)
    with torch.no_grad():  # the forward-only block
        _close(blk(x, rope), y64, tol, "out without a graph")


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2)])
def test_attention_module_with_options(dtype, tol):
    torch.manual_seed(5)
    at = TM.MultiHeadSelfAttention(256, 2, attn_drop=0.0, options=ALL).to(DEV).eval()
    at.compute_dtype = dtype
    rope = A.rope_table_2d(4, 4, 128, device=DEV)
    x = torch.randn(2, 16, 256, device=DEV, requires_grad=True)
    y = at(x, rope)
    y.sum().backward()

    class Blk:
        attn = copy.deepcopy(at).double()
    q, k, v = F.linear(x.detach().double(), Blk.attn.qkv.weight, Blk.attn.qkv.bias).view(2, 16, 3, 2, 128).unbind(2)
    q, k = (_rot(_rms(t, w), rope[0].double(), rope[1].double()).transpose(1, 2) for t, w in ((q, Blk.attn.q_norm), (k, Blk.attn.k_norm)))
    i = torch.arange(16, device=DEV)
    s = 8.0 * torch.tanh(q @ k.transpose(-1, -2) * 128 ** -0.5 / 8.0) - Blk.attn.slopes.double()[:, None, None] * (i[:, None] - i).abs()
    o = (torch.softmax(s, -1) @ v.transpose(1, 2)).transpose(1, 2).reshape(2, 16, 256)
    _close(y, F.linear(o, Blk.attn.proj.weight, Blk.attn.proj.bias), tol, "out")
    assert at.q_norm.grad.abs().max() > 0 and at.k_norm.grad.abs().max() > 0 and torch.isfinite(x.grad).all()


def test_options_refusals_and_state_dict():
    with pytest.raises(ValueError, match="unknown"):
        TM.TransformerBlock(256, 4, options=dict(alibi=True))
    with pytest.raises(ValueError, match="softcap"):
        TM.attention_options(dict(softcap=-1.0))
    assert TM.attention_options(None) is None and TM.attention_options(dict(qk_norm=False)) is None
    plain, opt = TM.TransformerBlock(256, 4), TM.TransformerBlock(256, 4, options=ALL)
    assert set(opt.state_dict()) - set(plain.state_dict()) == {"attn.q_norm", "attn.k_norm"}
    assert opt.attn.attn_drop.p == 0.0 and plain.attn.attn_drop.p == 0.1
    x = torch.randn(1, 16, 256, device=DEV)
    opt = opt.to(DEV)
    with pytest.raises(ValueError, match="rotation table"):
        opt(x)
    with pytest.raises(ValueError, match="rotation table"):
        opt(x, A.rope_table_2d(2, 2, 64, device=DEV))
    opt.attn.attn_drop.p = 0.1
    with pytest.raises(ValueError, match="attention dropout"):
        opt.train()(x, A.rope_table_2d(4, 4, 64, device=DEV))


def test_hybrid_encoder_with_options_trains():
    """The encoder built from parameters: a training step (dropout after the projections on), gradients of every
    option's parameters, and the options' effect on the output."""
    P = copy.deepcopy(PR.small_parameters(dropout=0.0))
    for m in ("dwi", "dce"):
        mp = P[f"{m}_model_parameters"] = copy.deepcopy(P[f"{m}_model_parameters"])
        mp.update(use_hybrid_transformer=True, use_backbone=False, transformer_embed_dim=256, transformer_heads=4,
                  transformer_depth=2, enable_modality_attention=False)
        mp["transformer_attention"] = dict(ALL)
    torch.manual_seed(0)
    enc = MM.initialize_model(MM.ModelMaskHeadBackbone("dwi", P), True).to(DEV).train()
    x = torch.randn(2, P["dwi_channel_num"], 64, 64, device=DEV)
    logits = enc(x)[0]
    logits.float().square().sum().backward()
    for name, p in enc.transformer.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        if "q_norm" in name or "k_norm" in name:
            assert p.grad.abs().max() > 0, name
    enc.eval()
    with torch.no_grad():
        a = enc(x)[0].float()
        for blk in enc.transformer.transformer.layers:
            blk.attn.options["softcap"] = 0.5
        b = enc(x)[0].float()
    assert torch.isfinite(a).all() and (a - b).abs().max() > 0


def _step(q, k, v, w, cos, sin, docs, go):
    qn, kn = A.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)
    o = A.attention(qn, kn, v, softcap=20.0, causal=True, documents=docs)
    return (o.detach(), *torch.autograd.grad(o, (q, k, v, w), go))


def _inputs(b=2, n=200, hq=4, hk=2, d=64, dt=torch.bfloat16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda h: torch.randn(b, n, h, d, generator=g, device=DEV).to(dt).requires_grad_()  # noqa: E731
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).requires_grad_()
    docs = (torch.arange(n, device=DEV) // 70).int().expand(b, n).contiguous()
    docs[:, -9:] = -1
    return mk(hq), mk(hk), mk(hk), w, *A.rope_table(n, d, device=DEV), docs, mk(hq).detach()


def test_norm_rotation_and_attention_together_vs_float64():
    """The two ops as a block runs them, gradients through both, against the same formulas in 64 bits (f32 operands:
    the blocks' parity tolerance)."""
    q, k, v, w, cos, sin, docs, go = _inputs(dt=torch.float32)
    got = _step(q, k, v, w, cos, sin, docs, go)
    Q, K, V, W = (t.detach().double().requires_grad_() for t in (q, k, v, w))
    qn, kn = (_rot(_rms(t, W), cos.double(), sin.double()) for t in (Q, K))
    kr, vr = (t.repeat_interleave(2, 2) for t in (kn, V))
    z = 20.0 * torch.tanh(torch.einsum("bihd,bjhd->bhij", qn, kr) / 8 / 20.0)
    i = torch.arange(200, device=DEV)
    see = (docs[:, :, None] == docs[:, None]) & (docs >= 0)[:, :, None] & (i[:, None] >= i)
    p = torch.softmax(z.masked_fill(~see[:, None], -1e300), -1) * see[:, None]
    o = torch.einsum("bhij,bjhd->bihd", p, vr)
    ref = (o, *torch.autograd.grad(o, (Q, K, V, W), go.double()))
    for a, r, name in zip(got, ref, ("o", "dq", "dk", "dv", "dw")):
        _close(a, r, 1e-4, name)


def test_on_another_stream_and_after_it():
    args = _inputs()
    want = _step(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _step(*args)
    torch.cuda.current_stream().wait_stream(s)
    again = _step(*args)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_replayed_graphs_match_eager():
    """Two captured steps (forward, backward, split decode) sharing nothing, replayed in turn with new inputs and eager work
    between the replays."""
    torch.manual_seed(0)
    a, b = _inputs(seed=1), _inputs(seed=2)
    kc, vc = (torch.randn(2, 3000, 2, 64, device=DEV).bfloat16() for _ in range(2))
    q1, lens = torch.randn(2, 1, 4, 64, device=DEV).bfloat16(), torch.tensor([2900, 17], dtype=torch.int32, device=DEV)

    def run(args):
        with torch.no_grad():
            one = A.attention(q1, kc, vc, kv_lens=lens, causal=True)
        return (*_step(*args), one)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        for args in (a, b):
            for _ in range(2):
                run(args)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = run(args)
            graphs.append((g, out, args))
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        for g, out, args in graphs:
            with torch.no_grad():
                for t in args[:3]:
                    t.copy_(torch.randn_like(t))
                lens.copy_(torch.tensor([100 + 700 * i, 3000 - 11 * i], dtype=torch.int32))
            want = [t.clone() for t in run(args)]
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, want):
                assert torch.equal(x, y)


def test_offsets_past_32_bits():
    """A cache whose batch rows start more than 2^32 elements apart, and one whose tokens lie 2 MiB apart."""
    big = torch.empty(2 * (2 ** 32 + 4096) + 2 ** 22, dtype=torch.bfloat16, device=DEV)  # 17 GB, mostly untouched
    for shape, stride in (((2, 100, 2, 64), (2 ** 32 + 4096, 128, 64, 1)), ((1, 3000, 2, 64), (0, 2 ** 20, 64, 1))):
        k, v = torch.as_strided(big, shape, stride), torch.as_strided(big, shape, stride, 2 ** 19)
        for t, s in ((k, 1), (v, 2)):
            t.copy_(torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(s), device=DEV))
        for lq in (1, 70):
            q = torch.randn(shape[0], lq, 4, 64, device=DEV).bfloat16().requires_grad_()
            kk, vv = k.detach().requires_grad_(), v.detach().requires_grad_()
            o = A.attention(q, kk, vv, causal=True)
            go = torch.randn_like(o)
            got = (o, *torch.autograd.grad(o, (q, kk, vv), go))
            k2, v2 = (t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (k, v))
            o2 = A.attention(q, k2, v2, causal=True)
            for a, b in zip(got, (o2, *torch.autograd.grad(o2, (q, k2, v2), go))):
                assert torch.equal(a, b)
    del big


def test_cache_rows_behind_the_length_and_inputs_are_left_alone():
    k, v = (torch.randn(2, 500, 2, 64, device=DEV).bfloat16() for _ in range(2))
    k[0, 40:] = float("nan")
    v[0, 40:] = float("inf")
    q = torch.randn(2, 3, 4, 64, device=DEV).bfloat16()
    before = [t.clone() for t in (q, k, v)]
    lens = torch.tensor([40, 500], dtype=torch.int32, device=DEV)
    o = A.attention(q, k, v, kv_lens=lens, causal=True)
    short = A.attention(q[:1], k[:1, :40], v[:1, :40], causal=True)
    assert torch.isfinite(o).all()
    _close(o[:1], short, 2.0 ** -7, "a row of a padded cache")   # two roundings of outputs below 2 (split or not)
    for a, b in zip((q, k, v), before):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_int64_lengths_bool_refused_and_wide_types():
    q, k, v, *_ = _inputs()
    o1 = A.attention(q, k, v, kv_lens=torch.tensor([200, 31], device=DEV), causal=True)
    o2 = A.attention(q, k, v, kv_lens=torch.tensor([200, 31], dtype=torch.int32, device=DEV), causal=True)
    assert torch.equal(o1, o2)
    with pytest.raises(ValueError, match="documents"):
        A.attention(q, k, v, documents=torch.ones(2, 200, dtype=torch.bool, device=DEV))


def test_options_refuse_cast_weights_tables_and_changes_before_the_backward():
    """What the kernels take as float32 arrays is refused in another type or shape; norm weights changed between the
    forward and the backward raise, as torch's own ops do."""
    rope = A.rope_table_2d(4, 4, 64, device=DEV)
    x = torch.randn(1, 16, 256, device=DEV, requires_grad=True)
    for change, match in ((lambda b: setattr(b.attn, "q_norm", torch.nn.Parameter(b.attn.q_norm.bfloat16())), "q_norm"),
                          (lambda b: setattr(b.attn, "slopes", b.attn.slopes[:2].clone()), "slopes"),
                          (lambda b: setattr(b.attn, "slopes", b.attn.slopes.double()), "slopes"),
                          (lambda b: setattr(b.attn, "k_norm", torch.nn.Parameter(torch.ones(32, device=DEV))), "k_norm")):
        blk = _block(ALL, 3)
        change(blk)
        with pytest.raises(ValueError, match=match):
            blk(x, rope)
    blk = _block(ALL, 3)
    with pytest.raises(ValueError, match="table"):
        blk(x, (rope[0].bfloat16(), rope[1].bfloat16()))
    with pytest.raises(ValueError, match="belong together"):
        blk(x, (rope[0], rope[1][:, :8].contiguous()))
    for m in (blk, blk.attn):
        y = m(x, rope)
        with torch.no_grad():
            blk.attn.q_norm.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
