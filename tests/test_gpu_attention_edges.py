"""GPU: calls of qk_norm_rope and attention (dmf_attention) at the edges of what they take, against the 64-bit
references and elementwise bounds of tests/test_gpu_token_attention.py."""
import pytest
import torch

import dmf_attention as A
import test_gpu_token_attention as T

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = T.TYPES


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,n,hq,hk,d", [(1, 1, 1, 1, 64), (1, 5, 3, 1, 128), (2, 37, 5, 3, 72), (3, 1187, 12, 5, 80), (1, 3, 2, 1, 512)])
def test_qk_norm_rope_without_an_eps(b, n, hq, hk, d, dt):
    """eps 0 with heads and tokens that leave places of the launch empty: finite inputs give finite weight gradients."""
    q, k = (T._randn((b, n, h, d), dt, s, 1.5).requires_grad_() for h, s in ((hq, 1), (hk, 2)))
    wq, wk = [(1 + 0.2 * T._randn((d,), torch.float32, s)).requires_grad_() for s in (3, 4)]
    cos, sin = A.rope_table(n, d // 4 * 2, device=DEV)
    pos = torch.arange(n, device=DEV).expand(b, n)
    gq, gk = T._randn(q.shape, dt, 5), T._randn(k.shape, dt, 6)
    y = A.qk_norm_rope(q, k, cos, sin, None, wq, wk, eps=0.0)
    grads = torch.autograd.grad(y, (q, k, wq, wk), (gq, gk))
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        y0, by, dx, bx, dw, bw = T._qk_ref(x.detach(), w.detach(), cos, sin, pos, 0.0, False, g, dt)
        T._within(y[i].detach(), y0, by, f"y{i}")
        T._within(grads[i], dx, bx, f"dx{i}")
        T._within(grads[2 + i], dw, bw, f"dw{i}")


def test_query_heads_past_32_bits():
    """Head-major queries whose heads lie 256 MiB apart (a group of them past 2^31 bytes), forward and backward."""
    far = 2 ** 27 + 64
    q = torch.as_strided(torch.empty(8 * far + 4096, dtype=torch.bfloat16, device=DEV), (1, 40, 8, 64), (0, 64, far, 1))
    q.copy_(T._randn((1, 40, 8, 64), torch.bfloat16, 1))
    k, v, go = (T._randn((1, 70, 1, 64), torch.bfloat16, 2), T._randn((1, 70, 1, 64), torch.bfloat16, 3),
                T._randn((1, 40, 8, 64), torch.bfloat16, 4))
    runs = []
    for x in (q, q.contiguous()):
        ins = [t.detach().requires_grad_() for t in (x, k, v)]
        assert ins[0].stride(2) == x.stride(2)
        o = A.attention(*ins, causal=True)
        runs.append((o.detach(), *torch.autograd.grad(o, ins, go)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_rows_up_to_the_grid():
    """More rows than 65535 blocks of 96 and keys that three-wave workgroups would take (one and a half tiles of 64): rows
    at both ends and across the blocks' edges."""
    n, lk, d = 200001 * 32, 257, 8
    q, k, v = (T._randn((1, m, 1, d), torch.bfloat16, s) for m, s in ((n, 1), (lk, 2), (lk, 3)))
    o = A.attention(q, k, v)
    for at in (0, 96 * 65535 - 500, n - 1000):
        see = torch.ones(1, 1000, lk, dtype=torch.bool)
        ref, bound = T._attn_ref(q[:, at:at + 1000], k, v, see, torch.zeros(1, 1000, dtype=torch.long), d ** -0.5, 0.0, None, None)
        T._within(o[:, at:at + 1000], ref, bound, f"o from {at}")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("cap,at", [(300.0, 0.9), (1000.0, 0.9), (1000.0, 0.45), (1e4, 0.9), (1e4, 0.45), (2e5, 0.01), (1e9, 1e-6)])
def test_attention_large_caps(cap, at, slopes, dt):
    """Scores that are a large share of a large cap, a few units apart: the bend of the cap shows in the probabilities."""
    n, d, scale = 48, 8, 0.01
    two = 2.0 if dt == torch.float16 else 1.0       # (f16 keeps the keys below 65504)
    far = torch.tensor(cap * at / scale / two).bfloat16().item()
    if dt == torch.float16 and far > 6e4:
        two, far = two * 256, far / 256
    q, k = torch.zeros(1, n, 2, d), torch.zeros(1, n, 1, d)
    q[..., 0], q[..., 1] = two, two * torch.linspace(0.5, 1.5, 2 * n).view(1, n, 2)
    k[..., 0], k[0, :, 0, 1] = far, torch.arange(n) % 16 * 100.0 / two
    q, k, v, go = q.to(DEV).to(dt), k.to(DEV).to(dt), T._randn((1, n, 1, d), dt, 3), T._randn((1, n, 2, d), dt, 4)
    sl = torch.tensor([0.02, 0.01], device=DEV) if slopes else None
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.attention(*ins, scale=scale, softcap=cap, slopes=sl)
    see, pos = T._see(1, n, n, False, None, None, None)
    ref = T._attn_ref(q, k, v, see, pos, scale, cap, sl, go)
    T._within(o.detach(), ref[0], ref[1], "o")
    for g, r, bound, what in zip(torch.autograd.grad(o, ins, go), ref[2::2], ref[3::2], ("dq", "dk", "dv")):
        T._within(g, r, bound, what)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cap", [1e-4, 1e-6, 1e-8])
def test_attention_tiny_caps(cap, dt):
    """Caps whose powers leave the range of f32, over scores from zero (a query of zeros) to far past the cap."""
    b, n, h, d = 1, 70, 2, 32
    q, k, v, go = (T._randn((b, n, h, d), dt, s) for s in (1, 2, 3, 4))
    q[:, :40] = 0.0
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.attention(*ins, softcap=cap, causal=True)
    see, pos = T._see(b, n, n, True, None, None, None)
    ref = T._attn_ref(q, k, v, see, pos, d ** -0.5, cap, None, go)
    T._within(o.detach(), ref[0], ref[1], "o")
    for g, r, bound, what in zip(torch.autograd.grad(o, ins, go), ref[2::2], ref[3::2], ("dq", "dk", "dv")):
        T._within(g, r, bound, what)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq", [1, 40, 700])
def test_attention_infinite_products_under_a_cap(lq, dt):
    """A product of -inf is a score of -cap: such keys keep their weight, alone in a tile or before finite ones."""
    n, d, cap = 700, 64, 2.0
    q, k, v = torch.zeros(1, lq, 2, d), torch.zeros(1, n, 1, d), torch.zeros(1, n, 1, d)
    q[..., :2] = 1.0
    k[0, :500, 0, 0], k[0, 500:, 0, 1] = -float("inf"), -2.0
    k[0, 600:620, 0, 0] = float("inf")
    v[0, :500], v[0, 620:] = 1.0, -0.5
    q, k, v = (t.to(DEV).to(dt) for t in (q, k, v))
    for m, causal in ((n, False), (400, False), (n, True)):
        if causal and lq > m:
            continue
        o = A.attention(q, k[:, :m], v[:, :m], scale=1.0, softcap=cap, causal=causal)
        see, pos = T._see(1, lq, m, causal, None, None, None)
        big = torch.where(k.double().isinf(), k.double().sign() * 1e6, k.double())  # (far past the cap: the same scores)
        # the products are exact, so a score errs by the cap's 10 e cap and the exponent's 8 e |s|
        s = cap * torch.tanh(big[0, :m, 0, :2].sum(-1) / cap)
        p = torch.softmax(s[None].expand(lq, m).masked_fill(~see[0].to(DEV), float("-inf")), -1)
        want, mag = p @ v[0, :m, 0].double(), p @ v[0, :m, 0].double().abs()
        u = T._u(dt)
        bound = (2 * (10 * T.E * cap + 8 * T.E * cap) + u + (m + 8) * T.E) * mag + u * want.abs() + T._tiny(dt) * (m + 1)
        for h in range(2):
            T._within(o[0, :, h], want, bound, f"o of head {h}")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("cap", [1e7, 1e9, 1e15])
def test_attention_caps_that_bend_nothing(cap, slopes, dt):
    """Scores of about 1000 under caps so far above that tanh is the identity to 1e-8: the bounds of no cap at all."""
    n, d, scale = 150, 8, 0.01
    q, k = torch.zeros(1, n, 2, d), torch.zeros(1, n, 1, d)
    q[..., 0], q[..., 1] = 2.0, torch.linspace(1.0, 3.0, 2 * n).view(1, n, 2)
    k[..., 0], k[0, :, 0, 1] = 49920.0, torch.arange(n) % 16 * 50.0
    q, k, v = q.to(DEV).to(dt), k.to(DEV).to(dt), T._randn((1, n, 1, d), dt, 3)
    go = T._randn((1, n, 2, d), dt, 4)
    sl = torch.tensor([0.02, 0.01], device=DEV) if slopes else None
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.attention(*ins, scale=scale, softcap=cap, slopes=sl, causal=True)
    see, pos = T._see(1, n, n, True, None, None, None)
    ref = T._attn_ref(q, k, v, see, pos, scale, 0.0, sl, go)
    T._within(o.detach(), ref[0], ref[1], "o")
    for g, r, bound, what in zip(torch.autograd.grad(o, ins, go), ref[2::2], ref[3::2], ("dq", "dk", "dv")):
        T._within(g, r, bound, what)


def _grads(q, k, v, go, **kw):
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.attention(*ins, **kw)
    return (o.detach(), *torch.autograd.grad(o, ins, go))


@pytest.mark.parametrize("mode", [dict(), dict(causal=True), dict(cap=20.0), dict(slopes=True, causal=True)], ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("shape", [(1, 130, 130, 4, 2, 64), (1, 257, 257, 3, 1, 128), (9, 200, 200, 32, 16, 32)])
def test_attention_f16_large_score_gradients(shape, mode):
    """Output gradients whose dS pass 65504 while dq, dk and dv do not, beside rows with small ones."""
    b, lq, lk, hq, hk, d = shape
    dt, mode = torch.float16, dict(mode)
    q, k, v = (T._randn((b, n, h, d), dt, s, 0.5) for n, h, s in ((lq, hq, 1), (lk, hk, 2), (lk, hk, 3)))
    v *= 16
    go = T._randn((b, lq, hq, d), dt, 4)
    go[:, ::3] *= 3000
    go[:, 1::3] *= 1e-3
    cap, causal = mode.get("cap", 0.0), mode.get("causal", False)
    sl = torch.tensor([2.0 ** (-4.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if mode.get("slopes") else None
    see, pos = T._see(b, lq, lk, causal, None, None, None)
    scale = 1 / 64
    got = _grads(q, k, v, go, softcap=cap, slopes=sl, causal=causal, scale=scale)
    ref = T._attn_ref(q, k, v, see, pos, scale, cap, sl, go)
    for i, name in enumerate(("o", "dq", "dk", "dv")):
        assert ref[2 * i].abs().max() < 65504, name
        T._within(got[i], ref[2 * i], ref[2 * i + 1], name)


def _ms(f):
    f()
    times = []
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("where", ["key 0", "gradient", "all"])
def test_attention_non_finite_inputs_cost_a_second_walk(where, causal, dt):
    """What is not finite and seen (a key that all see, an output gradient that overflowed, everything) makes a call at most
    a few times as long: a second walk over the tiles, and the pairs of its masked tiles one by one."""
    n, h, d = 2048, 8, 64
    q, k, v, go = (T._randn((1, n, h, d), dt, s) for s in (1, 2, 3, 4))

    def step():
        return _grads(q, k, v, go, causal=causal)

    clean = _ms(step)
    if where == "key 0":
        k[:, 0, :, 3], v[:, 0, :, 5] = float("nan"), float("inf")
    elif where == "gradient":
        go[:, n // 2, :, 7] = float("inf")
    else:
        for t in (q, k, v, go):
            t.fill_(float("nan"))
    bad = _ms(step)
    o, dq, dk, dv = step()
    if where == "gradient":
        assert torch.isfinite(o).all() and torch.isnan(dq[:, n // 2]).all() and torch.isinf(dv[:, 0, :, 7]).all()
        assert torch.isfinite(dq[:, n // 2 + 1:]).all() and torch.isfinite(dq[:, :n // 2]).all()
        if causal:
            assert torch.isfinite(dk[:, n // 2 + 1:]).all() and torch.isfinite(dv[:, n // 2 + 1:]).all()
    else:
        assert torch.isnan(o).all() and torch.isnan(dq).all()
    assert bad < 8 * clean, (bad, clean)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,mode", [(4, 1, 128, dict(cap=20.0)), (2, 2, 64, dict(slopes=True)), (3, 1, 80, dict())])
def test_attention_long_rows_hide_garbage(hq, hk, d, mode, causal, dt):
    """Packed documents beside padding that holds infinities and NaN in every operand, and a document whose last key nobody but
    its own query sees: tiles that rows see in part, rows split over workgroups."""
    n = 1300
    docs = torch.full((1, n), -1, dtype=torch.int32)
    for i, (a, b) in enumerate(((0, 7), (30, 500), (511, 640), (641, 1200))):
        docs[0, a:b] = i
    q, k, v, go = (T._randn((1, n, h, d), dt, s) for h, s in ((hq, 1), (hk, 2), (hk, 3), (hq, 4)))
    see, at = T._see(1, n, n, causal, None, None, docs)
    sl = torch.tensor([2.0 ** (-4.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if mode.get("slopes") else None
    cap = mode.get("cap", 0.0)
    ref = T._attn_ref(q, k, v, see, at, d ** -0.5, cap, sl, go)
    pad = (docs[0] < 0).to(DEV)
    for j, t in enumerate((q, k, v, go)):
        t[:, pad] = float("nan") if j % 2 else float("inf")
        t[:, pad, :, ::3] = -float("inf")
    if causal:
        v[0, 499, :, 1] = float("inf")      # the key of its document's last query
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.attention(*ins, causal=causal, documents=docs.to(DEV), softcap=cap, slopes=sl)
    grads = torch.autograd.grad(o, ins, go)
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    if causal:
        keep[499] = False                   # its output is infinite, its gradients not a number
        assert torch.isinf(o[0, 499, :, 1]).all()
    T._within(o.detach()[:, keep], ref[0][:, keep], ref[1][:, keep], "o")
    T._within(grads[0][:, keep], ref[2][:, keep], ref[3][:, keep], "dq")
    keep[30:500] &= not causal              # (its gradients reach its document's keys)
    T._within(grads[1][:, keep], ref[4][:, keep], ref[5][:, keep], "dk")
    keep[30:499] = True
    T._within(grads[2][:, keep], ref[6][:, keep], ref[7][:, keep], "dv")


@pytest.mark.parametrize("tail", [-14.9, -16.2, -17.5])
@pytest.mark.parametrize("mode", [dict(), dict(cap=1000.0), dict(slopes=True)], ids=lambda m: "-".join(m) or "plain")
def test_attention_f16_dominant_key_over_a_flat_tail(mode, tail):
    """One key far above thousands of equal ones, whose probabilities together are a thousandth: in f16 each of them errs by a
    half step of its own value down to 2^-32 of the largest (2^-40 in dV), not by 2^-25 (T._tiny, set accordingly)."""
    import dmf_native as N

    b, n, h, d, dt = 8, 4096, 4, 64, torch.float16
    assert N.load().dmf_mattn_fwd_ws_floats(N.dtype_code(dt), b, n, n, h, h, d, 0) == 0   # (no split of the keys)
    q, k, v = torch.zeros(b, n, h, d), torch.zeros(b, n, h, d), torch.ones(b, n, h, d)
    q[..., 0] = 1.0
    k[:, 1:, :, 0] = tail
    v[:, 0] = 0.0
    q, k, v = (t.to(DEV).to(dt) for t in (q, k, v))
    go = (1 + 0.5 * T._randn((b, n, h, d), torch.float32, 4)).mul(8).to(dt)
    sl = torch.full((h,), 1e-9, device=DEV) if mode.get("slopes") else None
    kw = dict(scale=1.0, softcap=mode.get("cap", 0.0), slopes=sl)
    o, _, _, dv = _grads(q, k, v, go, **kw)
    with torch.no_grad():
        o2 = A.attention(q, k, v, **kw)
    see, at = torch.ones(1, n, n, dtype=torch.bool), torch.arange(n)[None]
    tiny = T._tiny
    one = [t[:1, :, :1] for t in (q, k, v, go)]
    try:
        T._tiny = lambda dt: 2.0 ** -32
        ref = T._attn_ref(*one[:3], see, at, 1.0, kw["softcap"], None if sl is None else sl[:1], one[3])
        T._within(o[:1, :, :1], ref[0], ref[1] + 2.0 ** -25, "o")         # (2^-25: o's own rounding)
        T._within(o2[:1, :, :1], ref[0], ref[1] + 2.0 ** -25, "o without a gradient")
        T._tiny = lambda dt: 2.0 ** -40
        ref = T._attn_ref(*one[:3], see, at, 1.0, kw["softcap"], None if sl is None else sl[:1], one[3])
        T._within(dv[:1, :, :1], ref[6], ref[7] + 2.0 ** -25, "dv")
    finally:
        T._tiny = tiny


def test_forward_mode_derivatives_are_refused():
    """A tangent would be dropped without a word: dual inputs raise, plain ones inside a dual level do not."""
    from torch.autograd import forward_ad

    q, k = (T._randn((1, 6, 2, 32), torch.float32, s) for s in (1, 2))
    w = torch.ones(32, device=DEV)
    cos, sin = A.rope_table(6, 32, device=DEV)
    with forward_ad.dual_level():
        want = A.attention(q, k, k), *A.qk_norm_rope(q, k, cos, sin, None, w, w)
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (q, w, cos)]
        for args, kw in (((dual[0], k, k), {}), ((q, dual[0], k), {}), ((q, k, dual[0]), {}),
                         ((q, k, k), dict(slopes=forward_ad.make_dual(w[:2].clone(), w[:2].clone())))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.attention(*args, **kw)
        for args in ((dual[0], k, cos, sin, None, w, w), (q, dual[0], cos, sin, None, w, w), (q, k, cos, sin, None, dual[1], w),
                     (q, k, cos, sin, None, w, dual[1]), (q, k, dual[2], sin, None, w, w)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.qk_norm_rope(*args)
    assert torch.equal(want[0], A.attention(q, k, k))


def test_block_options_changed_before_the_backward_raise():
    """Slopes and rotation tables changed in place between the forward and the backward raise, as norm weights do; a table that a
    run under inference_mode made serves a training step."""
    import test_gpu_attention_options as TO
    import transformer_model as TM

    x = torch.randn(1, 16, 256, device=DEV, requires_grad=True)
    for what in ("slopes", "cos", "sin"):
        blk = TO._block(TO.ALL, 3)
        rope = A.rope_table_2d(4, 4, 64, device=DEV)
        for m in (blk, blk.attn):
            y = m(x, rope)
            with torch.no_grad():
                {"slopes": blk.attn.slopes, "cos": rope[0], "sin": rope[1]}[what].mul_(2.0)
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                y.sum().backward()
            m(x, rope).sum().backward()   # (and the changed values serve the next step)
    st = TM.TransformerStage(8, 256, depth=1, heads=4, attention=TO.ALL).to(DEV)
    im = torch.randn(2, 8, 16, 16, device=DEV)
    with torch.inference_mode():
        st.eval()(im)
    st.train()(im).float().square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in st.parameters())


@pytest.mark.parametrize("dt", TYPES)
def test_attention_scales_and_caps_at_the_ends_of_their_range(dt):
    """The smallest and largest scale and softcap that are taken, with slopes: finite outputs and gradients by the definition."""
    b, n, h, d = 1, 70, 2, 32
    q, k, v, go = (T._randn((b, n, h, d), dt, s) for s in (1, 2, 3, 4))
    sl = torch.tensor([0.1, 0.02], device=DEV)
    see, pos = T._see(b, n, n, True, None, None, None)
    for scale, cap in ((2.0 ** -60, 0.0), (2.0 ** -60, 2.0 ** -60), (2.0 ** -60, 2.0 ** 60), (1.0, 2.0 ** -60), (2.0 ** 60, 2.0 ** -60),
                       (2.0 ** 20, 5.0)):
        got = _grads(q, k, v, go, scale=scale, softcap=cap, slopes=sl, causal=True)
        ref = T._attn_ref(q, k, v, see, pos, scale, cap if cap < 1e9 else 0.0, sl, go)
        T._within(got[0], ref[0], ref[1], f"o at {scale}, {cap}")
        assert torch.isfinite(got[0]).all(), (scale, cap)
        # (1 - tanh^2 errs by up to 16 e absolute, and dq and dk carry that times the scale: past 65504 an f16 one may be infinite)
        assert all(torch.isfinite(t).all() for t in got[1:]) or (dt == torch.float16 and 16 * T.E * scale > 65504), (scale, cap)
        assert torch.isfinite(got[3]).all(), (scale, cap)
    for kw in (dict(softcap=1e-25), dict(softcap=1e30), dict(scale=1e-30), dict(scale=1e30)):
        with pytest.raises(ValueError, match="attention"):
            A.attention(q, k, v, **kw)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq,lk,d", [(2, 70, 128), (3, 3000, 64), (9, 3000, 128), (32, 200, 96), (100, 3000, 32), (257, 257, 64)])
def test_attention_every_launch_form_hides_the_future(lq, lk, d, dt):
    """Few and many queries, split keys and three row waves: what the last key holds reaches the last query alone."""
    hq, hk = 4, 2
    q, k, v, go = (T._randn((2, n, h, d), dt, s) for n, h, s in ((lq, hq, 1), (lk, hk, 2), (lk, hk, 3), (lq, hq, 4)))
    see, at = T._see(2, lq, lk, True, None, None, None)
    ref = T._attn_ref(q, k, v, see, at, d ** -0.5, 0.0, None, go)
    k[:, -1, :, 2], v[:, -1, :, 1] = float("nan"), -float("inf")
    with torch.no_grad():
        o2 = A.attention(q, k, v, causal=True)
    o, dq, _, _ = _grads(q, k, v, go, causal=True)
    for got in (o, o2):
        T._within(got[:, :-1], ref[0][:, :-1], ref[1][:, :-1], "o")
        assert torch.isnan(got[:, -1]).all()
    T._within(dq[:, :-1], ref[2][:, :-1], ref[3][:, :-1], "dq")


@pytest.mark.parametrize("dt", TYPES)
def test_attention_keys_behind_the_length_have_no_gradient(dt):
    """An output gradient that is not a number reaches the keys in use and none behind them, under key lengths alone."""
    b, n, lk, h, d = 3, 90, 140, 2, 64
    q, k, v, go = (T._randn((b, m, h, d), dt, s) for m, s in ((n, 1), (lk, 2), (lk, 3), (n, 4)))
    lens = [100, 140, 0]
    go[:, 7] = float("nan")
    _, dq, dk, dv = _grads(q, k, v, go, kv_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    for i, m in enumerate(lens):
        assert torch.isnan(dk[i, :m]).all() and torch.isnan(dv[i, :m]).all()
        assert not dk[i, m:].any() and not dv[i, m:].any()
    assert torch.isfinite(dq[:, 8:]).all() and torch.isnan(dq[:2, 7]).all() and not dq[2].any()


def test_stream_ptr_takes_what_torch_takes():
    """An index, a torch.device, a device's name or nothing name the same current stream, a side stream too."""
    import dmf_native as N

    for s in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            for d in (None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)):
                assert N.stream_ptr(d) == s.cuda_stream, d
    for d in ("cpu", torch.device("cpu")):
        with pytest.raises(ValueError):
            N.stream_ptr(d)
