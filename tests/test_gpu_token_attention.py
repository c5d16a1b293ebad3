"""GPU: qk_norm_rope and attention (dmf_attention; csrc/qknorm.hip, csrc/masked_attn*.h) against their
definitions in 64 bits, forward and backward.

Tolerances are elementwise bounds, derived from the arithmetic (u: half a step of the storage type relative to the
value, finfo.eps / 2; e = 2^-24: half a step of f32) and computed from the 64-bit reference:

* below f16's smallest normal number, 2^-14, a half step is 2^-25 whatever the value (_tiny): every rounding to f16 adds
  that much to its relative bound, for p and ds times what they multiply. The f32 exponent and the matrix instructions drop
  what is below 2^-126, the smallest normal number of f32 and bf16: the same term with that value.
* qk_norm_rope rounds once. y = rot(x r w): three products and one rotation sum in f32 (<= 8 e of
  |a cos| + |b sin|), r from a sum of d squares (its relative error <= (d + 4) e / 2 + 4 e), then u |y|.
* attention. A score errs by D = (d + 4) e scale sum|q k| (an f32 sum of d products, scaled) plus, capped, 10 e cap for the
  tanh of a 16-bit type (its polynomial's minimax error is 5.9e-7 < 10 e; 1 - 2 / (exp + 1) is closer) and plus 8 e |s| for its additions and the scaled exponent; p then
  errs by a factor of 1 +- 2 max D (its own score's and the normaliser's) and 16-bit types round it by u for the
  products. So |o - ref| <= (2 max D + u + (n + 8) e) sum_j p|v| + u|o|, n the number of keys summed; the same for dv
  with do in place of v. ds = p (dp - delta) bend: dp and delta err by E = (d + 4) e sum|do||v| (max over the keys),
  delta also by what o carries: (2 max D + u) sum_d |do_d| sum_j p|v_d|; with the rounding of ds
  |dq - ref| <= scale sum_j [(u + 4 max D)|ds| + p (E + delta's)] |k| + (n + 8) e (..) + u|dq|, and dk alike.
"""
import math

import pytest
import torch

import dmf_attention as A
import dmf_native as N

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _u(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126


def _randn(shape, dt, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)


# ------------------------------------------------------------- qk_norm_rope
def _rot_ref(x, cos, sin, inter, back=False):
    """(rotated, sum of the magnitudes each element is added up from), cos / sin broadcast over heads."""
    r = 2 * cos.shape[-1]
    y, mag = x.clone(), x.abs()
    ia = torch.arange(0, r, 2, device=x.device) if inter else torch.arange(r // 2, device=x.device)
    ib = ia + 1 if inter else ia + r // 2
    a, b = x[..., ia], x[..., ib]
    s = -sin if back else sin
    y[..., ia], y[..., ib] = a * cos - b * s, b * cos + a * s
    mag[..., ia], mag[..., ib] = (a * cos).abs() + (b * s).abs(), (b * cos).abs() + (a * s).abs()
    return y, mag


def _qk_ref(x, w, cos, sin, pos, eps, inter, gy, dt):
    """y, dx, dw in 64 bits with their bounds."""
    x = x.double()
    d = x.shape[-1]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if w is not None else torch.ones_like(x[..., :1])
    er = ((d + 4) / 2 + 4) * E if w is not None else 0.0
    ww = w.double() if w is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    n = x * r * ww
    if cos is not None:
        c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
        y, mag = _rot_ref(n, c, s, inter)
    else:
        y, mag = n, n.abs()
    by = (er + 8 * E) * mag + _u(dt) * y.abs() + _tiny(dt)
    if gy is None:
        return y, by
    g = gy.double()
    g, gm = _rot_ref(g, c, s, inter, True) if cos is not None else (g, g.abs())
    hat = x * r
    dw = (g * hat).sum((0, 1, 2))
    cnt = x.numel() // d
    # products of values off by (er + 8 e); a sum of cnt terms in f32: lanes, groups, blocks one after another
    bw = (er + 16 * E + (math.sqrt(cnt) + 64) * E) * (gm * hat.abs()).sum((0, 1, 2))
    gw, gwm = g * ww, gm * ww.abs()
    if w is None:
        return y, by, gw, 8 * E * gwm + _u(dt) * gw.abs() + _tiny(dt), dw, bw
    mean, mm = (gw * hat).mean(-1, keepdim=True), (gwm * hat.abs()).mean(-1, keepdim=True)
    dx = r * (gw - hat * mean)
    bx = r * ((2 * er + 16 * E) * gwm + hat.abs() * mm * (4 * er + (d + 16) * E)) + _u(dt) * dx.abs() + _tiny(dt)
    return y, by, dx, bx, dw, bw


def _within(got, ref, bound, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got.double() - ref).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0 and not torch.isnan(off).any(), \
        f"{what}: past its bound by {worst:.3e} (off {off.max().item():.3e}, bound {bound.max().item():.3e})"


QK_CASES = [
    # b, n, hq, hk, d, rot, interleaved, norm, positions
    (1, 1, 8, 2, 128, 128, False, True, "far"),
    (2, 37, 4, 4, 128, 128, False, True, None),
    (3, 65, 12, 12, 64, 64, True, True, None),
    (2, 19, 6, 2, 80, 40, True, True, "row"),       # 20 rotated pairs: 4-element units
    (2, 19, 3, 1, 72, 36, False, True, None),       # 18 pairs: single elements
    (1, 33, 2, 2, 96, 0, False, True, None),        # norm alone
    (2, 21, 4, 2, 32, 16, False, False, "i64"),     # rotation alone
    (1, 5, 1, 1, 2, 2, False, True, None),
    (1, 9, 2, 1, 512, 512, False, True, None),
    (1, 9, 2, 1, 258, 130, True, True, None),       # four units a lane
    (4, 700, 5, 3, 128, 64, False, True, None),     # several heads a lane group, a partial last chunk
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", QK_CASES)
def test_qk_norm_rope_vs_float64(case, dt):
    b, n, hq, hk, d, rot, inter, norm, where = case
    rows = _randn((b, n, hq + 2 * hk, d), dt, 1, 1.5)
    q, k = rows[:, :, :hq].detach().requires_grad_(), rows[:, :, hq:hq + hk].detach().requires_grad_()
    wq, wk = [(1 + 0.2 * _randn((d,), torch.float32, s)).requires_grad_() if norm else None for s in (2, 3)]
    cos = sin = positions = None
    pos = torch.arange(n, device=DEV).expand(b, n)
    if rot:
        table = 70000 if where == "far" else max(n, 300)
        cos, sin = A.rope_table(table, rot, device=DEV)
        if where == "far":
            pos = positions = torch.full((b, n), 69999, dtype=torch.int32, device=DEV)
        elif where == "row":
            pos = torch.randint(0, table, (n,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
            positions, pos = pos.int(), pos.expand(b, n)
        elif where == "i64":
            pos = positions = torch.randint(0, table, (b, n), device=DEV,
                                            generator=torch.Generator(device=DEV).manual_seed(4))
        pos = pos.long()
    yq, yk = A.qk_norm_rope(q, k, cos, sin, positions, wq, wk, 1e-6, inter)
    gq, gk = _randn((b, n, hq, d), dt, 5), _randn((b, n, hk, d), dt, 6)
    ins = [q, k] + ([wq, wk] if norm else [])
    grads = torch.autograd.grad((yq, yk), ins, (gq, gk))
    for i, (x, y, w, g) in enumerate(((q, yq, wq, gq), (k, yk, wk, gk))):
        y0, by, dx, bx, dw, bw = _qk_ref(x.detach(), None if w is None else w.detach(), cos, sin, pos, 1e-6, inter, g, dt)
        _within(y.detach(), y0, by, f"y{i}")
        _within(grads[i], dx, bx, f"dx{i}")
        if norm:
            _within(grads[2 + i], dw, bw, f"dw{i}")
    with torch.no_grad():  # the path without autograd
        yq2, yk2 = A.qk_norm_rope(q, k, cos, sin, positions, wq, wk, 1e-6, inter)
    assert torch.equal(yq2, yq) and torch.equal(yk2, yk)


def test_qk_norm_rope_against_differences():
    """The input and weight gradients against central differences of the f32 forward, along one direction each
    (third-order remainder and the f32 forward's rounding over 2 h: both far below 1e-2 of the slope)."""
    b, n, hq, hk, d = 2, 5, 2, 1, 32
    q, k = (_randn((b, n, h, d), torch.float32, s).requires_grad_() for h, s in ((hq, 1), (hk, 2)))
    w = [(1 + 0.1 * _randn((d,), torch.float32, s)).requires_grad_() for s in (3, 4)]
    cos, sin = A.rope_table(n, d, device=DEV)
    gq, gk = _randn(q.shape, torch.float32, 5), _randn(k.shape, torch.float32, 6)

    def f(q, k, wq, wk):
        y = A.qk_norm_rope(q, k, cos, sin, None, wq, wk)
        return y[0], y[1]

    grads = torch.autograd.grad(f(q, k, *w), (q, k, *w), (gq, gk))
    ins = [t.detach() for t in (q, k, *w)]
    h = 1e-2
    for i, t in enumerate(ins):
        dirn = _randn(t.shape, torch.float32, 20 + i)
        val = []
        for sgn in (1, -1):
            args = list(ins)
            args[i] = t + sgn * h * dirn
            y = f(*args)
            val.append((y[0].double() * gq.double()).sum() + (y[1].double() * gk.double()).sum())
        slope = ((val[0] - val[1]) / (2 * h)).item()
        want = (grads[i].double() * dirn.double()).sum().item()
        size = grads[i].double().norm().item() * dirn.double().norm().item()
        assert abs(slope - want) <= 1e-2 * size, (i, slope, want)


def test_qk_norm_rope_positions_outside_the_table_are_nan():
    q, k = _randn((1, 4, 2, 32), torch.bfloat16, 1), _randn((1, 4, 1, 32), torch.bfloat16, 2)
    cos, sin = A.rope_table(8, 16, device=DEV)
    pos = torch.tensor([[0, 8, -1, 7]], dtype=torch.int32, device=DEV)
    y, _ = A.qk_norm_rope(q, k, cos, sin, pos, torch.ones(32, device=DEV), torch.ones(32, device=DEV))
    bad = torch.isnan(y).float()
    assert bad[0, [0, 3]].sum() == 0
    assert bad[0, [1, 2], :, :16].min() == 1 and bad[0, [1, 2], :, 16:].sum() == 0


def test_qk_norm_rope_empty_and_deterministic():
    w = torch.ones(64, device=DEV, requires_grad=True)
    q, k = torch.empty(0, 7, 4, 64, device=DEV, requires_grad=True), torch.empty(0, 7, 2, 64, device=DEV)
    y = A.qk_norm_rope(q, k, q_weight=w, k_weight=w)
    g = torch.autograd.grad(y, (q, w), [torch.zeros_like(t) for t in y])
    assert y[0].shape == q.shape and g[0].shape == q.shape and g[1].eq(0).all()
    q, k = _randn((2, 3000, 4, 64), torch.bfloat16, 1).requires_grad_(), _randn((2, 3000, 2, 64), torch.bfloat16, 2)
    gy = [_randn(t.shape, torch.bfloat16, 3) for t in (q, k)]
    a, b = [torch.autograd.grad(A.qk_norm_rope(q, k, q_weight=w, k_weight=w), (q, w), gy) for _ in range(2)]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---------------------------------------------------------------- attention
def _see(b, lq, lk, causal, kv_lens, prefix, docs):
    """[b, lq, lk] visibility and the query positions [b, lq], written out query by query."""
    see = torch.zeros(b, lq, lk, dtype=torch.bool)
    at = torch.zeros(b, lq, dtype=torch.long)
    for i in range(b):
        n = lk if kv_lens is None else min(max(int(kv_lens[i]), 0), lk)
        pre = 0 if prefix is None else int(prefix[i])
        j = torch.arange(lk)
        for r in range(lq):
            p = n - lq + r
            at[i, r] = p
            ok = j < n
            first = 0
            if docs is not None:
                if p < 0 or docs[i, p] < 0:
                    continue
                first = p
                while first > 0 and docs[i, first - 1] == docs[i, p]:
                    first -= 1
                last = p
                while last + 1 < n and docs[i, last + 1] == docs[i, p]:
                    last += 1
                ok &= (j >= first) & (j <= last)
            if causal:
                ok &= (j <= p) | (j < first + pre)
            see[i, r] = ok
    return see, at


def _attn_ref(q, k, v, see, at, scale, cap, slopes, go):
    """o, dq, dk, dv in 64 bits with the bounds of this file's docstring."""
    dt = q.dtype
    u = _u(dt) if dt != torch.float32 else 0.0
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    g = hq // hk
    see = see.to(DEV)[:, None]
    Q = q.double().permute(0, 2, 1, 3)
    K, V = (t.double().permute(0, 2, 1, 3).repeat_interleave(g, 1) for t in (k, v))
    anyk, anyq = see.any(2)[:, :, :, None], see.any(3)[..., None]
    K, V = K.masked_fill(~anyk, 0.0), V.masked_fill(~anyk, 0.0)   # what nobody sees may hold anything
    Q = Q.masked_fill(~anyq, 0.0)
    z = scale * Q @ K.transpose(-1, -2)
    zabs = scale * Q.abs() @ K.abs().transpose(-1, -2)
    D = (d + 4) * E * zabs
    s, bend = z, torch.ones_like(z)
    if cap:
        t = torch.tanh(z / cap)
        s, bend = cap * t, 1 - t * t
        D = D + 10 * E * cap
    if slopes is not None:
        far = (at.to(DEV)[:, None, :, None] - torch.arange(lk, device=DEV)).abs()
        s = s - slopes.double()[None, :, None, None] * far
    D = D + 8 * E * s.abs()
    D = D.masked_fill(~see, 0.0)
    p = torch.softmax(s.masked_fill(~see, float("-inf")), -1).masked_fill(~see, 0.0)
    D = D.amax(-1, keepdim=True)
    n = see.sum(-1, keepdim=True).double()
    o, mag = p @ V, p @ V.abs()
    tiny, sees = _tiny(dt), see.double()
    bo = (2 * D + u + (n + 8) * E) * mag + (u or _u(dt)) * o.abs() + tiny * (sees @ V.abs() + 1)
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    if go is None:
        return back(o), back(bo)
    G = go.double().permute(0, 2, 1, 3).masked_fill(~anyq, 0.0)
    dp = G @ V.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * bend
    Edp = (d + 4) * E * (G.abs() @ V.abs().transpose(-1, -2)).masked_fill(~see, 0.0).amax(-1, keepdim=True)
    Edel = (G.abs() * mag).sum(-1, keepdim=True) * (2 * D + u + (n + d + 16) * E)
    # bend = 1 - t^2 errs by 2 |t| (D / cap + 4 e) + 2 e, absolute
    bb = (2 * (D / cap) + 16 * E) if cap else 0.0
    eds = (u + 4 * D + 8 * E) * ds.abs() + p * (Edp + Edel) + bb * p * (dp - delta).abs()
    dq, dk, dv = scale * ds @ K, scale * ds.transpose(-1, -2) @ Q, p.transpose(-1, -2) @ G
    nk = see.sum(2).double()[..., None] * g
    eds = eds + tiny * sees * (1 + (dp - delta).abs())
    bq = scale * (eds @ K.abs() + (n + 8) * E * ds.abs() @ K.abs()) + tiny
    bk = scale * (eds.transpose(-1, -2) @ Q.abs()) + (nk + 8) * E * scale * (ds.abs().transpose(-1, -2) @ Q.abs()) + tiny
    bv = ((2 * D + u) * p + tiny * sees).transpose(-1, -2) @ G.abs() + tiny + (nk + 8) * E * (p.transpose(-1, -2) @ G.abs())
    fold = lambda t: t.reshape(b, hk, g, lk, d).sum(2)  # noqa: E731
    dk, dv, bk, bv = fold(dk), fold(dv), fold(bk), fold(bv)
    r = u or _u(dt)
    return [back(t) for t in (o, bo, dq, bq + r * dq.abs(), dk, bk + r * dk.abs(), dv, bv + r * dv.abs())]


def _docs(b, n, lens, pad, seed):
    ids = torch.full((b, n), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(seed)
    for i in range(b):
        at = 0
        for d in range(10 ** 6):
            m = int(torch.randint(1, lens + 1, (1,), generator=g))
            if at + m > n - pad:
                break
            ids[i, at:at + m] = d
            at += m
    return ids


def _attn_case(b, lq, lk, hq, hk, d, dt, causal=False, kv_lens=None, prefix=None, docs=None, cap=0.0, slopes=False,
               packed=False, grad=True, seed=0, scale=None):
    if packed:
        rows = _randn((b, lq, hq + 2 * hk, d), dt, seed, 1.5)
        q, k, v = rows[:, :, :hq], rows[:, :, hq:hq + hk], rows[:, :, hq + hk:]
    else:
        q, k, v = _randn((b, lq, hq, d), dt, seed, 1.5), _randn((b, lk, hk, d), dt, seed + 1, 1.5), _randn((b, lk, hk, d), dt, seed + 2)
    sl = torch.tensor([2.0 ** (-4.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if slopes else None
    i32 = lambda t: None if t is None else torch.as_tensor(t, dtype=torch.int32)  # noqa: E731
    kv_lens, prefix, docs = i32(kv_lens), i32(prefix), i32(docs)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    q, k, v = (t.detach().requires_grad_(grad) for t in (q, k, v))
    o = A.attention(q, k, v, scale=scale, softcap=cap, slopes=sl, causal=causal, kv_lens=dev(kv_lens),
                    prefix=dev(prefix), documents=dev(docs))
    see, at = _see(b, lq, lk, causal, kv_lens, prefix, docs)
    go = _randn((b, lq, hq, d), dt, seed + 3) if grad else None
    ref = _attn_ref(q.detach(), k.detach(), v.detach(), see, at, scale or d ** -0.5, cap, sl, go)
    _within(o.detach(), ref[0], ref[1], "o")
    if grad:
        g = torch.autograd.grad(o, (q, k, v), go)
        for i, name in enumerate(("dq", "dk", "dv")):
            _within(g[i], ref[2 + 2 * i], ref[3 + 2 * i], name)
        with torch.no_grad():
            o2 = A.attention(q, k, v, scale=scale, softcap=cap, slopes=sl, causal=causal, kv_lens=dev(kv_lens),
                             prefix=dev(prefix), documents=dev(docs))
        _within(o2, ref[0], ref[1], "o without a gradient")
    return o


SHAPES = [
    # b, lq, lk, hq, hk, d
    (1, 1, 1, 1, 1, 8),
    (2, 7, 7, 4, 4, 128),
    (1, 33, 33, 4, 2, 64),
    (2, 130, 130, 6, 2, 32),
    (1, 257, 257, 3, 1, 80),
    (1, 200, 200, 2, 2, 96),
    (1, 129, 129, 4, 1, 128),
]
MODES = [dict(), dict(causal=True), dict(cap=20.0), dict(slopes=True, causal=True), dict(cap=5.0, slopes=True)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("mode", MODES, ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_vs_float64(shape, mode, dt):
    _attn_case(*shape, dt, **mode)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_key_lengths(causal, dt):
    """Lengths of 0, 1, inside a tile, at its edge, full, past the end and negative (clamped)."""
    _attn_case(8, 70, 140, 4, 2, 64, dt, causal=causal, kv_lens=[0, 1, 63, 64, 65, 140, 999, -5], cap=30.0)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_prefix(dt):
    _attn_case(5, 150, 150, 2, 1, 64, dt, causal=True, prefix=[0, 1, 64, 150, 400], slopes=True)
    _attn_case(3, 40, 150, 2, 1, 64, dt, causal=True, prefix=[120, 3, 0], kv_lens=[150, 99, 20])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_documents(causal, dt):
    """Packed documents of unequal length (many of one token), padding between and behind them, rows of padding."""
    docs = _docs(3, 300, 60, 40, 1)
    docs[0, 100:130] = -1
    docs[1] = _docs(1, 300, 3, 0, 2)[0]
    docs[2] = -1
    _attn_case(3, 300, 300, 4, 2, 64, dt, causal=causal, docs=docs, cap=30.0)
    # the keys of one long row split over workgroups: documents across the cuts, tiles that start off their grid
    assert N.load().dmf_mattn_fwd_ws_floats(N.dtype_code(dt), 1, 1100, 1100, 2, 1, 64, 0) > 0
    _attn_case(1, 1100, 1100, 2, 1, 64, dt, causal=causal, docs=_docs(1, 1100, 90, 10, 4))
    _attn_case(1, 1100, 1100, 2, 1, 64, dt, causal=causal, docs=_docs(1, 1100, 700, 10, 5))


def test_attention_documents_with_prefix_cache_and_lengths():
    docs = _docs(3, 200, 70, 0, 3)
    _attn_case(3, 200, 200, 2, 2, 128, torch.bfloat16, causal=True, docs=docs, prefix=[5, 0, 300])
    _attn_case(3, 50, 200, 2, 2, 128, torch.bfloat16, causal=True, docs=docs, kv_lens=[200, 70, 31])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hq,hk,lk", [(4, 4, 577), (8, 2, 1), (8, 1, 2050), (32, 8, 300), (32, 1, 999)])
def test_attention_single_query(hq, hk, lk, dt):
    _attn_case(2, 1, lk, hq, hk, 128, dt, causal=True, kv_lens=[lk, (lk + 1) // 2], cap=30.0, grad=False)
    _attn_case(2, 1, lk, hq, hk, 64, dt, slopes=True, causal=True, kv_lens=[0, lk], grad=False)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq", [2, 9, 100])
def test_attention_few_queries_split_over_keys(lq, dt):
    """Few rows against many keys: the keys are split over workgroups and joined, also for training."""
    n = N.load().dmf_mattn_fwd_ws_floats(N.dtype_code(dt), 2, lq, 3000, 4, 2, 64, 1)
    assert n > 0
    _attn_case(2, lq, 3000, 4, 2, 64, dt, causal=True, kv_lens=[3000, 700], slopes=True)
    _attn_case(1, lq, 3000, 4, 2, 64, dt, causal=True, prefix=[1500], cap=20.0, grad=False)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_packed_views_and_expanded_heads(dt):
    _attn_case(2, 100, 100, 4, 4, 64, dt, packed=True, cap=20.0)
    # head-major storage, a batch that shares one key row, an unaligned base (copied)
    q = _randn((2, 4, 90, 64), dt, 1).transpose(1, 2)
    k = _randn((1, 90, 2, 64), dt, 2).expand(2, 90, 2, 64)
    flat = _randn((2 * 90 * 2 * 64 + 1,), dt, 3)
    v = flat[1:].view(2, 90, 2, 64)
    see, at = _see(2, 90, 90, False, None, None, None)
    o = A.attention(q, k, v)
    ref, bound = _attn_ref(q, k, v, see, at, 0.125, 0.0, None, None)
    _within(o, ref, bound, "o")


@pytest.mark.parametrize("dt", TYPES)
def test_attention_garbage_where_nothing_is_seen(dt):
    """NaN and infinities in keys, values, queries and output gradients that a mask hides do not get through:
    beyond kv_len, in the future of a causal mask, in padding and in other documents."""
    b, n, hq, hk, d = 3, 160, 4, 2, 64
    docs = torch.zeros(b, n, dtype=torch.int32)
    docs[0, 100:] = -1
    docs[1, 70:] = 1
    docs[2, 150:] = -1
    see, at = _see(b, n, n, True, None, None, docs)
    q, k, v, go = (_randn((b, n, h, d), dt, s) for h, s in ((hq, 1), (hk, 2), (hk, 3), (hq, 4)))
    # row 0: everything in the padding; row 1: the second document's last key and query; row 2: the padding's values
    for t, fill in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (go, float("-inf"))):
        t[0, 100:] = fill
    k[1, 159] = float("nan")
    v[1, 159] = float("inf")
    go[1, 159] = float("nan")
    v[2, 155] = float("nan")
    seen = torch.ones(b, n, dtype=torch.bool)
    seen[1, 70:] = False     # dq of query 159 and all that its key and value touch (the second document)
    qq, kk, vv = (t.detach().requires_grad_() for t in (q, k, v))
    o = A.attention(qq, kk, vv, causal=True, documents=docs.to(DEV))
    dq, dk, dv = torch.autograd.grad(o, (qq, kk, vv), go)
    clean = [t.clone() for t in (q, k, v, go)]
    for t in clean:
        t[~torch.isfinite(t)] = 0.0
    ref = _attn_ref(*clean[:3], see, at, d ** -0.5, 0.0, None, clean[3])
    hide = (~seen).to(DEV)[:, :, None, None]
    for got, r, bound, what in ((o, ref[0], ref[1], "o"), (dq, ref[2], ref[3], "dq"), (dk, ref[4], ref[5], "dk"),
                                (dv, ref[6], ref[7], "dv")):
        _within(got.detach().masked_fill(hide, 0.0), r.masked_fill(hide, 0.0), bound, what)
    # in the second document only the last query sees the bad key: the outputs and dq before it are untouched
    keep = torch.zeros(b, n, dtype=torch.bool)
    keep[1, 70:159] = True
    keep = keep.to(DEV)[:, :, None, None]
    _within(o.detach().masked_fill(~keep, 0.0), ref[0].masked_fill(~keep, 0.0), ref[1], "o before a bad key")
    _within(dq.masked_fill(~keep, 0.0), ref[2].masked_fill(~keep, 0.0), ref[3], "dq before a bad key")
    assert torch.isnan(o[1, 159]).all()


def test_attention_against_differences():
    b, n, hq, hk, d = 1, 21, 4, 2, 16
    q, k, v = (_randn((b, n, h, d), torch.float32, s).requires_grad_() for h, s in ((hq, 1), (hk, 2), (hk, 3)))
    go = _randn((b, n, hq, d), torch.float32, 4)
    sl = torch.tensor([0.3, 0.1, 0.05, 0.01], device=DEV)
    docs = torch.tensor([[0] * 13 + [1] * 6 + [-1] * 2], dtype=torch.int32, device=DEV)

    def f(q, k, v):
        return A.attention(q, k, v, softcap=3.0, slopes=sl, causal=True, documents=docs)

    grads = torch.autograd.grad(f(q, k, v), (q, k, v), go)
    ins = [t.detach() for t in (q, k, v)]
    h = 1e-2
    for i, t in enumerate(ins):
        dirn = _randn(t.shape, torch.float32, 30 + i)
        val = []
        for sgn in (1, -1):
            args = list(ins)
            args[i] = t + sgn * h * dirn
            val.append((f(*args).double() * go.double()).sum())
        slope = ((val[0] - val[1]) / (2 * h)).item()
        want = (grads[i].double() * dirn.double()).sum().item()
        size = grads[i].double().norm().item() * dirn.double().norm().item()
        # second differences: h^2 times third derivatives of order one, and f32 rounding over 2 h
        assert abs(slope - want) <= 1e-2 * size, (i, slope, want, size)


def test_attention_empty_sizes():
    for b, lq, lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q = torch.randn(b, lq, 4, 32, device=DEV, requires_grad=True)
        k, v = (torch.randn(b, lk, 2, 32, device=DEV, requires_grad=True) for _ in range(2))
        o = A.attention(q, k, v)
        g = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert o.shape == q.shape and o.eq(0).all() and all(t.eq(0).all() for t in g)


def test_attention_same_bits_every_run():
    q, k, v = (_randn((2, 500, h, 64), torch.bfloat16, s).requires_grad_() for h, s in ((8, 1), (2, 2), (2, 3)))
    go = _randn((2, 500, 8, 64), torch.bfloat16, 4)
    runs = []
    for _ in range(3):
        o = A.attention(q, k, v, causal=True, softcap=20.0)
        runs.append((o.detach(), *torch.autograd.grad(o, (q, k, v), go)))
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


def test_attention_refusals():
    q, k, v = (_randn((2, 5, h, 64), torch.bfloat16, 1) for h in (4, 2, 2))
    bad = [
        (dict(), (q, k[:, :4], v)), (dict(), (q[:, :, :3], k, v)), (dict(), (q.float(), k, v)),
        (dict(), (q[..., :60], k[..., :60], v[..., :60])), (dict(scale=-1.0), (q, k, v)), (dict(scale=0.0), (q, k, v)),
        (dict(softcap=-2.0), (q, k, v)), (dict(softcap=float("nan")), (q, k, v)),
        (dict(prefix=torch.ones(2, dtype=torch.int32, device=DEV)), (q, k, v)),
        (dict(kv_lens=torch.ones(3, dtype=torch.int32, device=DEV)), (q, k, v)),
        (dict(kv_lens=torch.ones(2, device=DEV)), (q, k, v)),
        (dict(kv_lens=torch.ones(2, dtype=torch.int32)), (q, k, v)),
        (dict(documents=torch.ones(2, 4, dtype=torch.int32, device=DEV)), (q, k, v)),
        (dict(slopes=torch.ones(2, device=DEV)), (q, k, v)),
        (dict(slopes=torch.ones(4, device=DEV, requires_grad=True)), (q, k, v)),
        (dict(), (q[0], k, v)), (dict(), (q.int(), k.int(), v.int())),
    ]
    for kw, args in bad:
        with pytest.raises(ValueError, match="attention"):
            A.attention(*args, **kw)
    wide = _randn((1, 2, 1, 136), torch.bfloat16, 1)
    with pytest.raises(ValueError, match="head dim"):
        A.attention(wide, wide, wide)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.attention(q.cpu(), k.cpu(), v.cpu())


def test_qk_norm_rope_refusals():
    q, k = (_randn((2, 5, h, 64), torch.bfloat16, 1) for h in (4, 2))
    w = torch.ones(64, device=DEV)
    c, s = A.rope_table(5, 64, device=DEV)
    c4, s4 = A.rope_table(4, 64, device=DEV)
    pos = torch.zeros(2, 5, dtype=torch.int32, device=DEV)
    bad = [
        dict(), dict(q_weight=w), dict(q_weight=w, k_weight=w[:32]), dict(q_weight=w, k_weight=w.bfloat16()),
        dict(cos=c), dict(cos=c, sin=s[:, :8]), dict(cos=c4, sin=s4), dict(cos=c.double(), sin=s.double()),
        dict(cos=c, sin=s, positions=pos[:, :4]), dict(cos=c, sin=s, positions=pos.float()),
        dict(q_weight=w, k_weight=w, positions=pos), dict(q_weight=w, k_weight=w, eps=-1.0),
        dict(cos=c.clone().requires_grad_(), sin=s),
    ]
    for kw in bad:
        with pytest.raises(ValueError, match="qk_norm_rope"):
            A.qk_norm_rope(q, k, **kw)
    with pytest.raises(ValueError, match="differ"):
        A.qk_norm_rope(q, k[:, :4], c, s)
    with pytest.raises(ValueError, match="even"):
        A.qk_norm_rope(q[..., :63], k[..., :63], q_weight=w[:63], k_weight=w[:63])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_backward_of_many_key_blocks(d, dt):
    """More than one 128-key block for each CU (other tests have fewer, and blocks of 64 keys in 16-bit types): walks that a
    mask makes unequal, equal ones, and more blocks than two for each CU."""
    lens = [200, 1, 128, 129, 0, 150, 200, 77, 200]
    _attn_case(9, 200, 200, 32, 16, d, dt, causal=True, kv_lens=lens)
    _attn_case(9, 200, 200, 32, 16, d, dt, cap=20.0)
    _attn_case(9, 200, 200, 16, 16, d, dt, causal=True, docs=_docs(9, 200, 90, 20, 1))
    _attn_case(18, 150, 130, 32, 16, d, dt, causal=True, kv_lens=lens * 2, slopes=True)
    _attn_case(5, 200, 200, 32, 16, d, dt, docs=_docs(5, 200, 150, 20, 2))


def test_attention_backward_of_many_key_blocks_hides_garbage():
    """What a key's value or a query's gradient holds stays with the pairs that see it, in the 4-wave form too."""
    b, n, h, d = 9, 140, 16, 64
    q, k, v, go = (_randn((b, n, h, d), torch.bfloat16, s) for s in (1, 2, 3, 4))
    v[:, 139] = float("inf")       # seen by the last query alone
    go[:, 0] = float("nan")        # sees the first key alone
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o = A.attention(q, k, v, causal=True)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), go)
    see, at = _see(b, n, n, True, None, None, None)
    fin = [torch.where(torch.isfinite(t.detach()), t.detach(), 0.0) for t in (q, k, v, go)]
    ref = _attn_ref(*fin[:3], see, at, d ** -0.5, 0.0, None, fin[3])
    _within(o.detach()[:, :139], ref[0][:, :139], ref[1][:, :139], "o")
    _within(dq[:, 1:139], ref[2][:, 1:139], ref[3][:, 1:139], "dq")
    assert torch.isnan(dk).any() and torch.isnan(dv[:, 0]).all()
    _within(dv[:, 1:], ref[6][:, 1:], ref[7][:, 1:], "dv")


def test_attention_wide_integers():
    """64-bit ids and lengths keep their meaning past 32 bits: ids that agree in their low halves differ, those past 2^31
    are no padding, lengths and prefixes are clamped."""
    b, n, h, d = 2, 150, 2, 64
    low = _docs(b, n, 40, 20, 7)
    low[1, 60:90] = low[1, 30]          # one run in the low halves, three in the ids
    low[1, 30:60] = low[1, 30]
    wide = low.long()
    wide[1, 60:75] += 2 ** 32
    wide[1, 75:90] += 2 ** 31
    wide[0, :40] = torch.where(wide[0, :40] >= 0, wide[0, :40] + 2 ** 31 + 5, -2 ** 40)
    names = {int(x): i for i, x in enumerate(sorted(set(wide[wide >= 0].tolist())))}
    small = torch.tensor([[names[int(x)] if x >= 0 else -1 for x in r] for r in wide], dtype=torch.int32)
    q, k, v = (_randn((b, n, h, d), torch.bfloat16, s) for s in (1, 2, 3))
    for causal in (False, True):
        got = A.attention(q, k, v, causal=causal, documents=wide.to(DEV))
        assert torch.equal(got, A.attention(q, k, v, causal=causal, documents=small.to(DEV)))
        see, at = _see(b, n, n, causal, None, None, small)
        _within(got, *_attn_ref(q, k, v, see, at, d ** -0.5, 0.0, None, None), "o")
    lens = torch.tensor([2 ** 32 + 3, -2 ** 32 + 9], device=DEV)
    got = A.attention(q, k, v, causal=True, kv_lens=lens, prefix=lens)
    want = A.attention(q, k, v, causal=True, kv_lens=torch.tensor([n, 0], device=DEV), prefix=torch.tensor([n, 0], device=DEV))
    assert torch.equal(got, want) and not want[1].any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("mode", [dict(), dict(cap=20.0), dict(slopes=True), dict(cap=5.0, slopes=True)], ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("shape", [(32, 130, 127, 16, 8, 128), (17, 129, 97, 20, 20, 64), (41, 257, 33, 10, 10, 32)])
def test_attention_three_workgroups_a_cu(shape, mode, dt):
    """Unmasked rows whose workgroups come to three or five a CU (32-key tiles): odd key counts, shared heads."""
    _attn_case(*shape, dt, **mode)
