"""Token attention between a block's qkv projection and its output projection: the per-head norm of
queries and keys with the position rotation (``qk_norm_rope``), and attention with capped scores, a
distance bias and causal / prefix / document masks over shared key heads (``attention``), for training
and for single tokens against a long cache.

The reference's MultiHeadSelfAttention (transformer_model.py:83-116) is the case without any of these
(dmf_tokens); the blocks of transformer_model.TransformerStage take them as options. Both ops run on
csrc/qknorm.hip and csrc/masked_attn*.h through the C-ABI, on torch's current stream, with every
workspace from torch's allocator, so they can be captured into a graph; sizes are checked on the host, and
device-side values (positions, lengths, ids) are bounds-checked in the kernels. A backward is captured, as with
torch's own ops, on leaves that no eager graph still holds: torch's gradient accumulation would wait for that graph's
stream inside the capture.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

import dmf_native as N

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


def _launch(name, dev, *args):
    """N.call on ``dev``'s current stream; launches go to the tensors' device, also where another one is current."""
    if dev.index == torch.cuda.current_device():
        N.call(name, *args, N.stream_ptr(dev))
    else:
        with torch.cuda.device(dev):
            N.call(name, *args, N.stream_ptr(dev))


def _p(t):
    return None if t is None else t.data_ptr()


def _heads(what, name, t, like=None):
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"{what}: {name} must be [batch, length, heads, head_dim], got "
                         f"{tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__}")
    if not t.is_cuda:
        N.require_cuda(t)
    if like is None:
        if t.dtype not in _DTYPES:
            raise ValueError(f"{what}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    elif t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")


def _no_tangents(what, *tensors):
    """Forward-mode derivatives are refused: the kernels would drop the tangents."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: forward-mode derivatives are not supported")


def _strided(t, align, apart=0):
    """(tensor, (batch, token, head) strides) with contiguous head dims; strides and base multiples of ``align``
    elements and tokens at least ``apart`` elements apart, else of a contiguous copy."""
    n0, n1, n2, n3 = t.shape
    s0, s1, s2, s3 = t.stride()
    # (the stride of a dim of length 1 says nothing)
    s0, s1, s2 = (s0 if n0 > 1 else 0), (s1 if n1 > 1 else apart), (s2 if n2 > 1 else 0)
    if ((s3 == 1 or n3 == 1) and s0 % align == 0 and s1 % align == 0 and s2 % align == 0 and s1 >= apart
            and t.data_ptr() % (align * t.element_size()) == 0):
        return t, (s0, s1, s2)
    if t.is_contiguous():  # an unaligned base
        t = t.clone(memory_format=torch.contiguous_format)
    else:
        t = t.contiguous()
    return t, (n1 * n2 * n3, n2 * n3, n3)


def _plain(t):
    """Contiguous, 16-byte aligned form of a gradient."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _small(what, name, t, shape, dtype, device):
    if t.dtype == dtype and t.shape == shape and t.device == device and t.is_contiguous():
        return t
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: {name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, expected {device}")
    if t.is_floating_point() != dtype.is_floating_point or t.dtype == torch.bool:
        raise ValueError(f"{what}: {name} must be {dtype}, got {t.dtype}")
    if dtype == torch.int32:  # (a wider integer past 32 bits keeps its meaning as a bound)
        t = t.clamp(-2 ** 31, 2 ** 31 - 1) if t.dtype == torch.int64 else t
    return t.to(dtype).contiguous()


# -------------------------------------------------------- norm and rotation
def rope_table(length, dims, theta=10000.0, device=None):
    """(cos, sin), each f32 [length, dims / 2]: pair p of position t turns by t * theta^(-2 p / dims)
    (angles in 64 bits: far positions keep their phase)."""
    if dims < 2 or dims % 2 or length < 1:
        raise ValueError(f"rope_table: dims {dims} must be even and positive, length {length} positive")
    f = theta ** (-torch.arange(dims // 2, dtype=torch.float64, device=device) * 2 / dims)
    a = torch.arange(length, dtype=torch.float64, device=device)[:, None] * f
    return a.cos().float(), a.sin().float()


def rope_table_2d(height, width, dims, theta=100.0, device=None):
    """(cos, sin), each f32 [height * width, dims / 2], of a token grid in row-major order: the first half of
    the pairs turns with the row, the rest with the column."""
    if dims < 4 or dims % 4 or height < 1 or width < 1:
        raise ValueError(f"rope_table_2d: dims {dims} must be a positive multiple of 4, the grid {height} x {width} not empty")
    c, s = rope_table(max(height, width), dims // 2, theta, device)
    y = torch.arange(height, device=device).repeat_interleave(width)
    x = torch.arange(width, device=device).repeat(height)
    return torch.cat([c[y], c[x]], 1).contiguous(), torch.cat([s[y], s[x]], 1).contiguous()


def _qk_call(name, q, k, cos, sin, pos, wq, wk, norm, eps, interleaved, *rest):
    b, n, hq, d = q.shape
    q, qs = _strided(q, 1)
    k, ks = _strided(k, 1)
    rows, rot = (0, 0) if cos is None else (cos.shape[0], 2 * cos.shape[1])
    pos_sb = 0 if pos is None or pos.dim() == 1 else pos.stride(0)
    _launch(name, q.device, _DTYPES[q.dtype], q.data_ptr(), *qs, hq, k.data_ptr(), *ks, k.shape[2], b, n, d, rot,
            interleaved, norm, eps, _p(wq), _p(wk), _p(cos), _p(sin), _p(pos), pos_sb,
            pos is not None and pos.dtype == torch.int64, rows, *rest)


def _qk_fwd(q, k, cos, sin, pos, wq, wk, norm, eps, interleaved):
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _qk_call("dmf_qk_norm_rope", q, k, cos, sin, pos, wq, wk, norm, eps, interleaved, qo.data_ptr(), ko.data_ptr())
    return qo, ko


def _qk_bwd(q, k, cos, sin, pos, wq, wk, norm, eps, interleaved, gq, gk, weights):
    """dq, dk and, with ``weights``, dwq, dwk (else None)."""
    gq, gk = _plain(gq), _plain(gk)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dwq = dwk = ws = None
    if weights:
        d = q.shape[3]
        dwq, dwk = torch.empty((2, d), dtype=torch.float32, device=q.device)
        ws = torch.empty(N.load().dmf_qk_norm_rope_bwd_ws_floats(q.shape[2], k.shape[2], d), dtype=torch.float32,
                         device=q.device)
    _qk_call("dmf_qk_norm_rope_bwd", q, k, cos, sin, pos, wq, wk, norm, eps, interleaved, gq.data_ptr(), gk.data_ptr(),
             dq.data_ptr(), dk.data_ptr(), _p(dwq), _p(dwk), _p(ws))
    return dq, dk, dwq, dwk


class _QkNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, pos, norm, eps, interleaved):
        ctx.save_for_backward(q, k, wq, wk, cos, sin, pos)
        ctx.cfg = (norm, eps, interleaved)
        return _qk_fwd(q, k, cos, sin, pos, wq, wk, *ctx.cfg)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, cos, sin, pos = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = _qk_bwd(q, k, cos, sin, pos, wq, wk, *ctx.cfg, gq, gk, need[2] or need[3])
        return tuple(x if n else None for x, n in zip(g, need)) + (None,) * 6


def qk_norm_rope(q, k, cos=None, sin=None, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    """Norm and rotation of queries [b, n, hq, d] and keys [b, n, hk, d] (any strides, e.g. views of packed qkv
    rows) in one pass: ``rot(x * rsqrt(mean(x^2) + eps) * weight)`` per head, in 32 bits, rounded once. Returns
    contiguous (q, k); differentiable in q, k and the weights.

    ``q_weight`` / ``k_weight`` f32 [d]: both given, or both None for the rotation alone (no norm).
    ``cos`` / ``sin`` f32 [rows, rot / 2] (rope_table, rope_table_2d): the first ``rot`` dims turn, as pairs
    (p, p + rot / 2) or, ``interleaved``, (2p, 2p + 1); None for the norm alone. ``positions`` int [b, n] or
    [n]: each token's table row (default: its index); one outside the table makes its rotated dims NaN.
    """
    what = "qk_norm_rope"
    _heads(what, "q", q)
    _heads(what, "k", k, q)
    b, n, hq, d = q.shape
    if k.shape[:2] != q.shape[:2] or k.shape[3] != d or hq < 1 or k.shape[2] < 1:
        raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, length or head dim")
    if d % 2 or not 2 <= d <= 512:
        raise ValueError(f"{what}: head dim {d} must be even and at most 512")
    if (q_weight is None) != (k_weight is None) or (cos is None) != (sin is None):
        raise ValueError(f"{what}: q_weight and k_weight, cos and sin are given together")
    if q_weight is None and cos is None:
        raise ValueError(f"{what}: neither norm weights nor a rotation table")
    norm = q_weight is not None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if norm and (tuple(w.shape) != (d,) or w.dtype != torch.float32 or w.device != q.device or not w.is_contiguous()):
            raise ValueError(f"{what}: {name} must be contiguous float32 [{d}] on {q.device}")
    if cos is not None:
        if (cos.dim() != 2 or cos.shape != sin.shape or not 1 <= cos.shape[1] <= d // 2 or cos.shape[0] < 1
                or cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != q.device
                or sin.device != q.device):
            raise ValueError(f"{what}: cos and sin must be float32 [rows, up to {d // 2}] on {q.device}")
        if cos.requires_grad or sin.requires_grad:
            raise ValueError(f"{what}: no gradient reaches cos and sin")
        cos, sin = cos.contiguous(), sin.contiguous()
    if positions is not None:
        if cos is None:
            raise ValueError(f"{what}: positions without a rotation table")
        if (tuple(positions.shape) not in ((b, n), (n,)) or positions.dtype not in (torch.int32, torch.int64)
                or positions.device != q.device):
            raise ValueError(f"{what}: positions must be int32 or int64 [{b}, {n}] or [{n}] on {q.device}")
        if n > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
    elif cos is not None and cos.shape[0] < n:
        raise ValueError(f"{what}: the table has {cos.shape[0]} rows for {n} tokens")
    _no_tangents(what, q, k, q_weight, k_weight, cos, sin)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"{what}: eps {eps}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad
                                    or (norm and (q_weight.requires_grad or k_weight.requires_grad))):
        return _QkNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, positions, norm, float(eps), bool(interleaved))
    return _qk_fwd(q, k, cos, sin, positions, q_weight, k_weight, norm, float(eps), bool(interleaved))


# ---------------------------------------------------------------- attention
def _spans(documents, kv_lens, prefix, b, lq, lk, causal):
    spans = torch.empty((b, lq, 2), dtype=torch.int32, device=documents.device)
    name = "dmf_mattn_spans64" if documents.dtype == torch.int64 else "dmf_mattn_spans"
    _launch(name, documents.device, documents.data_ptr(), lk, _p(kv_lens), _p(prefix), b, lq, lk, causal, spans.data_ptr())
    return spans


def _attn_dims(q, k, v, cfg, kv_lens, prefix, slopes, spans):
    """The leading arguments dmf_mattn_fwd and dmf_mattn_bwd share, and the tensors they point into."""
    scale, softcap, causal = cfg
    align = 16 // q.element_size()
    d = q.shape[3]
    (q, qs), (k, ks), (v, vs) = _strided(q, align, d), _strided(k, align, d), _strided(v, align, d)
    args = (_DTYPES[q.dtype], q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs, q.shape[0], q.shape[1],
            k.shape[1], q.shape[2], k.shape[2], d, scale, softcap, _p(slopes), causal, _p(kv_lens),
            None if spans is not None else _p(prefix), _p(spans))
    return args, (q, k, v)


def _attn_fwd(q, k, v, cfg, kv_lens, prefix, slopes, spans, train):
    b, lq, hq, d = q.shape
    args, keep = _attn_dims(q, k, v, cfg, kv_lens, prefix, slopes, spans)
    o = torch.empty((b, lq, hq, d), dtype=q.dtype, device=q.device)
    o_lo = torch.empty_like(o) if train and q.dtype != torch.float32 else None
    lse = torch.empty(b * lq * hq, dtype=torch.float32, device=q.device) if train else None
    n = N.load().dmf_mattn_fwd_ws_floats(_DTYPES[q.dtype], b, lq, k.shape[1], hq, k.shape[2], d, int(kv_lens is not None))
    ws = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    _launch("dmf_mattn_fwd", q.device, *args, o.data_ptr(), _p(o_lo), _p(lse), _p(ws))
    del keep
    return o, o_lo, lse


def _attn_bwd(q, k, v, cfg, kv_lens, prefix, slopes, spans, o, o_lo, lse, go):
    args, keep = _attn_dims(q, k, v, cfg, kv_lens, prefix, slopes, spans)
    go = _plain(go)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    ws = torch.empty(q.shape[0] * q.shape[1] * (q.shape[2] + 2), dtype=torch.float32, device=q.device)
    _launch("dmf_mattn_bwd", q.device, *args, o.data_ptr(), _p(o_lo), lse.data_ptr(), go.data_ptr(), ws.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
    del keep
    return dq, dk, dv


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cfg, kv_lens, prefix, slopes, spans):
        o, o_lo, lse = _attn_fwd(q, k, v, cfg, kv_lens, prefix, slopes, spans, True)
        ctx.save_for_backward(q, k, v, kv_lens, prefix, slopes, spans, o, o_lo, lse)
        ctx.cfg = cfg
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, kv_lens, prefix, slopes, spans, o, o_lo, lse = ctx.saved_tensors
        g = _attn_bwd(q, k, v, ctx.cfg, kv_lens, prefix, slopes, spans, o, o_lo, lse, go)
        return tuple(x if n else None for x, n in zip(g, ctx.needs_input_grad)) + (None,) * 5


def attention(q, k, v, *, scale=None, softcap=0.0, slopes=None, causal=False, kv_lens=None, prefix=None,
              documents=None):
    """softmax(score) v per head, [b, lq, hq, d], of queries [b, lq, hq, d] over keys and values [b, lk, hk, d]
    (any strides; hq a multiple of hk: query head h reads key head h // (hq // hk)). Differentiable in q, k, v.

    score = softcap * tanh(z / softcap) - slopes[h] * |p - j|, z = scale * q.k (scale: d^-0.5; softcap 0 and
    slopes None leave their term out; both numbers lie in 2^-60 .. 2^60; slopes f32 [hq] is not differentiated). Query i stands at position
    p = kv_len - lq + i: the queries are the last lq of the kv_len tokens, so one new token against a cache of
    capacity lk has lq = 1. It sees the keys j < kv_len (``kv_lens`` int [b], clamped to [0, lk]; default lk),
    under ``causal`` those with j <= p and, all queries, the first ``prefix`` (int [b]) keys, and with
    ``documents`` (int [b, lk] ids) those of its own document: the run of equal ids >= 0 it stands in (a
    negative id belongs to none; the prefix then counts from the document's start). For a padded batch give
    the padding a negative id. A query that sees nothing yields zeros and no gradient, and what a key or a value holds
    does not reach the queries that do not see it (but the last bits of a rounding, which the rows of a tile share; under a
    softcap, up to 6e-7 of it in a score). Inputs that are not finite make a masked call up to about ten times as long.

    Arithmetic is in 32 bits; in 16-bit types the probabilities and, in the backward, the score gradients are rounded once
    to the type as operands of the matrix products (the error against 64 bits is 1.1 to 1.3 times that of rounding the
    output alone for o, about 1.4 times for the gradients).
    """
    what = "attention"
    _heads(what, "q", q)
    _heads(what, "k", k, q)
    _heads(what, "v", v, q)
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"{what}: {hq} query heads must be a multiple of {hk} key heads")
    if d % 8 or not 8 <= d <= 128:
        raise ValueError(f"{what}: head dim {d} must be a multiple of 8 up to 128")
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not 2.0 ** -60 <= scale <= 2.0 ** 60 or not (softcap == 0 or 2.0 ** -60 <= softcap <= 2.0 ** 60):
        raise ValueError(f"{what}: scale {scale} must be in 2^-60 .. 2^60 and softcap {softcap} too, or 0")
    if prefix is not None and not causal:
        raise ValueError(f"{what}: a prefix needs causal=True")
    if slopes is not None and slopes.requires_grad:
        raise ValueError(f"{what}: no gradient reaches slopes")
    _no_tangents(what, q, k, v, slopes)
    dev = q.device
    if slopes is not None:
        slopes = _small(what, "slopes", slopes, (hq,), torch.float32, dev)
    if kv_lens is not None:
        kv_lens = _small(what, "kv_lens", kv_lens, (b,), torch.int32, dev)
    if prefix is not None:
        prefix = _small(what, "prefix", prefix, (b,), torch.int32, dev)
    spans = None
    if documents is not None:
        documents = _small(what, "documents", documents, (b, lk),
                           torch.int64 if documents.dtype == torch.int64 else torch.int32, dev)
        spans = _spans(documents, kv_lens, prefix, b, lq, lk, causal)
    cfg = (scale, softcap, bool(causal))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFn.apply(q, k, v, cfg, kv_lens, prefix, slopes, spans)
    return _attn_fwd(q, k, v, cfg, kv_lens, prefix, slopes, spans, False)[0]
