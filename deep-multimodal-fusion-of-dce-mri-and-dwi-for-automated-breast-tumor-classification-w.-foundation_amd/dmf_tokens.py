"""Token-stream ops of the hybrid TransformerStage (configuration 5) on the
MFMA GEMM (csrc/gemm.hip) and the token kernels (csrc/tokens.hip).

Reference: ``code/transformer_model.py`` -- PatchEmbed :7-32 (conv k=s=patch,
then LayerNorm over tokens), TransformerBlock :68-81 (pre-LN, LayerScale
gamma, residual), MultiHeadSelfAttention :83-116 (qkv Linear, softmax(q k^T *
scale), attn_drop, P v, proj, proj_drop), MLP :118-134 (fc1, GELU, drop,
fc2, drop).

A whole TransformerBlock is ONE autograd node (`_BlockFn`): the forward is 6
GEMM launches + softmax/dropout + 2 LayerNorms with every bias / GELU /
dropout / LayerScale / residual fused into a GEMM epilogue, and the backward
is written out by hand (13 GEMMs, the dropout masks re-drawn from the Philox
snapshot instead of stored). Residual stream: f32 [B*N, E]; accumulation
and weight grads: f32; GEMM operands and saved activations in the compute
dtype -- bf16 (throughput: 16x16x32 bf16 MFMA) or f32 (the parity mode,
``set_compute_dtype(float32)``: 16x16x4 f32 MFMA, f32 probabilities and
pre-activations, so the block matches the fp32 oracle to rounding).
"""
from __future__ import annotations

import torch

import dmf_attention as A
import dmf_native as N
import dmf_ops as O

F32, BF16 = N.F32, N.BF16


def _s():
    return N.stream_ptr()


def gemm(out, a, b, M, Nn, K, ta=0, tb=0, lda=None, ldb=None, ldc=None, batch=(1, 1), sa=(0, 0), sb=(0, 0),
         sc=(0, 0), a_off=0, b_off=0, c_off=0, bias=None, act="none", colscale=None, res=None, aux=None, pre=None,
         dropout_p=0.0, rng=None, site=0, dbias=None, alpha=1.0):
    """out[z] = epilogue(alpha * op(A[z]) op(B[z])) -- see include/dmf_hip.h
    dmf_gemm_bf16 / dmf_gemm_f32 (picked by the operand dtype; aux and pre are
    in the operand dtype). Offsets are in elements of the operand's dtype."""
    N.require_cuda(out, a, b)
    if a.dtype == torch.bfloat16 and b.dtype == torch.bfloat16:
        fn, esz = "dmf_gemm_bf16", 2
    elif a.dtype == torch.float32 and b.dtype == torch.float32:
        fn, esz = "dmf_gemm_f32", 4
    else:
        raise TypeError(f"gemm: operands must both be bf16 or both f32, got {a.dtype} / {b.dtype}")
    for t in (aux, pre):
        if t is not None and t.dtype != a.dtype:
            raise TypeError("gemm: aux / pre must have the operand dtype")
    esz_c = out.element_size()
    args = (F32 if out.dtype == torch.float32 else BF16, int(ta), int(tb), int(M), int(Nn), int(K),
            float(alpha), a.data_ptr() + esz * a_off, int(lda), int(sa[0]), int(sa[1]),
            b.data_ptr() + esz * b_off, int(ldb), int(sb[0]), int(sb[1]),
            out.data_ptr() + esz_c * c_off, int(ldc), int(sc[0]), int(sc[1]), int(batch[0]), int(batch[1]),
            O._p(bias), O.ACT[act], O._p(colscale), O._p(res), int(res.stride(0)) if res is not None else 0,
            O._p(aux), int(aux.stride(0)) if aux is not None else 0,
            O._p(pre), int(pre.stride(0)) if pre is not None else 0,
            float(dropout_p), O._p(rng), int(site), O._p(dbias))
    # dbias: per-128-row-tile column sums, summed in tile order by the launcher (deterministic)
    dbias_ws = torch.empty(((int(M) + 127) // 128) * int(Nn), dtype=torch.float32, device=out.device) \
        if dbias is not None else None
    args = args + (O._p(dbias_ws),)
    N.call(fn, *args, _s())
    probe = O.PROBE["tok_gemm"]
    in_place = res is not None and out.data_ptr() == res.data_ptr()
    if probe is not None and not in_place and dbias is None:
        # (an in-place residual or a dbias accumulation would change state on a replay: not probed; the
        # proj / fc2 residual epilogues write a fresh tensor and replay identically)
        nb = int(batch[0]) * int(batch[1])
        probe.append({"fn": fn, "args": args, "keep": (out, a, b, bias, colscale, aux, pre, rng, res),
                      "flops": 2.0 * M * Nn * K * nb,
                      "bytes": nb * (esz * (M * K + K * Nn) + esz_c * M * Nn
                                     + (res.element_size() * M * Nn if res is not None else 0)),
                      "shape": (fn, M, Nn, K, nb)})
    return out


def cast_bf16(x):
    x = x.contiguous()
    y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    N.call("dmf_cast_bf16", x.data_ptr(), x.numel(), y.data_ptr(), _s())
    return y


def cast_f32(x):
    x = x.contiguous()
    y = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    N.call("dmf_cast_f32", x.data_ptr(), x.numel(), y.data_ptr(), _s())
    return y


def ln_fwd(x2d, gamma, beta, eps, out_dtype):
    r, e = x2d.shape
    y = torch.empty((r, e), dtype=out_dtype, device=x2d.device)
    save = torch.empty(2 * r, dtype=torch.float32, device=x2d.device)
    N.call("dmf_tok_layernorm_fwd", O.dt(x2d), x2d.data_ptr(), x2d.stride(0), r, e, gamma.data_ptr(),
           beta.data_ptr(), float(eps), O.dt(y), y.data_ptr(), e, save.data_ptr(), _s())
    return y, save


def _tok_ws(r, e, dev):
    """Workspace of the token backward's ordered column sums (dmf_tok_bwd_ws_floats)."""
    return torch.empty(N.load().dmf_tok_bwd_ws_floats(r, e), dtype=torch.float32, device=dev)


def ln_bwd(dy, x2d, save, gamma, dres, dgamma, dbeta):
    r, e = x2d.shape
    dx = dres if dres is not None else torch.empty((r, e), dtype=torch.float32, device=dy.device)
    N.call("dmf_tok_layernorm_bwd", dy.data_ptr(), O.dt(x2d), x2d.data_ptr(), x2d.stride(0), save.data_ptr(), r, e,
           gamma.data_ptr(), O._p(dres), dx.data_ptr(), O._p(dgamma), O._p(dbeta), (ws := _tok_ws(r, e, dy.device)).data_ptr(), _s())
    return dx


# ------------------------------------------------------------- patch embed
class _TokLNFn(torch.autograd.Function):
    """LayerNorm over the channels of NHWC-stored conv output viewed as
    tokens [B, h*w, E] (PatchEmbed :26-31: flatten(2).transpose(1,2), norm)."""

    @staticmethod
    def forward(ctx, y, gamma, beta, eps):
        b, e, h, w = y.shape
        x2d = y.permute(0, 2, 3, 1).reshape(b * h * w, e)  # NHWC storage: a view
        out, save = ln_fwd(x2d, gamma, beta, eps, torch.float32)
        ctx.save_for_backward(x2d, save, gamma)
        ctx.shape = (b, e, h, w)
        ctx.ydtype = y.dtype
        return out.view(b, h * w, e)

    @staticmethod
    def backward(ctx, dt):
        x2d, save, gamma = ctx.saved_tensors
        b, e, h, w = ctx.shape
        dgamma = torch.zeros_like(gamma)
        dbeta = torch.zeros_like(gamma)
        dx = ln_bwd(dt.reshape(-1, e).contiguous().float(), x2d, save, gamma, None, dgamma, dbeta)
        if ctx.ydtype == torch.bfloat16:
            dx = cast_bf16(dx)
        dy = dx.view(b, h, w, e).permute(0, 3, 1, 2)  # NCHW logical, NHWC storage
        return dy, dgamma, dbeta, None


class _PatchEmbedFp8Fn(torch.autograd.Function):
    """PatchEmbed.proj (conv k = s = P, transformer_model.py:17-22) forward on
    the e4m3 MFMA GEMM (per-token / per-channel scales, csrc/fp8.hip); the
    backward is the bf16 conv backward of the same conv (straight-through
    through the quantisation)."""

    @staticmethod
    def forward(ctx, x, weight, bias, conv, caches):
        n, c, h, w, ldx = O.nhwc(x)
        p = conv.kernel_size[0]
        e = weight.shape[0]
        ho, wo = h // p, w // p
        m, k = n * ho * wo, p * p * c
        dev = x.device
        q = torch.empty((m, k), dtype=torch.uint8, device=dev)
        rs = torch.empty(m, dtype=torch.float32, device=dev)
        N.call("dmf_patch_quant_fp8", x.data_ptr(), n, h, w, c, ldx, p, q.data_ptr(), k, rs.data_ptr(), _s())
        wq = torch.empty((e, k), dtype=torch.uint8, device=dev)
        cs = torch.empty(e, dtype=torch.float32, device=dev)
        wc = weight.detach().float().contiguous()
        N.call("dmf_weight_quant_fp8", wc.data_ptr(), e, c, p, wq.data_ptr(), cs.data_ptr(), _s())
        y = O.empty_nhwc(n, e, ho, wo, torch.bfloat16, dev)
        args = (m, e, k, q.data_ptr(), k, rs.data_ptr(), wq.data_ptr(), k, cs.data_ptr(), O._p(bias), y.data_ptr(),
                O.nhwc(y)[4])
        N.call("dmf_gemm_fp8", *args, _s())
        probe = O.PROBE["fp8_gemm"]
        if probe is not None:
            probe.append({"fn": "dmf_gemm_fp8", "args": args, "keep": (q, rs, wq, cs, bias, y),
                          "flops": 2.0 * m * e * k, "bytes": m * k + e * k + 2 * m * e, "shape": (m, e, k)})
        ctx.save_for_backward(x, weight, bias)
        ctx.conv, ctx.caches = conv, caches
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = O._conv_backward(x, weight, bias, O.ConvGeom(ctx.conv), ctx.caches, dy, need[0], need[1],
                                      bias is not None and need[2])
        return dx, dw, db, None, None


def patch_embed_fp8(x, conv, caches):
    """NHWC bf16 x -> NHWC bf16 patch-embed conv output via e4m3 MFMA."""
    p = conv.kernel_size[0]
    if (conv.kernel_size[0] != conv.kernel_size[1] or conv.stride[0] != p or conv.stride[1] != p
            or conv.padding[0] != 0 or conv.dilation[0] != 1 or x.dtype != torch.bfloat16):
        raise ValueError("patch_embed_fp8: needs a bf16 input and a conv with kernel == stride, no padding")
    _, c, h, w, _ = O.nhwc(x)
    if c % 8 or h % p or w % p or (p * p * c) % 16:
        raise ValueError(f"patch_embed_fp8: unsupported shape C={c} H={h} W={w} P={p}")
    return _PatchEmbedFp8Fn.apply(x, conv.weight, conv.bias, conv, caches)


def patch_tokens_layernorm(y, ln):
    return _TokLNFn.apply(y, ln.weight, ln.bias, ln.eps)


class _TokensToMapFn(torch.autograd.Function):
    """tokens f32 [B, N, E] -> NCHW-logical, NHWC-stored map in the compute
    dtype (TokensToFeatureMap :34-52: transpose(1,2).reshape)."""

    @staticmethod
    def forward(ctx, t, h, w, dtype):
        b, n, e = t.shape
        if dtype == torch.bfloat16:
            o = cast_bf16(t)
        elif dtype == torch.float16:
            o = t.contiguous().to(torch.float16)
        else:
            o = t.contiguous().clone()
        return o.view(b, h, w, e).permute(0, 3, 1, 2)

    @staticmethod
    def backward(ctx, dm):
        b, e, h, w = dm.shape
        d = dm.permute(0, 2, 3, 1).contiguous()
        d = cast_f32(d) if d.dtype == torch.bfloat16 else d.float()
        return d.view(b, h * w, e), None, None, None


def tokens_to_map(t, h, w, dtype):
    return _TokensToMapFn.apply(t, h, w, dtype)


# ------------------------------------------------------- transformer block
# The two residual branches as forward / backward helpers, shared by the
# fused TransformerBlock node and the standalone MultiHeadSelfAttention / MLP
# modules. Rows r = B*N, width e; `a` is the branch input in the compute
# dtype, the branch output f32:
#   attention: out = res + drop(proj(drop(softmax(q k^T * scale)) v)) * gamma
#   MLP:       out = res + drop(fc2(drop(gelu(fc1(a))))) * gamma
# (res / gamma absent for the standalone modules: out = the branch itself).
def _wcast(cdt, *ws):
    if cdt == torch.bfloat16:
        return tuple(cast_bf16(w) for w in ws)
    return tuple(w.contiguous() for w in ws)


def _sfx(cdt):
    return "" if cdt == torch.bfloat16 else "_f32"


class AttnCore:
    """What a block's attention does between its qkv and output projections beyond softmax(q k^T / sqrt(d)) v
    (dmf_attention): norm weights f32 [d] or None, rotation table (cos, sin) or None, softcap, slopes f32 [heads]
    or None."""

    __slots__ = ("wq", "wk", "cos", "sin", "softcap", "slopes")
    EPS = 1e-6

    def __init__(self, wq=None, wk=None, rope=None, softcap=0.0, slopes=None):
        self.wq, self.wk = wq, wk
        self.cos, self.sin = rope if rope is not None else (None, None)
        self.softcap, self.slopes = float(softcap), slopes

    def tensors(self):
        """What the backward reads again: saved by the nodes, so that a change in place before it raises."""
        return self.wq, self.wk, self.cos, self.sin, self.slopes

    def check(self, what, n, d, heads, dev):
        for name, t, shape in (("q_norm", self.wq, (d,)), ("k_norm", self.wk, (d,)), ("slopes", self.slopes, (heads,)),
                               ("the table's cos", self.cos, None), ("the table's sin", self.sin, None)):
            if t is not None and (t.dtype != torch.float32 or t.device != dev or not t.is_contiguous()
                                  or (t.dim() != 2 if shape is None else tuple(t.shape) != shape)):
                raise ValueError(f"{what}: {name} must be contiguous float32 {shape or '[tokens, pairs]'} on {dev}, got "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        if (self.wq is None) != (self.wk is None) or (self.cos is not None and self.cos.shape != self.sin.shape):
            raise ValueError(f"{what}: q_norm and k_norm, cos and sin belong together")
        if d > 128 or d % 8:
            raise ValueError(f"{what}: attention options need a head dim that is a multiple of 8 up to 128, got {d}")
        if self.cos is not None and (self.cos.shape[0] < n or 2 * self.cos.shape[1] > d):
            raise ValueError(f"{what}: rotation table {tuple(self.cos.shape)} for {n} tokens, head dim {d}")


def _core_heads(qkv, b, n, heads):
    e = qkv.shape[1] // 3
    x = qkv.view(b, n, 3, heads, e // heads)
    return x[:, :, 0], x[:, :, 1], x[:, :, 2]


def _core_fwd(qkv, b, n, heads, core, train):
    """o [b*n, e] from the packed qkv rows, and what the backward reads."""
    q, k, v = _core_heads(qkv, b, n, heads)
    if core.wq is not None or core.cos is not None:
        q, k = A._qk_fwd(q, k, core.cos, core.sin, None, core.wq, core.wk, core.wq is not None, core.EPS, False)
    cfg = (q.shape[3] ** -0.5, core.softcap, False)
    o, o_lo, lse = A._attn_fwd(q, k, v, cfg, None, None, core.slopes, None, train)
    return o.view(b * n, -1), (qkv, q, k, o_lo, lse)


def _core_bwd(do, o, saved, b, n, heads, core):
    """do (packed rows) -> dqkv (packed rows), dwq, dwk."""
    qkv, q, k, o_lo, lse = saved
    q0, k0, v = _core_heads(qkv, b, n, heads)
    cfg = (q.shape[3] ** -0.5, core.softcap, False)
    dq, dk, dv = A._attn_bwd(q, k, v, cfg, None, None, core.slopes, None, o, o_lo, lse, do.view(q.shape))
    dwq = dwk = None
    if core.wq is not None or core.cos is not None:
        dq, dk, dwq, dwk = A._qk_bwd(q0, k0, core.cos, core.sin, None, core.wq, core.wk, core.wq is not None, core.EPS,
                                     False, dq, dk, core.wq is not None)
    return torch.cat([dq, dk, dv], 2).view(b * n, -1), dwq, dwk


def _attn_fwd(a, wq, qkvb, wp, projb, b, n, heads, p_attn, p_proj, rng, s_attn, s_proj, gamma=None, res=None, nv=None,
              core=None):
    r, e = a.shape
    d = e // heads
    cdt, dev = a.dtype, a.device
    bf = dict(dtype=cdt, device=dev)
    f32 = dict(dtype=torch.float32, device=dev)
    qkv = gemm(torch.empty((r, 3 * e), **bf), a, wq, r, 3 * e, e, lda=e, ldb=e, ldc=3 * e, bias=qkvb)
    if core is not None:
        o, saved = _core_fwd(qkv, b, n, heads, core, True)
        y = torch.empty((r, e), **bf)
        out = gemm(torch.empty((r, e), **f32), o, wp, r, e, e, lda=e, ldb=e, ldc=e, bias=projb, colscale=gamma, res=res,
                   aux=y, dropout_p=p_proj, rng=rng, site=s_proj)
        return out, (*saved, o, y)
    S = torch.empty((b, heads, n, n), **f32)
    gemm(S, qkv, qkv, n, n, d, lda=3 * e, ldb=3 * e, ldc=n, batch=(b, heads), sa=(n * 3 * e, d),
         sb=(n * 3 * e, d), sc=(heads * n * n, n * n), b_off=e)
    P = torch.empty((b, heads, n, n), **bf)
    Pd = torch.empty((b, heads, n, n), **bf) if p_attn > 0 else P
    N.call("dmf_softmax_dropout" + _sfx(cdt), S.data_ptr(), n, b * heads * n, n, int(nv or n), float(d ** -0.5),
           float(p_attn), O._p(rng), int(s_attn), P.data_ptr(), Pd.data_ptr(), n, _s())
    del S
    o = gemm(torch.empty((r, e), **bf), Pd, qkv, n, d, n, tb=1, lda=n, ldb=3 * e, ldc=e, batch=(b, heads),
             sa=(heads * n * n, n * n), sb=(n * 3 * e, d), sc=(n * e, d), b_off=2 * e)
    y = torch.empty((r, e), **bf)
    out = gemm(torch.empty((r, e), **f32), o, wp, r, e, e, lda=e, ldb=e, ldc=e, bias=projb, colscale=gamma, res=res,
               aux=y, dropout_p=p_proj, rng=rng, site=s_proj)
    return out, (qkv, P, Pd, o, y)


def _attn_bwd(dout, a, saved, wq, wp, b, n, heads, p_attn, p_proj, rng, s_attn, s_proj, gamma, grads, core=None):
    """dout (f32 [r, e]) -> d a (f32); grads: dqkvw, dqkvb, dprojw, dprojb, dgamma (nullable). With ``core``:
    (d a, dwq, dwk), the norm weights' gradients (None without them)."""
    *inner, o, y = saved
    r, e = a.shape
    d = e // heads
    cdt, dev = a.dtype, a.device
    bf = dict(dtype=cdt, device=dev)
    f32 = dict(dtype=torch.float32, device=dev)
    dqkvw, dqkvb, dprojw, dprojb, dgamma = grads
    dy = torch.empty((r, e), **bf)
    N.call("dmf_tok_scale_dropout_bwd" + _sfx(cdt), dout.data_ptr(), y.data_ptr(), r, e, gamma.data_ptr(),
           float(p_proj), O._p(rng), int(s_proj), dy.data_ptr(), O._p(dgamma), dprojb.data_ptr(), (ws := _tok_ws(r, e, dev)).data_ptr(),
           _s())
    gemm(dprojw, dy, o, e, e, r, ta=1, tb=1, lda=e, ldb=e, ldc=e)
    do = gemm(torch.empty((r, e), **bf), dy, wp, r, e, e, tb=1, lda=e, ldb=e, ldc=e)
    del dy
    if core is not None:
        dqkv, dwq, dwk = _core_bwd(do, o, inner, b, n, heads, core)
        return _qkv_bwd(dqkv, a, wq, dqkvw, dqkvb), dwq, dwk
    qkv, P, Pd = inner
    dPd = torch.empty((b, heads, n, n), **f32)
    gemm(dPd, do, qkv, n, n, d, lda=e, ldb=3 * e, ldc=n, batch=(b, heads), sa=(n * e, d), sb=(n * 3 * e, d),
         sc=(heads * n * n, n * n), b_off=2 * e)
    dqkv = torch.empty((r, 3 * e), **bf)
    # dV = Pd^T dO
    gemm(dqkv, Pd, do, n, d, n, ta=1, tb=1, lda=n, ldb=e, ldc=3 * e, batch=(b, heads), sa=(heads * n * n, n * n),
         sb=(n * e, d), sc=(n * 3 * e, d), c_off=2 * e)
    dS = torch.empty((b, heads, n, n), **bf)
    N.call("dmf_softmax_dropout_bwd" + _sfx(cdt), P.data_ptr(), n, dPd.data_ptr(), n, b * heads * n, n,
           float(d ** -0.5), float(p_attn), O._p(rng), int(s_attn), dS.data_ptr(), n, _s())
    del dPd
    # dQ = dS K, dK = dS^T Q
    gemm(dqkv, dS, qkv, n, d, n, tb=1, lda=n, ldb=3 * e, ldc=3 * e, batch=(b, heads), sa=(heads * n * n, n * n),
         sb=(n * 3 * e, d), sc=(n * 3 * e, d), b_off=e)
    gemm(dqkv, dS, qkv, n, d, n, ta=1, tb=1, lda=n, ldb=3 * e, ldc=3 * e, batch=(b, heads),
         sa=(heads * n * n, n * n), sb=(n * 3 * e, d), sc=(n * 3 * e, d), c_off=e)
    del dS
    return _qkv_bwd(dqkv, a, wq, dqkvw, dqkvb)


def _qkv_bwd(dqkv, a, wq, dqkvw, dqkvb):
    """The qkv linear's backward: weight and bias (nullable) gradients, d a (f32)."""
    r, e = a.shape
    dev = a.device
    gemm(dqkvw, dqkv, a, 3 * e, e, r, ta=1, tb=1, lda=3 * e, ldb=e, ldc=e)
    if dqkvb is not None:
        if a.dtype == torch.bfloat16:
            ws = torch.empty(N.load().dmf_colsum_bf16_ws_floats(r, 3 * e), dtype=torch.float32, device=dev)
            N.call("dmf_colsum_bf16", dqkv.data_ptr(), 3 * e, r, 3 * e, dqkvb.data_ptr(), ws.data_ptr(), _s())
        else:
            N.call("dmf_colsum_f32", dqkv.data_ptr(), 3 * e, r, 3 * e, dqkvb.data_ptr(), 1, _s())
    return gemm(torch.empty((r, e), dtype=torch.float32, device=dev), dqkv, wq, r, e, 3 * e, tb=1, lda=3 * e, ldb=e,
                ldc=e)


def _mlp_fwd(a, w1, b1, w2, b2, p, rng, s1, s2, gamma=None, res=None):
    r, e = a.shape
    hid = w1.shape[0]
    cdt, dev = a.dtype, a.device
    bf = dict(dtype=cdt, device=dev)
    hpre = torch.empty((r, hid), **bf)
    h = gemm(torch.empty((r, hid), **bf), a, w1, r, hid, e, lda=e, ldb=e, ldc=hid, bias=b1, act="gelu", aux=hpre,
             dropout_p=p, rng=rng, site=s1)
    y = torch.empty((r, e), **bf)
    out = gemm(torch.empty((r, e), dtype=torch.float32, device=dev), h, w2, r, e, hid, lda=hid, ldb=hid, ldc=e,
               bias=b2, colscale=gamma, res=res, aux=y, dropout_p=p, rng=rng, site=s2)
    return out, (hpre, h, y)


def _mlp_bwd(dout, a, saved, w1, w2, p, rng, s1, s2, gamma, grads):
    """dout (f32 [r, e]) -> d a (f32); grads: dfc1w, dfc1b, dfc2w, dfc2b, dgamma (nullable)."""
    hpre, h, y = saved
    r, e = a.shape
    hid = w1.shape[0]
    cdt, dev = a.dtype, a.device
    bf = dict(dtype=cdt, device=dev)
    dfc1w, dfc1b, dfc2w, dfc2b, dgamma = grads
    dy = torch.empty((r, e), **bf)
    N.call("dmf_tok_scale_dropout_bwd" + _sfx(cdt), dout.data_ptr(), y.data_ptr(), r, e, gamma.data_ptr(), float(p),
           O._p(rng), int(s2), dy.data_ptr(), O._p(dgamma), dfc2b.data_ptr(), (ws := _tok_ws(r, e, dev)).data_ptr(), _s())
    gemm(dfc2w, dy, h, e, hid, r, ta=1, tb=1, lda=e, ldb=hid, ldc=hid)
    dpre = gemm(torch.empty((r, hid), **bf), dy, w2, r, hid, e, tb=1, lda=e, ldb=hid, ldc=hid, act="gelu",
                pre=hpre, dropout_p=p, rng=rng, site=s1, dbias=dfc1b)
    del dy
    gemm(dfc1w, dpre, a, hid, e, r, ta=1, tb=1, lda=hid, ldb=e, ldc=e)
    return gemm(torch.empty((r, e), dtype=torch.float32, device=dev), dpre, w1, r, e, hid, tb=1, lda=hid, ldb=e,
                ldc=e)


def _zeros(dev, *shapes):
    return [torch.zeros(s, dtype=torch.float32, device=dev) for s in shapes]


class _BlockFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cfg, rng, ln1w, ln1b, qkvw, qkvb, projw, projb, ln2w, ln2b, fc1w, fc1b, fc2w, fc2b, g1, g2,
                core=None, qnw=None, knw=None):
        heads, eps1, eps2, p_attn, p_proj, p_mlp, sites, cdt, nv = cfg
        s_attn, s_proj, s_m1, s_m2 = sites
        b, n, e = x.shape
        x = x.contiguous().view(b * n, e)
        wq, wp, w1, w2 = _wcast(cdt, qkvw, projw, fc1w, fc2w)
        # attention branch: x1 = x + drop(proj(attn(ln1(x)))) * g1
        ln1, save1 = ln_fwd(x, ln1w, ln1b, eps1, cdt)
        x1, sa = _attn_fwd(ln1, wq, qkvb, wp, projb, b, n, heads, p_attn, p_proj, rng, s_attn, s_proj, g1, x, nv, core)
        # MLP branch: x2 = x1 + drop(fc2(drop(gelu(fc1(ln2(x1)))))) * g2
        ln2, save2 = ln_fwd(x1, ln2w, ln2b, eps2, cdt)
        x2, sm = _mlp_fwd(ln2, w1, fc1b, w2, fc2b, p_mlp, rng, s_m1, s_m2, g2, x1)
        # (and what the core reads again: saved, it is checked for changes in place)
        ctx.save_for_backward(x, ln1, save1, *sa, x1, ln2, save2, *sm, wq, wp, w1, w2, ln1w, ln2w, g1, g2, rng,
                              *(core.tensors() if core is not None else ()))
        ctx.cfg, ctx.core, ctx.na = cfg, core, len(sa)
        ctx.dims = (b, n, e)
        return x2.view(b, n, e)

    @staticmethod
    def backward(ctx, dx2):
        t = ctx.saved_tensors
        (x, ln1, save1), sa, t = t[:3], t[3:3 + ctx.na], t[3 + ctx.na:]
        (x1, ln2, save2), sm = t[:3], t[3:6]
        wq, wp, w1, w2, ln1w, ln2w, g1, g2, rng = t[6:15]
        heads, eps1, eps2, p_attn, p_proj, p_mlp, sites, cdt, _ = ctx.cfg
        s_attn, s_proj, s_m1, s_m2 = sites
        b, n, e = ctx.dims
        hid = w1.shape[0]
        dev = x.device
        dln1w, dln1b, dqkvw, dqkvb, dprojw, dprojb = _zeros(dev, e, e, (3 * e, e), 3 * e, (e, e), e)
        dln2w, dln2b, dfc1w, dfc1b, dfc2w, dfc2b, dg1, dg2 = _zeros(dev, e, e, (hid, e), hid, (e, hid), e, e, e)
        dx2 = dx2.contiguous().view(b * n, e).float()
        dln2 = _mlp_bwd(dx2, ln2, sm, w1, w2, p_mlp, rng, s_m1, s_m2, g2, (dfc1w, dfc1b, dfc2w, dfc2b, dg2))
        dx1 = ln_bwd(dln2, x1, save2, ln2w, dx2.clone(), dln2w, dln2b)
        dqnw = dknw = None
        dln1 = _attn_bwd(dx1, ln1, sa, wq, wp, b, n, heads, p_attn, p_proj, rng, s_attn, s_proj, g1,
                         (dqkvw, dqkvb, dprojw, dprojb, dg1), ctx.core)
        if ctx.core is not None:
            dln1, dqnw, dknw = dln1
        dx = ln_bwd(dln1, x, save1, ln1w, dx1, dln1w, dln1b)
        return (dx.view(b, n, e), None, None, dln1w, dln1b, dqkvw, dqkvb, dprojw, dprojb, dln2w, dln2b,
                dfc1w, dfc1b, dfc2w, dfc2b, dg1, dg2, None, dqnw, dknw)


# ------------------------------------------------ forward-only block (no autograd graph)
# A block whose parameters and input need no gradient (frozen encoders, mode A) skips everything a
# backward would read: the pre-activation / branch copies (aux), the undropped probabilities; the
# attention core is one fused launch (dmf_flash_attn_fwd: no [b*h, n, n] scores or probabilities in
# HBM) for head dim 128, and the qkv linear runs on the conv engine's persistent 1x1 form (register
# epilogue; tools/gemm_bench.py: 18432x1536x512 63.6 -> 41.4 us). fc1 follows it when no dropout
# follows the GELU (the conv epilogue has none). Knob "token_fwd_fused" = False keeps the training
# path's kernels.
FWD_FUSED = True
# fc1 under MLP dropout on the conv engine too (dmf_conv2d_fwd_drop; knob "fc1_drop_conv")
FC1_DROP_CONV = True
# proj / fc2 with their LayerScale + dropout + f32 residual epilogue on the conv engine's persistent 1x1 form
# (dmf_conv2d_fwd_tokres) where it takes the shape (>= the launch's tile threshold: inside the two-encoder
# fork at config 5's B = 32); knob "tokres_conv"
TOKRES_CONV = True
_FA_HEAD_DIM = 128


class _Geom1x1:
    stride, padding, dilation, kernel_size = (1, 1), (0, 0), (1, 1), (1, 1)


_G1 = O.ConvGeom(_Geom1x1)


def _linear_conv(x2d, lin, b, n, act="none"):
    """act(x W^T + bias) of [b*n, K] bf16 token rows as a 1x1 conv over the NHWC view (b, K, n, 1): the
    conv engine's forms with their bias + activation epilogue, bf16 out (forward only). Its launches are
    recorded in the token-GEMM probe family."""
    r, k = x2d.shape
    nout = lin.weight.shape[0]
    caches = lin.__dict__.get("_dmf_conv_caches")
    if caches is None:
        caches = lin.__dict__["_dmf_conv_caches"] = (O.WeightCache(), O.WeightCache())
    x4 = x2d.view(b, n, 1, k).permute(0, 3, 1, 2)
    saved = O.PROBE["conv_fwd"]
    O.PROBE["conv_fwd"] = O.PROBE["tok_gemm"]
    try:
        y, _ = O._conv_forward_raw(x4, lin.weight.view(nout, k, 1, 1), lin.bias, _G1, caches, False, act)
    finally:
        O.PROBE["conv_fwd"] = saved
    return y.permute(0, 2, 3, 1).reshape(r, nout)


def _linear_conv_drop(x2d, lin, b, n, p, rng, site):
    """dropout(gelu(x W^T + bias)) on the conv engine's persistent 1x1 form in one launch
    (dmf_conv2d_fwd_drop): the keep masks are the token GEMM's (element row * Nout + col, same site)."""
    r, k = x2d.shape
    nout = lin.weight.shape[0]
    caches = lin.__dict__.get("_dmf_conv_caches")
    if caches is None:
        caches = lin.__dict__["_dmf_conv_caches"] = (O.WeightCache(), O.WeightCache())
    wk = caches[0].get(lin.weight.view(nout, k, 1, 1), x2d.dtype, k, 0)
    y = torch.empty((r, nout), dtype=x2d.dtype, device=x2d.device)
    x4 = x2d.view(b, n, 1, k).permute(0, 3, 1, 2)
    saved = O.PROBE["conv_fwd"]
    O.PROBE["conv_fwd"] = O.PROBE["tok_gemm"]
    try:
        O._conv_launch("dmf_conv2d_fwd_drop",
                       (O.dt(x2d), x2d.data_ptr(), b, n, 1, k, k, wk.data_ptr(), nout, O._p(lin.bias), y.data_ptr(),
                        nout, N.ACT_GELU, float(p), O._p(rng), int(site)),
                       (x2d, wk, y, lin.bias, rng), x4, b, n, 1, k, nout, 1, 1, _G1, n, 1)
    finally:
        O.PROBE["conv_fwd"] = saved
    return y


def _linear_conv_tokres(x2d, lin, b, n, colscale, res, p, rng, site):
    """res + colscale * dropout(x W^T + bias) with an f32 residual stream, f32 out, on the conv engine's
    persistent 1x1 form in one launch (dmf_conv2d_fwd_tokres): a forward-only block's proj / fc2 with the
    token GEMM's epilogue and keep masks (element row * Nout + col, same site)."""
    r, k = x2d.shape
    nout = lin.weight.shape[0]
    caches = lin.__dict__.get("_dmf_conv_caches")
    if caches is None:
        caches = lin.__dict__["_dmf_conv_caches"] = (O.WeightCache(), O.WeightCache())
    wk = caches[0].get(lin.weight.view(nout, k, 1, 1), x2d.dtype, k, 0)
    y = torch.empty((r, nout), dtype=torch.float32, device=x2d.device)
    x4 = x2d.view(b, n, 1, k).permute(0, 3, 1, 2)
    saved = O.PROBE["conv_fwd"]
    O.PROBE["conv_fwd"] = O.PROBE["tok_gemm"]
    try:
        # (y_maps = 4: the f32 residual read and the f32 output, in 2-byte output maps)
        O._conv_launch("dmf_conv2d_fwd_tokres",
                       (O.dt(x2d), x2d.data_ptr(), b, n, 1, k, k, wk.data_ptr(), nout, O._p(lin.bias),
                        O._p(colscale), res.data_ptr(), res.stride(0), float(p), O._p(rng), int(site), y.data_ptr(),
                        nout),
                       (x2d, wk, y, lin.bias, colscale, res, rng), x4, b, n, 1, k, nout, 1, 1, _G1, n, 1, y_maps=4)
    finally:
        O.PROBE["conv_fwd"] = saved
    return y


def _linear_conv_tokres_ok(x2d, lin, n, res):
    r, k = x2d.shape
    return (TOKRES_CONV and _linear_conv_ok(x2d, lin, n) and res.dtype == torch.float32 and res.stride(1) == 1
            and res.shape == (r, lin.weight.shape[0]) and res.data_ptr() % 16 == 0 and res.stride(0) % 4 == 0
            and bool(N.load().dmf_conv2d_fwd_tokres_ok(N.BF16, r // n, n, 1, k, lin.weight.shape[0])))


def _linear_conv_drop_ok(x2d, lin, n):
    r, k = x2d.shape
    return (_linear_conv_ok(x2d, lin, n) and lin.bias is not None
            and bool(N.load().dmf_conv2d_fwd_drop_ok(N.BF16, r // n, n, 1, k, lin.weight.shape[0])))


def _linear_conv_ok(x2d, lin, n):
    r, k = x2d.shape
    return (x2d.dtype == torch.bfloat16 and x2d.is_contiguous() and k % 64 == 0 and lin.weight.shape[0] % 8 == 0
            and r % n == 0 and x2d.data_ptr() % 16 == 0)


def flash_attention(qkv, b, n, nv, e, heads, p_attn, rng, site):
    """o [b*n, e] bf16 = dropout(softmax(q k^T / sqrt(d))) v per head from the packed qkv rows (one launch)."""
    o = torch.empty((b * n, e), dtype=torch.bfloat16, device=qkv.device)
    d = e // heads
    args = (qkv.data_ptr(), qkv.stride(0), b, n, int(nv), e, heads, float(d ** -0.5), float(p_attn), O._p(rng),
            int(site), o.data_ptr(), e)
    N.call("dmf_flash_attn_fwd", *args, _s())
    probe = O.PROBE["tok_gemm"]
    if probe is not None:
        probe.append({"fn": "dmf_flash_attn_fwd", "args": args, "keep": (qkv, o, rng),
                      "flops": 2.0 * 2.0 * b * heads * n * n * d,
                      "bytes": 2.0 * (b * n * 3 * e + b * n * e), "shape": ("flash", b, n, e, heads)})
    return o


def _block_fwd_nograd(x, blk, rng, cfg, g1, g2, core=None):
    heads, eps1, eps2, p_attn, p_proj, p_mlp, sites, cdt, nv = cfg
    s_attn, s_proj, s_m1, s_m2 = sites
    at, ml = blk.attn, blk.mlp
    b, n, e = x.shape
    d = e // heads
    bf = dict(dtype=cdt, device=x.device)
    f32 = dict(dtype=torch.float32, device=x.device)
    x2d = x.contiguous().view(b * n, e)
    wp, w2 = _wcast(cdt, at.proj.weight, ml.fc2.weight)
    r = b * n
    # attention branch: x1 = x + drop(proj(attn(ln1(x)))) * g1
    ln1, _ = ln_fwd(x2d, blk.norm1.weight, blk.norm1.bias, eps1, cdt)
    if _linear_conv_ok(ln1, at.qkv, n):
        qkv = _linear_conv(ln1, at.qkv, b, n)
    else:
        (wq,) = _wcast(cdt, at.qkv.weight)
        qkv = gemm(torch.empty((r, 3 * e), **bf), ln1, wq, r, 3 * e, e, lda=e, ldb=e, ldc=3 * e, bias=at.qkv.bias)
    if core is not None:
        o, _ = _core_fwd(qkv, b, n, heads, core, False)
    elif d == _FA_HEAD_DIM and cdt == torch.bfloat16:
        o = flash_attention(qkv, b, n, nv or n, e, heads, p_attn, rng, s_attn)
    else:
        S = torch.empty((b, heads, n, n), **f32)
        gemm(S, qkv, qkv, n, n, d, lda=3 * e, ldb=3 * e, ldc=n, batch=(b, heads), sa=(n * 3 * e, d),
             sb=(n * 3 * e, d), sc=(heads * n * n, n * n), b_off=e)
        P = torch.empty((b, heads, n, n), **bf)
        N.call("dmf_softmax_dropout" + _sfx(cdt), S.data_ptr(), n, b * heads * n, n, int(nv or n),
               float(d ** -0.5), float(p_attn), O._p(rng), int(s_attn), P.data_ptr(), P.data_ptr(), n, _s())
        del S
        o = gemm(torch.empty((r, e), **bf), P, qkv, n, d, n, tb=1, lda=n, ldb=3 * e, ldc=e, batch=(b, heads),
                 sa=(heads * n * n, n * n), sb=(n * 3 * e, d), sc=(n * e, d), b_off=2 * e)
    del qkv
    if _linear_conv_tokres_ok(o, at.proj, n, x2d):
        x1 = _linear_conv_tokres(o, at.proj, b, n, g1, x2d, p_proj, rng, s_proj)
    else:
        x1 = gemm(torch.empty((r, e), **f32), o, wp, r, e, e, lda=e, ldb=e, ldc=e, bias=at.proj.bias, colscale=g1,
                  res=x2d, dropout_p=p_proj, rng=rng, site=s_proj)
    del o
    # MLP branch: x2 = x1 + drop(fc2(drop(gelu(fc1(ln2(x1)))))) * g2
    ln2, _ = ln_fwd(x1, blk.norm2.weight, blk.norm2.bias, eps2, cdt)
    hid = ml.fc1.weight.shape[0]
    if p_mlp == 0.0 and _linear_conv_ok(ln2, ml.fc1, n):
        h = _linear_conv(ln2, ml.fc1, b, n, act="gelu")
    elif p_mlp > 0.0 and rng is not None and FC1_DROP_CONV and _linear_conv_drop_ok(ln2, ml.fc1, n):
        h = _linear_conv_drop(ln2, ml.fc1, b, n, p_mlp, rng, s_m1)
    else:
        (w1,) = _wcast(cdt, ml.fc1.weight)
        h = gemm(torch.empty((r, hid), **bf), ln2, w1, r, hid, e, lda=e, ldb=e, ldc=hid, bias=ml.fc1.bias,
                 act="gelu", dropout_p=p_mlp, rng=rng, site=s_m1)
    if _linear_conv_tokres_ok(h, ml.fc2, n, x1):
        x2 = _linear_conv_tokres(h, ml.fc2, b, n, g2, x1, p_mlp, rng, s_m2)
    else:
        x2 = gemm(torch.empty((r, e), **f32), h, w2, r, e, hid, lda=hid, ldb=hid, ldc=e, bias=ml.fc2.bias,
                  colscale=g2, res=x1, dropout_p=p_mlp, rng=rng, site=s_m2)
    return x2.view(b, n, e)


def _branch_input(x, cdt):
    b, n, e = x.shape
    x2d = x.reshape(b * n, e)
    if cdt == torch.bfloat16:
        return cast_bf16(x2d.float()) if x2d.dtype != torch.bfloat16 else x2d.contiguous()
    return x2d.float().contiguous()


class _MHSAFn(torch.autograd.Function):
    """Standalone MultiHeadSelfAttention.forward (transformer_model.py:100-116)."""

    @staticmethod
    def forward(ctx, x, cfg, rng, qkvw, qkvb, projw, projb, core=None, qnw=None, knw=None):
        heads, p_attn, p_proj, sites, cdt = cfg
        b, n, e = x.shape
        a = _branch_input(x, cdt)
        wq, wp = _wcast(cdt, qkvw, projw)
        out, sa = _attn_fwd(a, wq, qkvb, wp, projb, b, n, heads, p_attn, p_proj, rng, sites[0], sites[1], core=core)
        ones = torch.ones(e, dtype=torch.float32, device=x.device)
        ctx.save_for_backward(a, *sa, wq, wp, ones, rng, *(core.tensors() if core is not None else ()))
        ctx.cfg, ctx.dims, ctx.xdtype, ctx.core, ctx.na = cfg, (b, n, e), x.dtype, core, len(sa)
        return out.view(b, n, e)

    @staticmethod
    def backward(ctx, dout):
        a, *rest = ctx.saved_tensors
        sa, (wq, wp, ones, rng) = rest[:ctx.na], rest[ctx.na:ctx.na + 4]
        heads, p_attn, p_proj, sites, cdt = ctx.cfg
        b, n, e = ctx.dims
        need = ctx.needs_input_grad
        dqkvw, dqkvb, dprojw, dprojb = _zeros(a.device, (3 * e, e), 3 * e, (e, e), e)
        da = _attn_bwd(dout.contiguous().view(b * n, e).float(), a, sa, wq, wp, b, n, heads, p_attn, p_proj, rng,
                       sites[0], sites[1], ones, (dqkvw, dqkvb if need[4] else None, dprojw, dprojb, None), ctx.core)
        dqnw = dknw = None
        if ctx.core is not None:
            da, dqnw, dknw = da
        return (da.view(b, n, e).to(ctx.xdtype), None, None, dqkvw, dqkvb if need[4] else None, dprojw, dprojb, None,
                dqnw, dknw)


class _MLPFn(torch.autograd.Function):
    """Standalone MLP.forward (transformer_model.py:128-134)."""

    @staticmethod
    def forward(ctx, x, cfg, rng, fc1w, fc1b, fc2w, fc2b):
        p, sites, cdt = cfg
        b, n, e = x.shape
        a = _branch_input(x, cdt)
        w1, w2 = _wcast(cdt, fc1w, fc2w)
        out, sm = _mlp_fwd(a, w1, fc1b, w2, fc2b, p, rng, sites[0], sites[1])
        ones = torch.ones(e, dtype=torch.float32, device=x.device)
        ctx.save_for_backward(a, *sm, w1, w2, ones, rng)
        ctx.cfg, ctx.dims, ctx.xdtype = cfg, (b, n, e), x.dtype
        return out.view(b, n, e)

    @staticmethod
    def backward(ctx, dout):
        a, hpre, h, y, w1, w2, ones, rng = ctx.saved_tensors
        p, sites, cdt = ctx.cfg
        b, n, e = ctx.dims
        hid = w1.shape[0]
        dfc1w, dfc1b, dfc2w, dfc2b = _zeros(a.device, (hid, e), hid, (e, hid), e)
        da = _mlp_bwd(dout.contiguous().view(b * n, e).float(), a, (hpre, h, y), w1, w2, p, rng, sites[0], sites[1],
                      ones, (dfc1w, dfc1b, dfc2w, dfc2b, None))
        return da.view(b, n, e).to(ctx.xdtype), None, None, dfc1w, dfc1b, dfc2w, dfc2b


def _check_tokens(what, x, e, head_dim=8):
    if e % 256 or e > 1024 or head_dim % 8:
        raise ValueError(f"{what}: embed_dim {e} must be a multiple of 256 (<= 1024), head_dim % 8 == 0")
    if x.dim() != 3 or x.shape[-1] != e:
        raise ValueError(f"{what}: expected tokens [B, N, {e}], got {tuple(x.shape)}")
    if x.shape[1] % 8:
        raise ValueError(f"{what}: token count {x.shape[1]} must be a multiple of 8")


def token_dtype(dt):
    """The token kernels' arithmetic type for a model compute dtype: the GEMM / attention / LayerNorm token
    kernels run bf16 or f32, so under the reference's "16-mixed" (fp16 CNN encoders) the token stages run
    bf16 -- the other 16-bit mixed-precision type, fp32 accumulation either way -- and cast at their
    boundaries (TransformerStage / the ViT backbone under "16-mixed")."""
    return torch.bfloat16 if dt == torch.float16 else dt


def _check_dtype(what, dtype):
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what}: compute dtype must be bf16 or f32, got {dtype}")


def _need_rng(what, rng, *ps):
    if rng is None and any(p > 0 for p in ps):
        raise RuntimeError(f"{what}: dropout requested without an rng snapshot")


def _check_core(what, core, x, heads, p_attn):
    core.check(what, x.shape[1], x.shape[2] // heads, heads, x.device)
    if p_attn > 0:
        raise ValueError(f"{what}: attention options have no attention dropout (p = {p_attn})")


def multihead_self_attention(x, at, rng, dtype=torch.bfloat16, core=None):
    """MultiHeadSelfAttention.forward (transformer_model.py:100-116) as one node; ``core``: AttnCore options."""
    p_attn = float(at.attn_drop.p) if at.attn_drop.training else 0.0
    p_proj = float(at.proj_drop.p) if at.proj_drop.training else 0.0
    _need_rng("MultiHeadSelfAttention", rng, p_attn, p_proj)
    _check_tokens("MultiHeadSelfAttention", x, at.embed_dim, at.head_dim)
    _check_dtype("MultiHeadSelfAttention", dtype)
    if at.qkv.bias is None:
        raise ValueError("MultiHeadSelfAttention: qkv_bias=False is not supported by the fused path")
    cfg = (at.num_heads, p_attn, p_proj, tuple(at._sites), dtype)
    if core is not None:
        _check_core("MultiHeadSelfAttention", core, x, at.num_heads, p_attn)
        return _MHSAFn.apply(x, cfg, rng, at.qkv.weight, at.qkv.bias, at.proj.weight, at.proj.bias, core, core.wq,
                             core.wk)
    return _MHSAFn.apply(x, cfg, rng, at.qkv.weight, at.qkv.bias, at.proj.weight, at.proj.bias)


def mlp(x, m, rng, dtype=torch.bfloat16):
    """MLP.forward (transformer_model.py:128-134) as one node."""
    p = float(m.drop.p) if m.drop.training else 0.0
    _need_rng("MLP", rng, p)
    _check_tokens("MLP", x, m.fc1.in_features)
    _check_dtype("MLP", dtype)
    return _MLPFn.apply(x, (p, tuple(m._sites), dtype), rng, m.fc1.weight, m.fc1.bias, m.fc2.weight, m.fc2.bias)


def transformer_block(x, blk, rng, sites, dtype=torch.bfloat16, n_valid=None, gammas=None, core=None):
    """TransformerBlock.forward (transformer_model.py:78-81) as one node;
    ``dtype`` is the compute dtype (bf16, or f32 for the parity mode).
    ``n_valid``: tokens beyond it are key padding (masked out of every
    softmax row); ``gammas``: LayerScale vectors for a block without them
    (ones: timm's ViT Block, init_values=None). ``core``: AttnCore options."""
    at, ml = blk.attn, blk.mlp
    # the nn.Dropout modules' own flags (train() / eval() set them with the
    # block's; MC dropout turns on only these, train_fusion.py:445-449)
    p_attn = float(at.attn_drop.p) if at.attn_drop.training else 0.0
    p_proj = float(at.proj_drop.p) if at.proj_drop.training else 0.0
    p_mlp = float(ml.drop.p) if ml.drop.training else 0.0
    _need_rng("TransformerBlock", rng, p_attn, p_proj, p_mlp)
    _check_tokens("TransformerBlock", x, at.embed_dim, at.head_dim)
    _check_dtype("TransformerBlock", dtype)
    if at.qkv.bias is None:
        raise ValueError("TransformerBlock: qkv_bias=False is not supported by the fused path")
    cfg = (at.num_heads, blk.norm1.eps, blk.norm2.eps, p_attn, p_proj, p_mlp, tuple(sites), dtype, n_valid)
    g1 = blk.gamma1 if gammas is None else gammas[0]
    g2 = blk.gamma2 if gammas is None else gammas[1]
    if core is not None:
        _check_core("TransformerBlock", core, x, at.num_heads, p_attn)
        if n_valid is not None and n_valid != x.shape[1]:
            raise ValueError("TransformerBlock: attention options have no key padding (n_valid)")
    if FWD_FUSED and dtype == torch.bfloat16 and not O.needs_grad(x, *blk.parameters(), g1, g2):
        with torch.no_grad():
            return _block_fwd_nograd(x, blk, rng, cfg, g1, g2, core)
    return _BlockFn.apply(x, cfg, rng, blk.norm1.weight, blk.norm1.bias, at.qkv.weight, at.qkv.bias, at.proj.weight,
                          at.proj.bias, blk.norm2.weight, blk.norm2.bias, ml.fc1.weight, ml.fc1.bias,
                          ml.fc2.weight, ml.fc2.bias, g1, g2, *((core, core.wq, core.wk) if core is not None else ()))
