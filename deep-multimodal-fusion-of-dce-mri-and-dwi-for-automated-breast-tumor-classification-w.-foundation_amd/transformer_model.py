"""Hybrid CNN -> Transformer stage -- MI355X build of the reference's
``code/transformer_model.py`` (used when ``use_hybrid_transformer`` replaces
block3, model_module.py:564-579, :701-703; configuration 5).

Module and parameter names match the reference (PatchEmbed :7-32,
TokensToFeatureMap :34-52, TransformerEncoder :54-66, TransformerBlock
:68-81, MultiHeadSelfAttention :83-116, MLP :118-134, TransformerStage
:137-175). Patch embedding runs on the conv engine; LayerNorm, the linear
layers and attention on the MFMA GEMM + token kernels (dmf_tokens), in the
module's compute dtype (bf16, or f32 for the parity mode).
"""
from __future__ import annotations

import torch
import torch.nn as nn

import dmf_attention as A
import dmf_ops as O
import dmf_tokens as D


def _caches(conv):
    c = getattr(conv, "_dmf_caches", None)
    if c is None:
        c = (O.WeightCache(), O.WeightCache())
        conv._dmf_caches = c
    return c


def _rng_if(x, *drops):
    """The Philox snapshot when any of the nn.Dropout modules draws (their own
    train flags: MC dropout turns on only them) -- the enclosing encoder's
    snapshot if there is one, else a fresh one."""
    if not any(d.training and d.p > 0 for d in drops):
        return None
    cur = O.RNG_CURRENT[0]
    return cur if cur is not None else O.RNG.snapshot(x.device)


class PatchEmbed(nn.Module):
    def __init__(self, in_ch, embed_dim, patch_size=2, dim=2):
        super().__init__()
        assert dim in (2, 3)
        self.dim = dim
        self.norm = nn.LayerNorm(embed_dim)
        self.proj = nn.Conv2d(in_ch, embed_dim, kernel_size=patch_size, stride=patch_size)

    # config 5: the projection on e4m3 MFMA; set by
    # TransformerStage from parameters "patch_embed_fp8" (bf16 compute only)
    use_fp8 = False

    def forward(self, x):
        dt = D.token_dtype(getattr(self, "compute_dtype", torch.bfloat16))
        x = O.as_nhwc(x.to(dt))
        if self.use_fp8 and dt == torch.bfloat16:
            y = D.patch_embed_fp8(x, self.proj, _caches(self.proj))
        else:
            y = O.conv2d(x, self.proj, _caches(self.proj))       # [B, E, h, w] NHWC
        h, w = y.shape[-2:]
        return D.patch_tokens_layernorm(y, self.norm), (h, w)    # NHWC storage == token order


class TokensToFeatureMap(nn.Module):
    def __init__(self, dim=2):
        super().__init__()
        assert dim in (2, 3)
        self.dim = dim

    def forward(self, tokens, spatial_shape):
        b, n, c = tokens.shape
        h, w = spatial_shape
        return tokens.reshape(b, h, w, c).permute(0, 3, 1, 2)   # NCHW logical, NHWC storage


def attention_options(options):
    """The attention options of a TransformerStage, beyond the reference's plain softmax attention, or None:
    ``qk_norm`` (per-head RMS norm of queries and keys, with weights), ``rope`` (rotation by the token grid's
    rows and columns), ``softcap`` (scores capped by a tanh), ``distance_bias`` (falls off linearly with the
    distance in token order, another slope for each head). They have no attention dropout."""
    if not options:
        return None
    known = {"qk_norm": False, "rope": False, "softcap": 0.0, "distance_bias": False}
    extra = sorted(set(options) - set(known))
    if extra:
        raise ValueError(f"attention options: {extra} unknown (known: {sorted(known)})")
    got = {**known, **options}
    got["softcap"] = float(got["softcap"])
    if not (got["softcap"] == 0.0 or 2.0 ** -60 <= got["softcap"] <= 2.0 ** 60):
        raise ValueError(f"attention options: softcap {got['softcap']} must be 0 (none) or in 2^-60 .. 2^60")
    return got if any(got.values()) else None


class MultiHeadSelfAttention(nn.Module):
    def __init__(self, embed_dim, num_heads, qkv_bias=True, attn_drop=0.1, proj_drop=0.1, options=None):
        super().__init__()
        assert embed_dim % num_heads == 0, "embed_dim must be divisible by num_heads"
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        self.scale = self.head_dim ** -0.5
        self.qkv = nn.Linear(embed_dim, embed_dim * 3, bias=qkv_bias)
        self.attn_drop = nn.Dropout(attn_drop)
        self.proj = nn.Linear(embed_dim, embed_dim)
        self.proj_drop = nn.Dropout(proj_drop)
        self._sites = (O.RNG.new_site(), O.RNG.new_site())   # Philox: attn_drop, proj_drop
        self.options = attention_options(options)
        if self.options:
            if self.options["qk_norm"]:
                self.q_norm = nn.Parameter(torch.ones(self.head_dim))
                self.k_norm = nn.Parameter(torch.ones(self.head_dim))
            if self.options["distance_bias"]:
                slopes = [2.0 ** (-8.0 * (h + 1) / num_heads) for h in range(num_heads)]
                self.register_buffer("slopes", torch.tensor(slopes), persistent=False)

    def core(self, rope=None):
        """The options' AttnCore (None without options); ``rope``: the token grid's (cos, sin)."""
        o = self.options
        if not o:
            return None
        if o["rope"] and rope is None:
            raise ValueError("MultiHeadSelfAttention: the rope option needs the token grid's rotation table")
        return D.AttnCore(self.q_norm if o["qk_norm"] else None, self.k_norm if o["qk_norm"] else None,
                          rope if o["rope"] else None, o["softcap"], self.slopes if o["distance_bias"] else None)

    def forward(self, x, rope=None):
        rng = _rng_if(x, self.attn_drop, self.proj_drop)
        return D.multihead_self_attention(x, self, rng, D.token_dtype(getattr(self, "compute_dtype", torch.bfloat16)),
                                          self.core(rope))


class MLP(nn.Module):
    def __init__(self, embed_dim, mlp_ratio=4.0, drop=0.1):
        super().__init__()
        hidden_dim = int(embed_dim * mlp_ratio)
        self.fc1 = nn.Linear(embed_dim, hidden_dim)
        self.act = nn.GELU()
        self.fc2 = nn.Linear(hidden_dim, embed_dim)
        self.drop = nn.Dropout(drop)
        self._sites = (O.RNG.new_site(), O.RNG.new_site())   # Philox: drop after GELU, drop after fc2

    def forward(self, x):
        rng = _rng_if(x, self.drop)
        return D.mlp(x, self, rng, D.token_dtype(getattr(self, "compute_dtype", torch.bfloat16)))


class TransformerBlock(nn.Module):
    def __init__(self, embed_dim, heads, init_scale=0.1, options=None):
        super().__init__()
        self.norm1 = nn.LayerNorm(embed_dim)
        self.attn = (MultiHeadSelfAttention(embed_dim, heads, attn_drop=0.0, options=options)
                     if attention_options(options) else MultiHeadSelfAttention(embed_dim, heads))
        self.norm2 = nn.LayerNorm(embed_dim)
        self.mlp = MLP(embed_dim)
        self.gamma1 = nn.Parameter(init_scale * torch.ones(embed_dim))
        self.gamma2 = nn.Parameter(init_scale * torch.ones(embed_dim))
        # Philox sites: attn_drop, proj_drop, MLP drop after GELU, MLP drop after fc2
        self._sites = self.attn._sites + self.mlp._sites

    def forward(self, x, rope=None):
        rng = _rng_if(x, self.attn.attn_drop, self.attn.proj_drop, self.mlp.drop)
        return D.transformer_block(x.float(), self, rng, self._sites,
                                   D.token_dtype(getattr(self, "compute_dtype", torch.bfloat16)),
                                   core=self.attn.core(rope))


class TransformerEncoder(nn.Module):
    def __init__(self, embed_dim, depth=4, heads=8, options=None):
        super().__init__()
        self.layers = nn.ModuleList([TransformerBlock(embed_dim, heads=heads, options=options) for _ in range(depth)])

    def forward(self, x, rope=None):
        for layer in self.layers:
            x = layer(x, rope)
        return x


class TransformerStage(nn.Module):
    def __init__(self, in_ch, embed_dim, depth=2, heads=8, patch_size=2, dim=2, attention=None):
        super().__init__()
        assert dim in (2, 3)
        self.dim = dim
        self.patch_embed = PatchEmbed(in_ch=in_ch, embed_dim=embed_dim, patch_size=patch_size, dim=dim)
        self.transformer = TransformerEncoder(embed_dim=embed_dim, depth=depth, heads=heads, options=attention)
        self.tokens_to_map = TokensToFeatureMap(dim=dim)
        self.attention = attention_options(attention)
        if self.attention and self.attention["rope"] and (embed_dim // heads) % 4:
            raise ValueError(f"TransformerStage: the rope option needs a head dim ({embed_dim // heads}) of a multiple of 4")
        self._head_dim = embed_dim // heads
        self._rope = {}  # (grid, device) -> rotation table: one per image size

    def rope(self, hw, device):
        """The rotation table of an h x w token grid (None without the rope option)."""
        if not (self.attention and self.attention["rope"]):
            return None
        key = (tuple(hw), str(device))
        if key not in self._rope:
            if torch.cuda.is_current_stream_capturing():  # (a table made in a capture is not filled before a replay)
                raise RuntimeError(f"TransformerStage: run one step on a {hw[0]} x {hw[1]} grid before capturing it")
            with torch.inference_mode(False):  # (a training step saves it for its backward)
                table = A.rope_table_2d(hw[0], hw[1], self._head_dim, device=device)
            if table[0].is_cuda:  # (later steps may run on other streams)
                torch.cuda.current_stream(table[0].device).synchronize()
            self._rope[key] = table
        return self._rope[key]

    def forward(self, x):
        # under "16-mixed" the CNN around the stage runs fp16 and the stage bf16 (D.token_dtype): the map
        # leaves in the dtype it came in
        dt = getattr(self, "compute_dtype", torch.bfloat16)
        tokens, hw = self.patch_embed(x)
        tokens = self.transformer(tokens, self.rope(hw, tokens.device))
        return D.tokens_to_map(tokens, hw[0], hw[1], dt)
