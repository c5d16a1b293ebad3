"""CPU: the argument checks of the token attention's C entry points (status -1 and a message before any launch; the
pointers below are never followed), the rotation tables, and the options of the token blocks."""
import math

import pytest
import torch

import dmf_attention as A
import dmf_native as N
import transformer_model as TM

PTR = 1 << 20   # aligned, never dereferenced


def _qk(**kw):
    a = dict(dtype=N.BF16, q=PTR, q_sb=640, q_sl=64, q_sh=64, hq=2, k=PTR, k_sb=640, k_sl=64, k_sh=64, hk=1, batch=1,
             len=5, d=64, rot=64, inter=0, norm=1, eps=1e-6, wq=PTR, wk=PTR, cos=PTR, sin=PTR, pos=None, pos_sb=0,
             pos64=0, rows=5, qo=PTR, ko=PTR, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=7), "dtype"), (dict(d=63), "head dim"), (dict(d=514), "head dim"), (dict(rot=66), "rotated dims"),
    (dict(rot=31), "rotated dims"), (dict(rows=4), "4 rows for 5 positions"), (dict(cos=None), "tables"),
    (dict(norm=0), "weights without the norm"), (dict(hq=0), "heads"), (dict(q=None), "null"), (dict(batch=-1), "tokens"),
    (dict(batch=1 << 20, len=1 << 12), "tokens"),
])
def test_qk_norm_rope_entry_refuses(kw, match):
    with pytest.raises(RuntimeError, match=match):
        N.call("dmf_qk_norm_rope", *_qk(**kw))


def test_qk_norm_rope_backward_entry_refuses():
    head = _qk()[:-3]
    for tail, match in (((PTR, PTR, PTR, PTR, PTR, None, PTR, None), "weight gradients"),
                        ((PTR, PTR, PTR, PTR, PTR, PTR, None, None), "weight gradients"),
                        ((None, PTR, PTR, PTR, PTR, PTR, PTR, None), "null")):
        with pytest.raises(RuntimeError, match=match):
            N.call("dmf_qk_norm_rope_bwd", *head, *tail)
    assert N.load().dmf_qk_norm_rope_bwd_ws_floats(4, 2, 64) >= 6 * 64


def _dims(**kw):
    a = dict(dtype=N.BF16, q=PTR, q_sb=4096, q_sl=256, q_sh=64, k=PTR, k_sb=4096, k_sl=128, k_sh=64, v=PTR, v_sb=4096,
             v_sl=128, v_sh=64, batch=2, lq=5, lk=7, hq=4, hk=2, d=64, scale=0.125, cap=0.0, slopes=None, causal=1,
             kv_lens=None, prefix=None, spans=None)
    a.update(kw)
    return list(a.values())


BAD = [
    (dict(dtype=3), "dtype"), (dict(hq=3), "multiple of"), (dict(hk=0), "multiple of"), (dict(d=12), "head dim"),
    (dict(d=136), "head dim"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"), (dict(cap=-1.0), "softcap"), (dict(cap=math.nan), "softcap"),
    (dict(causal=0, prefix=PTR), "prefix"), (dict(q_sl=260), "stride"), (dict(k_sb=-128), "stride"),
    (dict(k_sl=32), "token strides"), (dict(q=PTR + 2), "aligned"), (dict(k_sl=1 << 28), "2 GiB"),
    (dict(lq=1 << 30, hq=64, hk=1), "exceed"), (dict(lk=1 << 30), "exceed"), (dict(batch=-1), "multiple of"),
]


@pytest.mark.parametrize("kw,match", BAD)
def test_attention_entries_refuse(kw, match):
    with pytest.raises(RuntimeError, match=match):
        N.call("dmf_mattn_fwd", *_dims(**kw), PTR, None, None, PTR, None)
    with pytest.raises(RuntimeError, match=match):
        N.call("dmf_mattn_bwd", *_dims(**kw), PTR, None, PTR, PTR, PTR, PTR, PTR, PTR, None)


def test_attention_entries_refuse_missing_buffers():
    with pytest.raises(RuntimeError, match="null"):
        N.call("dmf_mattn_fwd", *_dims(), None, None, None, None, None)
    with pytest.raises(RuntimeError, match="o_lo"):
        N.call("dmf_mattn_fwd", *_dims(), PTR, None, PTR, None, None)
    need = N.load().dmf_mattn_fwd_ws_floats(N.BF16, 1, 1, 4096, 4, 2, 64, 0)
    assert need > 0
    with pytest.raises(RuntimeError, match="workspace"):
        N.call("dmf_mattn_fwd", *_dims(batch=1, lq=1, lk=4096, k_sb=1 << 20, v_sb=1 << 20), PTR, None, None, None, None)
    with pytest.raises(RuntimeError, match="null"):
        N.call("dmf_mattn_bwd", *_dims(), PTR, None, PTR, PTR, None, PTR, PTR, PTR, None)
    with pytest.raises(RuntimeError, match="aligned"):
        N.call("dmf_mattn_bwd", *_dims(), PTR, None, PTR, PTR + 4, PTR, PTR, PTR, PTR, None)
    with pytest.raises(RuntimeError, match="null"):
        N.call("dmf_mattn_spans", None, 7, None, None, 1, 5, 7, 0, PTR, None)
    with pytest.raises(RuntimeError, match="batch"):
        N.call("dmf_mattn_spans", PTR, 7, None, None, 1 << 17, 5, 7, 0, PTR, None)


def test_workspace_covers_the_plan_over_many_sizes():
    """Sizes drawn over the whole range: a workspace that holds whole splits of all rows, bounded splits, none where a size
    is 0, and the same answer each time."""
    f = N.load().dmf_mattn_fwd_ws_floats
    g = torch.Generator().manual_seed(0)
    for _ in range(3000):
        r = [int(2 ** (torch.rand(1, generator=g).item() * t)) for t in (7, 14, 18, 4, 4)]
        b, lq, lk, hk, grp = r
        for dt in (N.F32, N.BF16):
            for ragged in (0, 1):
                n = f(dt, b, lq, lk, hk * grp, hk, 64, ragged)
                one = b * lq * hk * grp * 68
                assert n % one == 0 and n // one != 1 and n // one <= max(66, lk // 64 + 1) and n // one <= 8193, (r, n)
                assert n == f(dt, b, lq, lk, hk * grp, hk, 64, ragged)
    assert f(1, 0, 1, 100, 4, 4, 64, 0) == f(1, 1, 0, 100, 4, 4, 64, 0) == f(1, 1, 1, 0, 4, 4, 64, 0) == 0


def test_empty_calls_launch_nothing():
    N.call("dmf_qk_norm_rope", *_qk(batch=0, q=None, k=None, qo=None, ko=None))
    N.call("dmf_mattn_fwd", *_dims(batch=0), None, None, None, None, None)
    N.call("dmf_mattn_fwd", *_dims(lq=0), None, None, None, None, None)
    N.call("dmf_mattn_bwd", *_dims(lq=0, lk=0), None, None, None, None, None, None, None, None, None)
    N.call("dmf_mattn_spans", None, 0, None, None, 0, 0, 0, 0, None, None)


def test_rope_tables():
    c, s = A.rope_table(100001, 8, theta=10000.0)
    assert c.shape == s.shape == (100001, 4) and c.dtype == torch.float32
    for p in range(4):   # a far position keeps its phase (angle in 64 bits)
        a = 100000 * 10000.0 ** (-2 * p / 8)
        assert abs(c[100000, p].item() - math.cos(a)) < 1e-6 and abs(s[100000, p].item() - math.sin(a)) < 1e-6
    c, s = A.rope_table_2d(3, 5, 8)
    assert c.shape == (15, 4)
    for r in range(3):
        for x in range(5):
            want = [math.sin(r), math.sin(r * 0.1), math.sin(x), math.sin(x * 0.1)]
            assert all(abs(s[r * 5 + x, i].item() - want[i]) < 1e-6 for i in range(4))
    for bad in ((0, 8), (5, 7), (5, 0)):
        with pytest.raises(ValueError):
            A.rope_table(*bad)
    with pytest.raises(ValueError):
        A.rope_table_2d(3, 3, 6)


def test_cpu_tensors_are_refused():
    q, k = torch.randn(1, 4, 2, 32), torch.randn(1, 4, 1, 32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.attention(q, k, k)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.qk_norm_rope(q, k, q_weight=torch.ones(32), k_weight=torch.ones(32))
    with pytest.raises(ValueError, match=r"\[batch, length, heads, head_dim\]"):
        A.attention(q[0], k, k)


def test_block_options():
    assert TM.attention_options({}) is None
    got = TM.attention_options(dict(softcap=30))
    assert got == dict(qk_norm=False, rope=False, softcap=30.0, distance_bias=False)
    with pytest.raises(ValueError, match="unknown"):
        TM.attention_options(dict(cap=3))
    st = TM.TransformerStage(8, 256, depth=1, heads=4, attention=dict(rope=True, qk_norm=True))
    assert {k for k in st.state_dict() if "q_norm" in k or "k_norm" in k} == \
        {"transformer.layers.0.attn.q_norm", "transformer.layers.0.attn.k_norm"}
    assert TM.TransformerStage(8, 256, depth=1, heads=4).state_dict().keys() == \
        TM.TransformerStage(8, 256, depth=1, heads=4, attention=dict(rope=True)).state_dict().keys()
    with pytest.raises(ValueError, match="multiple of 4"):
        TM.TransformerStage(8, 12, depth=1, heads=2, attention=dict(rope=True))
