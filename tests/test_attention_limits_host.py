"""CPU: limits of the token attention's C entry points (status -1 and a message before any launch; the pointers below are
never followed)."""
import pytest

import dmf_native as N
from test_attention_host import PTR


@pytest.mark.parametrize("name", ["dmf_mattn_spans", "dmf_mattn_spans64"])
@pytest.mark.parametrize("lq,lk", [(5, 2 ** 31 - 1), (5, 2 ** 31 - 1024), (2 ** 31 - 1024, 5), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_spans_refuse_lengths_past_their_index(name, lq, lk):
    """Positions are stepped over 1024 at a time: the last step has to stay below 2^31."""
    with pytest.raises(RuntimeError, match="lengths"):
        N.call(name, PTR, lk, None, None, 1, lq, lk, 0, PTR, None)


def test_queries_heads_may_lie_far_apart():
    """A tile holds rows of one head, so the distance of a group's heads is no limit (the call gets as far as its missing
    output); the distance of a tile's tokens is."""
    from test_attention_host import _dims

    far = dict(hq=8, hk=1, q_sh=1 << 28, q_sb=1 << 31)
    with pytest.raises(RuntimeError, match="null"):
        N.call("dmf_mattn_fwd", *_dims(**far), None, None, None, None, None)
    with pytest.raises(RuntimeError, match="null"):
        N.call("dmf_mattn_bwd", *_dims(**far), None, None, PTR, PTR, PTR, PTR, PTR, PTR, None)
    with pytest.raises(RuntimeError, match="2 GiB"):
        N.call("dmf_mattn_fwd", *_dims(q_sl=1 << 28), None, None, None, None, None)


@pytest.mark.parametrize("kw,match", [(dict(cap=1e-25), "softcap"), (dict(cap=1e30), "softcap"), (dict(cap=1e-39), "softcap"),
                                      (dict(scale=1e-30), "scale"), (dict(scale=1e30), "scale")])
def test_scales_and_caps_past_the_range_of_their_constants(kw, match):
    """1 / softcap^2, scale / softcap and a slope over the scale have to be numbers of f32."""
    import transformer_model as TM
    from test_attention_host import _dims

    with pytest.raises(RuntimeError, match=match):
        N.call("dmf_mattn_fwd", *_dims(**kw), None, None, None, None, None)
    with pytest.raises(RuntimeError, match=match):
        N.call("dmf_mattn_bwd", *_dims(**kw), None, None, PTR, PTR, PTR, PTR, PTR, PTR, None)
    if "cap" in kw:
        with pytest.raises(ValueError, match="softcap"):
            TM.attention_options(dict(softcap=kw["cap"]))
