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
