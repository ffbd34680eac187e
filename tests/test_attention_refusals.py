"""Scales and caps of the attention operators at the ends of what 32 bits hold, on the host."""
import pytest

from test_cache_operators import INVALID, P, _batch


def calls(lib, batch, scale, cap):
    more = dict(scale=scale, cap=cap)
    return (lambda: lib.prompt_attention(0, P, 512, batch, 4, P, P, **more), lambda: lib.tree_attention(0, P, 512, batch, 4, P, P, P, **more),
            lambda: lib.window_attention(0, P, 512, batch, 4, P, P, 10, **more), lambda: lib.four_bit_attention(0, P, 512, batch, 4, P, P, **more))


@pytest.mark.parametrize("scale,cap", [(4e26, 2e38), (2e26, 1.2e38), (4e26, 2.3e38)])
def test_caps_whose_double_overflows_are_refused_where_scores_reach_them(lib, scale, cap):
    """A capped score is the cap less twice the cap times what e^2x leaves: in units of log 2 that double is infinite from 1.18e38 on."""
    for call in calls(lib, _batch(), scale, cap):
        with pytest.raises(lib.FlashLLMError, match=f"cudaError_t {INVALID}$"):
            call()


@pytest.mark.parametrize("scale,cap", [(4e26, 1.1e38), (1e26, 2.3e38), (1.0, 2.3e38), (4e26, 0.0), (0.125, 30.0)])
def test_others_are_accepted(lib, scale, cap):
    for call in calls(lib, _batch(tokens=0), scale, cap):
        call()
