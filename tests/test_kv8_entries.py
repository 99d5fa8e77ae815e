"""What the 8-bit cache's C entries refuse without a GPU, beyond shapes, types and pointers."""
import math

import pytest


@pytest.mark.parametrize("scale", [0.0, -0.125, math.nan, math.inf, -math.inf, 3.0e38])
@pytest.mark.parametrize("window", [False, True])
def test_prompt_attention_refuses_factors_it_cannot_mask_with(scale, window):
    """The kernel takes the maximum of the scores before their factor, and -inf times 0 is NaN."""
    from acorninfer_amd import _lib
    p = 64                                              # a pointer that is never followed
    meta = None if window else p
    assert _lib.lib().acorn_paged_prefill_attention_kv8(
        p, p, p, p, p, meta, p, meta, p, 1, 1, 1, 2, 2, 64, 16, 4, 1, scale, 2, None, 0,
        None) == _lib.ERR_VALUE
