"""The decoder layer's operators where ranges end: windows, sizes, scales and
products next to what their types hold, and combinations of masks, splits and
kernels.  References in 64 bits or in whole numbers, as in test_gpu_decoder."""

from __future__ import annotations

import pytest

from .test_gpu_decoder import FAR, _attend_case

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
def test_attention_in_a_window_past_every_token(gpu, window, dtype):
    """The widest windows, with queries that lie before the first token: position + 1 - window is below -2^31."""
    for bound in ({}, {"max_length": FAR}):
        _attend_case([1, 40, 9, 70], [5, 12, 41, 70], 4, 2, 64, 16, dtype, window=window, **bound)
    _attend_case([1, 700], [1, 1], 4, 2, 64, 16, dtype, window=window)
