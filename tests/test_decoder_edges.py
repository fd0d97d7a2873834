"""What the decoder layer's Python calls take and refuse by strides.  No GPU."""

from __future__ import annotations

import pytest

from spinnv2_amd import decoder

from .test_decoder import Fake, _cache


def test_attention_refuses_a_workspace_that_is_not_contiguous():
    """Its size is counted in elements: an expanded byte has as many as asked for, and memory for one."""
    c = _cache()
    q, table, lengths, offsets = Fake((3, 4, 64), "float16"), Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((3,), "int32")
    for work in (Fake((1 << 30,), "int8", strides=(0,)), Fake((1 << 30,), "int8", strides=(2,)), Fake((1 << 15, 1 << 15), "int8", strides=(0, 1)),
                 Fake((1 << 15, 1 << 15), "int8", strides=(1, 1 << 15))):
        with pytest.raises(ValueError):
            decoder.attention(q, c, table, lengths, offsets, q, max_queries=2, max_length=4096, workspace=work)
