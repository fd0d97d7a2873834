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


def test_cache_takes_any_stride_of_an_axis_of_one():
    """One head, or one page, made by moving axes: contiguous, whatever the stride that the axis carries."""
    pages, page, dim = 4, 16, 64
    codes, scales = Fake((pages, 1, page, dim), "int8", strides=(page * dim, dim, dim, 1)), Fake((pages, 1, page), "float32", strides=(page, 1, 1))
    decoder.KvCache(codes, codes, scales, scales)
    codes, scales = Fake((1, 2, page, dim), "int8", strides=(7, page * dim, dim, 1)), Fake((1, 2, page), "float32", strides=(0, page, 1))
    decoder.KvCache(codes, codes, scales, scales)
    for strides in ((2 * page * dim, page * dim, dim, 1), (page * dim, page * dim, dim, 2), (0, page * dim, dim, 1)):
        bad = Fake((pages, 1, page, dim), "int8", strides=strides)
        with pytest.raises(ValueError):
            decoder.KvCache(bad, bad, Fake((pages, 1, page), "float32"), Fake((pages, 1, page), "float32"))


def test_arrays_outside_their_buffer_are_refused():
    class Buffer:
        nbytes = 1024

    for kw in (dict(at=-1), dict(at=250), dict(strides=(-8, 1)), dict(strides=(8, -1)), dict(at=64, strides=(-8, 1)), dict(strides=(300, 1))):
        with pytest.raises(ValueError):
            decoder.DeviceArray((4, 8), "float32", buffer=Buffer(), **kw)
    decoder.DeviceArray((4, 8), "float32", buffer=Buffer(), at=224)
    decoder.DeviceArray((4, 8), "float32", buffer=Buffer(), strides=(0, 1))
