"""What the decoder layer's Python calls take and refuse by strides, and which
kernels the sizes of test_gpu_decoder_edges reach.  No GPU."""

from __future__ import annotations

import ctypes

import pytest

from spinnv2_amd import decoder
from spinnv2_amd.runtime import load_library

from .test_decoder import BF16, FP16, FP32, Fake, _cache

DTYPES = {"float32": FP32, "float16": FP16, "bfloat16": BF16}


def matmul_kernel(m, n, k, dtype, pads=(0, 0, 0)) -> str:
    name = ctypes.create_string_buffer(64)
    a = decoder._Matmul(m=m, n=n, k=k, a_stride=k + pads[0], b_stride=k + pads[1], out_stride=n + pads[2], dtype=DTYPES[dtype])
    assert load_library().spkv2_mi355x_matmul_i8_kernel_name(ctypes.byref(a), name, 64) == 0
    return name.value.decode()


def attention_kernel(counts, heads, kv, dim, dtype, bound) -> str:
    name = ctypes.create_string_buffer(64)
    c = decoder._Cache(k=1 << 20, v=1 << 20, k_scale=1 << 20, v_scale=1 << 20, pages=4, kv_heads=kv, page_size=16, head_dim=dim)
    a = decoder._Attention(queries=sum(counts), max_queries=max(counts), max_length=bound, sequences=len(counts), heads=heads, dtype=DTYPES[dtype])
    assert load_library().spkv2_mi355x_attention_i8_kernel_name(ctypes.byref(c), ctypes.byref(a), name, 64) == 0
    return name.value.decode()


def _products():
    """(kernel, m, n, k, dtype, bias, pads, at): each kernel of the product with k of one step of 128 bytes, two, three, four and
    more, whole pieces of 16 bytes and not, each type, ragged rows and channels, a bias or none, rows side by side or apart."""
    for kernel, sizes in (("matmul_rows<16x16,waves=8>", [(9, 333)] * 6), ("matmul_rows<16x32,waves=8>", [(3, 4100)] * 6),
                          ("matmul_rows<32x32,waves=8>", [(17, 4100)] * 6), ("matmul_rows<32x64,waves=8>", [None, None] + [(65, 3001)] * 4),
                          ("matmul_tiles<64x64>", [(3001, 130)] * 6), ("matmul_tiles<128x128>", [(700, 3001)] * 6),
                          ("matmul_tiles<256x256>", [(3001, 4100)] * 2 + [(2050, 4100)] * 4)):
        for i, (k, size) in enumerate(zip((100, 128, 200, 333, 500, 1040), sizes)):
            if size:
                yield (kernel, *size, k, ("float32", "bfloat16", "float16")[i % 3], i % 2 == 0, [(0, 0, 0), (16, 32, 8), (3, 5, 1)][i // 2], (0, 16, 1)[i // 2])
    for i, (m, n, k) in enumerate([(300, 3001, 7), (300, 3001, 15), (129, 4100, 2048), (129, 4100, 2111), (100, 4100, 3000)]):
        yield "matmul_rows<64x64,waves=4>", m, n, k, ("float32", "bfloat16", "float16")[i % 3], i % 2 == 0, [(0, 0, 0), (3, 5, 1)][i % 2], i % 2


PRODUCTS = list(_products())
#: counts, lengths, max_length, heads, kv_heads, head_dim, type, causal: calls of many rows with several splits that hold tokens
SPLIT = [([130, 120], [700, 400], 8192, 4, 2, dim, dtype, causal)
         for dim, dtype, causal in ((64, "float32", True), (128, "float32", False), (256, "float32", True), (128, "bfloat16", True),
                                    (96, "float16", False), (256, "bfloat16", False), (64, "float16", True))]


def test_sizes_reach_every_kernel_of_the_product():
    for kernel, m, n, k, dtype, bias, pads, at in PRODUCTS:
        assert matmul_kernel(m, n, k, dtype, pads) == kernel, (m, n, k)
    kernels = {p[0] for p in PRODUCTS}
    assert len(kernels) == 8
    for kernel in kernels:
        assert {p[4] for p in PRODUCTS if p[0] == kernel} == set(DTYPES)
    # whatever the sizes, no other kernel is taken
    for m in (1, 2, 15, 40, 100, 300, 1000, 5000, 50000):
        for n in (1, 60, 500, 4000, 30000):
            for k in (0, 1, 16, 100, 1000, 10000, 1 << 17):
                assert matmul_kernel(m, n, k, "bfloat16") in kernels


def test_rows_far_apart_take_no_tiles():
    """Offsets inside a tile are 32 bits."""
    assert "tiles" in matmul_kernel(700, 3001, 200, "bfloat16")
    for pads in ((1 << 23, 0, 0), (0, 1 << 23, 0)):
        assert "rows" in matmul_kernel(700, 3001, 200, "bfloat16", pads)


def test_sizes_reach_splits_of_many_rows():
    for counts, lengths, bound, heads, kv, dim, dtype, causal in SPLIT:
        assert attention_kernel(counts, heads, kv, dim, dtype, bound) == "attend_tiles<splits=32>"  # of 256 tokens


def test_kernel_names_refuse_what_the_calls_refuse():
    lib, name = load_library(), ctypes.create_string_buffer(64)
    assert lib.spkv2_mi355x_matmul_i8_kernel_name(None, name, 64) == -1
    a = decoder._Matmul(m=2, n=8, k=8, a_stride=8, b_stride=8, out_stride=7, dtype=FP16)
    assert lib.spkv2_mi355x_matmul_i8_kernel_name(ctypes.byref(a), name, 64) == -1
    a.out_stride = 8
    assert lib.spkv2_mi355x_matmul_i8_kernel_name(ctypes.byref(a), None, 64) == -1
    assert lib.spkv2_mi355x_matmul_i8_kernel_name(ctypes.byref(a), name, 64) == 0 and name.value
    a.m = 0
    assert lib.spkv2_mi355x_matmul_i8_kernel_name(ctypes.byref(a), name, 64) == 0 and not name.value
    assert lib.spkv2_mi355x_attention_i8_kernel_name(_cache()._ref, None, name, 64) == -1


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
