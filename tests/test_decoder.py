"""Refusals of the decoder layer's operators: arguments that the Python calls
and the C entry points turn down before anything is launched.  No GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from spinnv2_amd import decoder
from spinnv2_amd.runtime import load_library

FP32, INT8, FP16, BF16 = 1, 2, 3, 4
UNSUPPORTED = -32
PTR = 1 << 20  # never read: every call here ends before a launch


class Fake:
    """A tensor's shape, strides and type at an address that is never read."""

    def __init__(self, shape, dtype, strides=None, is_cuda=True):
        self.shape, self.dtype, self.is_cuda = tuple(shape), dtype, is_cuda
        self._strides = strides or tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))
        self.itemsize = 2 if dtype == "bfloat16" else np.dtype(dtype if dtype != "float64" else "float64").itemsize

    def stride(self):
        return self._strides

    def data_ptr(self):
        return PTR


def _cache(pages=4, heads=2, page=16, dim=64):
    shape = (pages, heads, page, dim)
    return decoder.KvCache(Fake(shape, "int8"), Fake(shape, "int8"), Fake(shape[:3], "float32"), Fake(shape[:3], "float32"))


# ------------------------------------------------------------ Python checks

def test_norm_refuses_what_does_not_fit():
    x, w, q, s = Fake((4, 32), "bfloat16"), Fake((32,), "bfloat16"), Fake((4, 32), "int8"), Fake((4,), "float32")
    for args, kw in (((Fake((4, 32), "int8"), w, q, s), {}),
                     ((Fake((4, 32, 1), "bfloat16"), w, q, s), {}),
                     ((x, Fake((31,), "bfloat16"), q, s), {}),
                     ((x, Fake((32,), "float16"), q, s), {}),
                     ((x, w, Fake((4, 31), "int8"), s), {}),
                     ((x, w, Fake((4, 32), "float32"), s), {}),
                     ((x, w, q, Fake((5,), "float32")), {}),
                     ((x, w, q, Fake((4,), "float16")), {}),
                     ((x, w, q, Fake((4,), "float32", strides=(2,))), {}),
                     ((Fake((4, 32), "bfloat16", strides=(64, 2)), w, q, s), {}),
                     ((Fake((4, 32), "bfloat16", is_cuda=False), w, q, s), {}),
                     ((x, w, q, s), {"residual": Fake((4, 32), "float32")}),
                     ((x, w, q, s), {"residual_out": Fake((4, 33), "bfloat16")})):
        with pytest.raises(ValueError):
            decoder.rmsnorm_i8(*args, **kw)


def test_matmul_refuses_what_does_not_fit():
    a, b, o = Fake((4, 32), "int8"), Fake((8, 32), "int8"), Fake((4, 8), "float16")
    sa, sb = Fake((4,), "float32"), Fake((8,), "float32")
    for args, kw in (((Fake((4, 31), "int8"), sa, b, sb, o), {}),
                     ((Fake((4, 32), "float16"), sa, b, sb, o), {}),
                     ((a, sb, b, sb, o), {}),
                     ((a, sa, b, sa, o), {}),
                     ((a, sa, b, sb, Fake((8, 4), "float16")), {}),
                     ((a, sa, b, sb, Fake((4, 8), "int8")), {}),
                     ((a, sa, b, sb, Fake((4, 8), "float16", strides=(1, 4))), {}),
                     ((a, sa, b, sb, o), {"bias": Fake((4,), "float32")})):
        with pytest.raises(ValueError):
            decoder.matmul_i8(*args, **kw)


def test_cache_refuses_what_does_not_fit():
    shape = (4, 2, 16, 64)
    k, s = Fake(shape, "int8"), Fake(shape[:3], "float32")
    for args in ((Fake(shape[:3], "int8"), k, s, s), (k, Fake((4, 2, 16, 32), "int8"), s, s), (k, k, Fake(shape[:2], "float32"), s),
                 (k, k, s, Fake(shape[:3], "float16")), (Fake(shape, "int8", strides=(2048, 64, 128, 1)), k, s, s),
                 (Fake(shape, "int8", is_cuda=False), k, s, s)):
        with pytest.raises(ValueError):
            decoder.KvCache(*args)
    c = _cache()
    x, slots = Fake((3, 2, 64), "float16"), Fake((3,), "int64")
    for args in ((Fake((3, 4, 64), "float16"), x, slots), (x, Fake((3, 2, 64), "float32"), slots), (x, x, Fake((3,), "int32")),
                 (x, x, Fake((4,), "int64")), (Fake((3, 2, 64), "float16", strides=(256, 128, 1)), x, slots)):
        with pytest.raises(ValueError):
            c.write(*args)
    table, first, offsets = Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((3,), "int32")
    for args in ((Fake((2, 4), "int64"), first, offsets, x, x), (table, Fake((3,), "int32"), offsets, x, x),
                 (table, first, Fake((2,), "int32"), x, x), (table, first, offsets, x, Fake((3, 2, 64), "bfloat16")),
                 (Fake((2, 4), "int32", strides=(8, 1)), first, offsets, x, x)):
        with pytest.raises(ValueError):
            c.read(*args)


def test_attention_refuses_what_does_not_fit():
    c = _cache()
    q, table, lengths, offsets = Fake((3, 4, 64), "float16"), Fake((2, 4), "int32"), Fake((2,), "int32"), Fake((3,), "int32")
    kw = dict(max_queries=2, max_length=64)
    for args, more in (((Fake((3, 4, 32), "float16"), c, table, lengths, offsets, q), {}),
                       ((q, c, table, Fake((3,), "int32"), offsets, q), {}),
                       ((q, c, table, lengths, Fake((2,), "int32"), q), {}),
                       ((q, c, table, lengths, offsets, Fake((3, 4, 64), "float32")), {}),
                       ((q, c, table, lengths, offsets, Fake((3, 2, 64), "float16")), {}),
                       ((q, c, Fake((2, 4), "int64"), lengths, offsets, q), {}),
                       ((q, c, table, lengths, offsets, q), {"workspace": Fake((64,), "float32")}),
                       ((q, c, table, lengths, offsets, q), {"workspace": Fake((64,), "int8", is_cuda=False)})):
        with pytest.raises(ValueError):
            decoder.attention(*args, **kw, **more)


# ---------------------------------------------------------- C entry points

def _refused(name, rc, code):
    assert rc == code, (name, rc)
    assert load_library().spkv2_mi355x_last_error()


def _norm(**kw):
    a = dict(x=PTR, weight=PTR, q=PTR, scale=PTR, rows=2, cols=8, x_stride=8, q_stride=8, residual_stride=8, residual_out_stride=8,
             dtype=FP32, weight_dtype=FP32, norm=1, eps=1e-6)
    a.update(kw)
    return load_library().spkv2_mi355x_rmsnorm_i8(ctypes.byref(decoder._RmsNorm(**a)), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(dtype=FP16, weight_dtype=BF16), -1), (dict(rows=-1), -1), (dict(cols=0), -1), (dict(x=None), -1),
    (dict(q=None), -1), (dict(scale=None), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(x_stride=7), -1),
    (dict(q_stride=7), -1), (dict(residual=PTR, residual_stride=7), -1), (dict(residual_out=PTR, residual_out_stride=0), -1),
    (dict(rows=1, cols=(1 << 24) + 1), UNSUPPORTED), (dict(rows=1 << 31), UNSUPPORTED)])
def test_norm_entry_refuses(kw, code):
    _refused("norm", _norm(**kw), code)


def test_entries_refuse_no_arguments():
    lib = load_library()
    for f in (lib.spkv2_mi355x_rmsnorm_i8, lib.spkv2_mi355x_dequantize_i8, lib.spkv2_mi355x_matmul_i8):
        _refused("none", f(None, None), -1)
    c = _cache()
    for f in (lib.spkv2_mi355x_kv_write_i8, lib.spkv2_mi355x_kv_read_i8, lib.spkv2_mi355x_attention_i8):
        _refused("none", f(c._ref, None, None), -1)
        _refused("none", f(None, None, None), -1)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(rows=-1), -1), (dict(q=None), -1), (dict(out=None), -1), (dict(scale=None), -1),
    (dict(q_stride=7), -1), (dict(out_stride=7), -1), (dict(rows=1 << 31), UNSUPPORTED)])
def test_dequantize_entry_refuses(kw, code):
    a = dict(q=PTR, scale=PTR, out=PTR, rows=2, cols=8, q_stride=8, out_stride=8, dtype=FP32)
    a.update(kw)
    _refused("dequantize", load_library().spkv2_mi355x_dequantize_i8(ctypes.byref(decoder._Dequantize(**a)), None), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(m=-1), -1), (dict(k=-1), -1), (dict(a=None), -1), (dict(b=None), -1), (dict(a_scale=None), -1),
    (dict(b_scale=None), -1), (dict(out=None), -1), (dict(a_stride=7), -1), (dict(b_stride=7), -1), (dict(out_stride=7), -1),
    (dict(k=(1 << 17) + 1, a_stride=1 << 18, b_stride=1 << 18), UNSUPPORTED), (dict(m=(1 << 22) + 1), UNSUPPORTED),
    (dict(n=(1 << 30) + 1, out_stride=1 << 31), UNSUPPORTED)])
def test_matmul_entry_refuses(kw, code):
    a = dict(a=PTR, b=PTR, a_scale=PTR, b_scale=PTR, out=PTR, m=2, n=8, k=8, a_stride=8, b_stride=8, out_stride=8, dtype=FP16)
    a.update(kw)
    _refused("matmul", load_library().spkv2_mi355x_matmul_i8(ctypes.byref(decoder._Matmul(**a)), None), code)


def _attention(cache=None, **kw):
    c = dict(k=PTR, v=PTR, k_scale=PTR, v_scale=PTR, pages=4, kv_heads=2, page_size=16, head_dim=64)
    c.update(cache or {})
    a = dict(q=PTR, out=PTR, table=PTR, lengths=PTR, offsets=PTR, queries=3, q_stride=256, out_stride=256, max_queries=2, max_length=64,
             sequences=2, table_width=4, heads=4, dtype=FP16, causal=1, window=0, scale=0.125)
    a.update(kw)
    return load_library().spkv2_mi355x_attention_i8(ctypes.byref(decoder._Cache(**c)), ctypes.byref(decoder._Attention(**a)), None)


@pytest.mark.parametrize("cache,code", [
    (dict(k=None), -1), (dict(v_scale=None), -1), (dict(k=PTR + 8), -1), (dict(v=PTR + 1), -1), (dict(k_scale=PTR + 4), -1),
    (dict(pages=0), -1), (dict(kv_heads=0), -1), (dict(page_size=0), -1), (dict(head_dim=-16), -1), (dict(page_size=24), UNSUPPORTED),
    (dict(head_dim=72), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED), (dict(kv_heads=65536), UNSUPPORTED),
    (dict(pages=1 << 31), UNSUPPORTED)])
def test_cache_is_refused_by_every_entry(cache, code):
    lib = load_library()
    c = dict(k=PTR, v=PTR, k_scale=PTR, v_scale=PTR, pages=4, kv_heads=2, page_size=16, head_dim=64)
    c.update(cache)
    c = decoder._Cache(**c)
    for f, a in ((lib.spkv2_mi355x_kv_write_i8, decoder._Write()), (lib.spkv2_mi355x_kv_read_i8, decoder._Read()),
                 (lib.spkv2_mi355x_attention_i8, decoder._Attention())):
        _refused(str(cache), f(ctypes.byref(c), ctypes.byref(a), None), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(queries=-1), -1), (dict(max_length=-1), -1), (dict(heads=3), -1), (dict(heads=0), -1),
    (dict(window=-1), -1), (dict(window=4, causal=0), -1), (dict(q=None), -1), (dict(out=None), -1), (dict(table=None), -1),
    (dict(lengths=None), -1), (dict(offsets=None), -1), (dict(q_stride=255), -1), (dict(out_stride=128), -1),
    (dict(max_length=4096), -1),  # split, without a workspace
    (dict(max_length=4096, workspace=PTR, workspace_size=64), -1), (dict(max_length=4096, workspace=PTR + 8, workspace_size=1 << 30), -1),
    (dict(heads=65538), UNSUPPORTED), (dict(sequences=65536), UNSUPPORTED), (dict(max_length=(1 << 30) + 1), UNSUPPORTED),
    (dict(queries=(1 << 24) + 1), UNSUPPORTED),
    (dict(queries=1 << 24, max_queries=1 << 40, sequences=65535), UNSUPPORTED),
    (dict(queries=1 << 24, max_queries=1 << 24, heads=256, q_stride=1 << 20, out_stride=1 << 20), UNSUPPORTED)])
def test_attention_entry_refuses(kw, code):
    _refused("attention", _attention(**kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(tokens=-1), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1),
    (dict(k_stride=127), -1), (dict(v_stride=0), -1), (dict(tokens=1 << 31), UNSUPPORTED)])
def test_write_entry_refuses(kw, code):
    a = dict(k=PTR, v=PTR, slots=PTR, tokens=3, k_stride=128, v_stride=128, dtype=FP16)
    a.update(kw)
    _refused("write", load_library().spkv2_mi355x_kv_write_i8(_cache()._ref, ctypes.byref(decoder._Write(**a)), None), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(tokens=-1), -1), (dict(sequences=-1), -1), (dict(table=None), -1), (dict(offsets=None), -1),
    (dict(k_stride=127), -1), (dict(v_stride=0), -1), (dict(tokens=1 << 31), UNSUPPORTED)])
def test_read_entry_refuses(kw, code):
    a = dict(table=PTR, offsets=PTR, k=PTR, v=PTR, tokens=3, k_stride=128, v_stride=128, sequences=2, table_width=4, dtype=FP16)
    a.update(kw)
    _refused("read", load_library().spkv2_mi355x_kv_read_i8(_cache()._ref, ctypes.byref(decoder._Read(**a)), None), code)


def test_nothing_to_do_is_no_error():
    lib = load_library()
    assert _norm(rows=0) == 0
    assert _attention(queries=0) == 0 and _attention(sequences=0) == 0 and _attention(max_queries=0) == 0
    assert lib.spkv2_mi355x_matmul_i8(ctypes.byref(decoder._Matmul(m=0, n=8, k=8, dtype=FP16)), None) == 0
    assert lib.spkv2_mi355x_dequantize_i8(ctypes.byref(decoder._Dequantize(rows=0, cols=8, dtype=FP16)), None) == 0
    c = _cache()
    assert lib.spkv2_mi355x_kv_write_i8(c._ref, ctypes.byref(decoder._Write(dtype=FP16)), None) == 0
    assert lib.spkv2_mi355x_kv_read_i8(c._ref, ctypes.byref(decoder._Read(dtype=FP16)), None) == 0


@pytest.mark.parametrize("sequences,queries,max_queries,max_length", [(1, 1, 1, 1), (1, 1, 1, 100000), (64, 64, 1, 16384), (3, 900, 700, 5000)])
def test_workspace_grows_with_what_is_split(sequences, queries, max_queries, max_length):
    """Rows of partial sums: as many bytes as whole splits of every row take, none where nothing is split."""
    c = _cache()
    size = decoder.attention_workspace(sequences, queries, 4, c, max_queries=max_queries, max_length=max_length)
    row = queries * 4 * (64 + 2) * 4
    assert size % row == 0 and size // row != 1
    if max_length == 1:
        assert size == 0


def test_bfloat16_rounding():
    values = np.array([0.0, 1.0, 1.00390625, 1.01171875, -3.1415926, 3.3e38, np.inf, np.nan], np.float32)
    got = (decoder.to_bfloat16(values).astype(np.uint32) << 16).view(np.float32)
    # 1 + 2^-8 and 1 + 3 2^-8 are ties: to the even one
    want = np.array([0.0, 1.0, 1.0, 1.015625, -3.140625, 3.2963e38, np.inf, np.nan], np.float32)
    np.testing.assert_allclose(got, want, rtol=1e-3)
    np.testing.assert_array_equal(got[:5], want[:5])
