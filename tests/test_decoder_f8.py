"""Refusals of the decoder layer's positions, 8-bit floats and experts: arguments
that the Python calls and the C entry points turn down before anything is
launched.  No GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from spinnv2_amd import decoder
from spinnv2_amd.runtime import load_library

from .test_decoder import BF16, FP16, FP32, INT8, PTR, UNSUPPORTED, _cache, _refused
from .test_decoder import Fake as _Fake


class Fake(_Fake):
    def __init__(self, shape, dtype, strides=None, is_cuda=True):
        super().__init__(shape, "int8" if dtype == "float8_e4m3fn" else dtype, strides, is_cuda)
        self.dtype = dtype


F8 = "float8_e4m3fn"


def _raises(f, args, cases):
    for at, value in cases:
        a, kw = list(args[0]), dict(args[1])
        if isinstance(at, int):
            a[at] = value
        else:
            kw[at] = value
        with pytest.raises(ValueError):
            f(*a, **kw)


# ------------------------------------------------------------ Python checks

def test_rotate_refuses_what_does_not_fit():
    q, k, v = Fake((3, 4, 64), "bfloat16"), Fake((3, 2, 64), "bfloat16"), Fake((3, 2, 64), "bfloat16")
    p, f, slots = Fake((3, 2), "int32"), Fake((32,), "float32"), Fake((3,), "int64")
    args = (q, k, p, f, q, k), dict(axes=Fake((32,), "int32"), norm=True, q_weight=Fake((64,), "bfloat16"), k_weight=Fake((64,), "bfloat16"),
                                    cache=_cache(), v=v, slots=slots)
    _raises(decoder.rotate, args, [
        (0, Fake((3, 4, 64), "int8")), (0, Fake((3, 256), "bfloat16")), (1, Fake((4, 2, 64), "bfloat16")), (1, Fake((3, 2, 64), "float16")),
        (1, Fake((3, 2, 32), "bfloat16")), (1, Fake((3, 1, 64), "bfloat16")), (2, Fake((3, 2), "int64")), (2, Fake((4, 2), "int32")),
        (2, Fake((3, 2), "int32", strides=(1, 3))), (2, Fake((4,), "int32")), (2, Fake((3, 2, 1), "int32")), (3, Fake((32,), "float16")),
        (3, Fake((32, 1), "float32")), (3, Fake((32,), "float32", strides=(2,))), (4, Fake((3, 4, 64), "float32")), (4, None),
        (5, Fake((3, 2, 64), "float32")), (5, Fake((3, 2, 64), "bfloat16", strides=(256, 128, 1))), ("axes", Fake((31,), "int32")),
        ("axes", Fake((32,), "int64")), ("q_weight", Fake((64,), "float16")), ("q_weight", Fake((32,), "bfloat16")),
        ("q_weight", Fake((64,), "float32")),  # of another type than the keys'
        ("v", None), ("slots", None), ("slots", Fake((3,), "int32")), ("v", Fake((3, 2, 64), "float16")), ("cache", _cache(heads=4)),
        ("cache", _cache(dim=32)), ("q_weight", Fake((64,), "bfloat16", is_cuda=False))])
    with pytest.raises(ValueError):
        decoder.rotate(None, None, p, f, None, None)
    with pytest.raises(ValueError):
        decoder.rotate(q, k, p, f, q, None)  # keys that go nowhere


def test_rows_f8_refuse_what_does_not_fit():
    x, w, q, s = Fake((4, 300), "bfloat16"), Fake((300,), "bfloat16"), Fake((4, 300), F8), Fake((4, 3), "float32")
    _raises(decoder.rmsnorm_f8, ((x, w, q, s), {}), [
        (0, Fake((4, 300), "int8")), (0, Fake((4, 301), "bfloat16")), (1, Fake((299,), "bfloat16")), (1, Fake((300,), "float16")),
        (2, Fake((4, 300), "int8")), (2, Fake((4, 300, 1), F8)), (3, Fake((4,), "float32")), (3, Fake((4, 2), "float32")),
        (3, Fake((4, 3), "float16")), (3, Fake((4, 3), "float32", strides=(1, 4))), ("residual", Fake((4, 300), "float32")),
        ("residual_out", Fake((4, 301), "bfloat16"))])
    _raises(decoder.gate_f8, ((Fake((4, 600), "bfloat16"), q, s), {}), [(0, x), (0, Fake((4, 600), "int8")), (1, Fake((4, 600), F8)),
                                                                       (2, Fake((4, 5), "float32"))])
    _raises(decoder.quantize_f8, ((x, q, s), {}), [(0, Fake((4, 600), "bfloat16")), (2, Fake((3, 3), "float32"))])
    _raises(decoder.dequantize_f8, ((q, s, x), {}), [(0, Fake((4, 300), "int8")), (1, Fake((4,), "float32")), (2, Fake((4, 300), "int8")),
                                                    (2, Fake((4, 299), "float32"))])


def test_products_refuse_what_does_not_fit():
    a, sa, b, sb, o = Fake((4, 300), F8), Fake((4, 3), "float32"), Fake((200, 300), F8), Fake((2, 3), "float32"), Fake((4, 200), "float16")
    _raises(decoder.matmul_f8, ((a, sa, b, sb, o), {}), [
        (0, Fake((4, 299), F8)), (0, Fake((4, 300), "int8")), (1, Fake((4,), "float32")), (1, Fake((4, 3), "float16")),
        (2, Fake((200, 300), "int8")), (3, Fake((200, 3), "float32")), (3, Fake((2, 2), "float32")), (4, Fake((4, 201), "float16")),
        (4, Fake((4, 200), "int8")), (4, Fake((4, 200), "float16", strides=(1, 4))), ("bias", Fake((4,), "float32"))])
    b, sb, off, order = Fake((5, 200, 300), F8), Fake((5, 2, 3), "float32"), Fake((6,), "int32"), Fake((8,), "int32")
    o = Fake((8, 200), "float16")
    _raises(decoder.matmul_f8_experts, ((a, sa, b, sb, off, o), dict(order=order, per_token=2)), [
        (0, Fake((4, 299), F8)), (1, Fake((8, 3), "float32")), (2, Fake((200, 300), F8)), (2, Fake((5, 200, 300), "int8")),
        (3, Fake((5, 2, 2), "float32")), (3, Fake((4, 2, 3), "float32")), (4, Fake((5,), "int32")), (4, Fake((6,), "int64")),
        (5, Fake((8, 100), "float16")), (5, Fake((8, 200), "int8")), ("order", Fake((4,), "int32")), ("order", Fake((8,), "int64")),
        ("bias", Fake((200,), "float32")), (2, Fake((5, 200, 300), F8, strides=(60000, 1, 200)))])


def test_experts_order_refuses_what_does_not_fit():
    ids, off, order, place = Fake((4, 2), "int32"), Fake((6,), "int32"), Fake((8,), "int32"), Fake((4, 2), "int32")
    _raises(decoder.sort_tokens, ((ids, off, order, place), {}), [
        (0, Fake((4, 2), "float32")), (0, Fake((8,), "int32")), (0, Fake((4, 2), "int32", strides=(4, 1))), (1, Fake((6,), "int64")),
        (1, Fake((6, 1), "int32")), (2, Fake((7,), "int32")), (3, Fake((4, 3), "int32")), (3, Fake((4, 2), "int64"))])
    y, w, out = Fake((8, 64), "bfloat16"), Fake((4, 2), "float32"), Fake((4, 64), "bfloat16")
    _raises(decoder.combine, ((y, place, w, out), {}), [
        (0, Fake((8, 64), "int8")), (0, Fake((8,), "bfloat16")), (1, Fake((4, 2), "int64")), (2, Fake((4, 2), "bfloat16")),
        (2, Fake((4, 3), "float32")), (3, Fake((4, 64), "float32")), (3, Fake((5, 64), "bfloat16")), ("residual", Fake((4, 63), "bfloat16")),
        ("residual", Fake((4, 64), "float32"))])


# ---------------------------------------------------------- C entry points

def test_entries_refuse_no_arguments():
    lib = load_library()
    for f in (lib.spkv2_mi355x_rows_f8, lib.spkv2_mi355x_dequantize_f8, lib.spkv2_mi355x_matmul_f8, lib.spkv2_mi355x_matmul_f8_experts,
              lib.spkv2_mi355x_sort_tokens, lib.spkv2_mi355x_combine):
        _refused("none", f(None, None), -1)
    _refused("none", lib.spkv2_mi355x_rotate(None, None, None), -1)
    for f in (lib.spkv2_mi355x_matmul_f8_kernel_name, lib.spkv2_mi355x_matmul_f8_experts_kernel_name):
        _refused("none", f(None, ctypes.create_string_buffer(8), 8), -1)
        _refused("none", f(None, None, 0), -1)


def _rotate(cache=None, **kw):
    a = dict(q=PTR, q_out=PTR, k=PTR, k_out=PTR, positions=PTR, frequencies=PTR, tokens=3, q_stride=256, q_out_stride=256, k_stride=128,
             k_out_stride=128, v_stride=128, position_stride=1, heads=4, kv_heads=2, head_dim=64, pairs=32, axes=1, dtype=FP16, weight_dtype=FP16)
    a.update(kw)
    return load_library().spkv2_mi355x_rotate(cache and cache._ref, ctypes.byref(decoder._Rotate(**a)), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(tokens=-1), -1), (dict(heads=-1), -1), (dict(kv_heads=-1), -1), (dict(pairs=-1), -1), (dict(head_dim=-16), -1),
    (dict(axes=0), -1), (dict(pairs=33), -1), (dict(norm=1, eps=-1.0), -1), (dict(norm=1, eps=float("nan")), -1),
    (dict(norm=1, q_weight=PTR, weight_dtype=BF16), -1), (dict(head_dim=72, pairs=1), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED),
    (dict(q=None), -1), (dict(q_out=None), -1), (dict(k=None), -1), (dict(k_out=None), -1), (dict(positions=None), -1),
    (dict(frequencies=None), -1), (dict(q_stride=255), -1), (dict(q_out_stride=0), -1), (dict(k_stride=127), -1), (dict(k_out_stride=64), -1),
    (dict(axes=2), -1), (dict(tokens=1 << 31), UNSUPPORTED), (dict(heads=65536, q_stride=1 << 30, q_out_stride=1 << 30), UNSUPPORTED),
    (dict(tokens=1 << 28), UNSUPPORTED)])
def test_rotate_entry_refuses(kw, code):
    _refused("rotate", _rotate(**kw), code)


def test_rotate_entry_refuses_caches():
    for cache, kw in ((_cache(heads=4), {}), (_cache(dim=32), {}), (_cache(), dict(v=None)), (_cache(), dict(slots=None)), (_cache(), dict(v_stride=127))):
        _refused("rotate", _rotate(cache, **{**dict(v=PTR, slots=PTR), **kw}), -1)


def _rows(**kw):
    a = dict(x=PTR, q=PTR, scale=PTR, rows=2, cols=300, x_stride=600, q_stride=300, scale_stride=3, residual_stride=300, residual_out_stride=300,
             kind=1, dtype=FP16, weight_dtype=FP16, eps=1e-6)
    a.update(kw)
    return load_library().spkv2_mi355x_rows_f8(ctypes.byref(decoder._RowsF8(**a)), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(kind=3), -1), (dict(kind=-1), -1), (dict(kind=0, weight=PTR), -1), (dict(kind=2, residual=PTR), -1),
    (dict(kind=0, residual_out=PTR), -1), (dict(weight=PTR, weight_dtype=BF16), -1), (dict(rows=-1), -1), (dict(cols=0), -1), (dict(cols=-1), -1),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(x=None), -1), (dict(q=None), -1), (dict(scale=None), -1), (dict(x_stride=299), -1),
    (dict(kind=2, x_stride=599), -1), (dict(q_stride=299), -1), (dict(scale_stride=2), -1), (dict(residual=PTR, residual_stride=299), -1),
    (dict(residual_out=PTR, residual_out_stride=299), -1), (dict(rows=1, cols=(1 << 24) + 1), UNSUPPORTED), (dict(rows=1 << 31), UNSUPPORTED),
    (dict(kind=0, rows=1 << 27), UNSUPPORTED)])
def test_rows_entry_refuses(kw, code):
    _refused("rows", _rows(**kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(rows=-1), -1), (dict(q=None), -1), (dict(out=None), -1), (dict(scale=None), -1), (dict(q_stride=299), -1),
    (dict(out_stride=299), -1), (dict(scale_stride=2), -1), (dict(rows=1 << 31), UNSUPPORTED), (dict(rows=1, cols=(1 << 24) + 1), UNSUPPORTED)])
def test_dequantize_entry_refuses(kw, code):
    a = dict(q=PTR, scale=PTR, out=PTR, rows=2, cols=300, q_stride=300, scale_stride=3, out_stride=300, dtype=FP32)
    a.update(kw)
    _refused("dequantize", load_library().spkv2_mi355x_dequantize_f8(ctypes.byref(decoder._DequantizeF8(**a)), None), code)


_PRODUCT = dict(a=PTR, b=PTR, a_scale=PTR, b_scale=PTR, out=PTR, m=2, n=200, k=300, a_stride=300, b_stride=300, out_stride=200, a_scale_stride=3,
                b_scale_stride=3, dtype=FP16)
_PRODUCTS = [
    (dict(dtype=INT8), -1), (dict(m=-1), -1), (dict(n=-1), -1), (dict(k=-1), -1), (dict(a=None), -1), (dict(b=None), -1), (dict(a_scale=None), -1),
    (dict(b_scale=None), -1), (dict(out=None), -1), (dict(a_stride=299), -1), (dict(b_stride=299), -1), (dict(out_stride=199), -1),
    (dict(a_scale_stride=2), -1), (dict(b_scale_stride=2), -1), (dict(m=1 << 21), UNSUPPORTED), (dict(n=1 << 27, out_stride=1 << 27), UNSUPPORTED),
    (dict(k=1 << 25, a_stride=1 << 25, b_stride=1 << 25, a_scale_stride=1 << 18, b_scale_stride=1 << 18), UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", _PRODUCTS)
def test_matmul_entry_refuses(kw, code):
    a = decoder._MatmulF8(**{**_PRODUCT, **kw})
    _refused("matmul", load_library().spkv2_mi355x_matmul_f8(ctypes.byref(a), None), code)


@pytest.mark.parametrize("kw,code", _PRODUCTS + [
    (dict(offsets=None), -1), (dict(experts=0), -1), (dict(experts=4097), UNSUPPORTED), (dict(per_token=0), -1), (dict(a_rows=-1), -1),
    (dict(a_rows=0), -1), (dict(b_expert_stride=59999), -1), (dict(b_scale_expert_stride=5), -1)])
def test_experts_entry_refuses(kw, code):
    a = dict(_PRODUCT, offsets=PTR, a_rows=4, b_expert_stride=60000, b_scale_expert_stride=6, experts=5, per_token=1)
    if "k" in kw:
        kw = dict(kw, b_expert_stride=1 << 40, b_scale_expert_stride=1 << 40)
    if "n" in kw:
        kw = dict(kw, b_expert_stride=1 << 40, b_scale_expert_stride=1 << 40)
    a.update(kw)
    _refused("experts", load_library().spkv2_mi355x_matmul_f8_experts(ctypes.byref(decoder._MatmulF8Experts(**a)), None), code)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), -1), (dict(per_token=-1), -1), (dict(experts=0), -1), (dict(experts=4097), UNSUPPORTED), (dict(tokens=1 << 30), UNSUPPORTED),
    (dict(ids=None), -1), (dict(offsets=None), -1), (dict(order=None), -1), (dict(place=None), -1), (dict(tokens=0, offsets=None), -1)])
def test_sort_entry_refuses(kw, code):
    a = dict(ids=PTR, offsets=PTR, order=PTR, place=PTR, tokens=4, per_token=2, experts=5)
    a.update(kw)
    _refused("sort", load_library().spkv2_mi355x_sort_tokens(ctypes.byref(decoder._SortTokens(**a)), None), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=INT8), -1), (dict(rows=-1), -1), (dict(tokens=-1), -1), (dict(cols=-1), -1), (dict(per_token=0), -1), (dict(y=None), -1),
    (dict(place=None), -1), (dict(weights=None), -1), (dict(out=None), -1), (dict(y_stride=63), -1), (dict(out_stride=63), -1),
    (dict(residual=PTR, residual_stride=63), -1), (dict(tokens=1 << 31), UNSUPPORTED)])
def test_combine_entry_refuses(kw, code):
    a = dict(y=PTR, place=PTR, weights=PTR, out=PTR, rows=8, tokens=4, cols=64, y_stride=64, out_stride=64, per_token=2, dtype=BF16)
    a.update(kw)
    _refused("combine", load_library().spkv2_mi355x_combine(ctypes.byref(decoder._Combine(**a)), None), code)


def test_nothing_to_do_is_no_error():
    lib = load_library()
    assert _rotate(tokens=0) == 0 and _rotate(heads=0, kv_heads=0) == 0 and _rows(rows=0) == 0
    for kw in (dict(m=0), dict(n=0)):
        assert lib.spkv2_mi355x_matmul_f8(ctypes.byref(decoder._MatmulF8(**{**_PRODUCT, **kw})), None) == 0
        a = dict(_PRODUCT, offsets=PTR, a_rows=4, b_expert_stride=60000, b_scale_expert_stride=6, experts=5, per_token=1, **kw)
        assert lib.spkv2_mi355x_matmul_f8_experts(ctypes.byref(decoder._MatmulF8Experts(**{**a, **kw})), None) == 0
    assert lib.spkv2_mi355x_dequantize_f8(ctypes.byref(decoder._DequantizeF8(rows=0, cols=8, dtype=FP16)), None) == 0
    assert lib.spkv2_mi355x_combine(ctypes.byref(decoder._Combine(tokens=0, cols=8, per_token=1, dtype=FP32)), None) == 0


def test_structs_are_the_headers_own(tmp_path):
    """Sizes and the last fields' offsets of the argument structs as a C compiler lays them out."""
    import subprocess
    from pathlib import Path

    kinds = [("Spkv2Rotate", decoder._Rotate), ("Spkv2RowsF8", decoder._RowsF8), ("Spkv2DequantizeF8", decoder._DequantizeF8),
             ("Spkv2MatmulF8", decoder._MatmulF8), ("Spkv2MatmulF8Experts", decoder._MatmulF8Experts), ("Spkv2SortTokens", decoder._SortTokens),
             ("Spkv2Combine", decoder._Combine)]
    source, program = tmp_path / "sizes.c", tmp_path / "sizes"
    lines = [f'printf("%zu %zu\\n", sizeof({c}), offsetof({c}, {py._fields_[-1][0]}));' for c, py in kinds]
    source.write_text('#include <stdio.h>\n#include "spkv2_decoder.h"\nint main(void) {' + "".join(lines) + "return 0;}\n")
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", f"-I{include}", str(source), "-o", str(program)], check=True)
    out = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()
    for (c, py), line in zip(kinds, out):
        assert line == f"{ctypes.sizeof(py)} {getattr(py, py._fields_[-1][0]).offset}", c


def test_float8_rounding():
    table = decoder._FLOAT8
    assert table[:8].tolist() == [i * 2.0 ** -9 for i in range(8)] and table[8] == 2.0 ** -6 and table[126] == 448 and np.isnan(table[[127, 255]]).all()
    np.testing.assert_array_equal(decoder.to_float8(table[:127]), np.arange(127))
    np.testing.assert_array_equal(decoder.to_float8(table[128:255]), np.arange(128, 255))
    half = (table[1:127].astype(np.float64) + table[:126]) / 2
    np.testing.assert_array_equal(decoder.to_float8(half), (np.arange(126) + 1) // 2 * 2)  # ties to the even code
    np.testing.assert_array_equal(decoder.to_float8(half * (1 - 1e-9)), np.arange(126))
    np.testing.assert_array_equal(decoder.to_float8(-half * (1 + 1e-9)), np.arange(1, 127) | 128)
    assert decoder.to_float8([np.inf, np.nan, 500, 464, -0.0]).tolist() == [127, 127, 127, 126, 128]


# ------------------------------------------------------- which kernel a call takes

FORMS = ["rows<16x16>", "rows<16x32>", "rows<16x64>", "rows<32x64>"] + [
    f"tiles<{tile},{how}>" for tile in ("64x64,groups=1", "64x64,groups=2", "64x64,groups=4", "32x128,groups=1", "128x128,groups=1", "128x256,groups=1", "256x256,groups=1")
    for how in ("direct", "staged")]
TYPES = {"float32": FP32, "float16": FP16, "bfloat16": BF16}


def kernel_of(dtype, m, n, k, experts=0, a_rows=0, pad=0):
    """The kernel that a product of contiguous rows (rows `pad` elements apart) takes."""
    name = ctypes.create_string_buffer(64)
    blocks = -(-k // 128)
    a = dict(m=m, n=n, k=k, a_stride=k + pad, b_stride=k + pad, out_stride=n, a_scale_stride=blocks, b_scale_stride=blocks, dtype=TYPES[dtype])
    lib = load_library()
    if experts:
        a.update(a_rows=a_rows, b_expert_stride=n * (k + pad), b_scale_expert_stride=-(-n // 128) * blocks, experts=experts, per_token=1)
        rc = lib.spkv2_mi355x_matmul_f8_experts_kernel_name(ctypes.byref(decoder._MatmulF8Experts(**a)), name, 64)
    else:
        rc = lib.spkv2_mi355x_matmul_f8_kernel_name(ctypes.byref(decoder._MatmulF8(**a)), name, 64)
    assert rc == 0
    return name.value.decode()


def sizes_of_kernels(dtype, by_expert):
    """For each kernel that some call takes, the smallest sizes found that take it, none of them a multiple of a tile."""
    found = {}
    for rows in (1, 3, 9, 18, 33, 50, 70, 100, 130, 200, 300, 520, 700, 1030, 1500, 2100, 3000, 4100):
        for n in (17, 33, 65, 100, 130, 190, 260, 390, 515, 770, 1029, 2050, 4100):
            for k in (47, 48, 129, 144, 300, 304, 513, 528, 1030, 1040, 2050, 2064, 4100, 4112, 8200, 8208):
                for experts in ((1, 3, 7, 40) if by_expert else (0,)):
                    if rows * n * k * max(experts, 1) > 4e9 or rows * n > 1.7e7:
                        continue
                    kernel = kernel_of(dtype, rows, n, k, experts, rows)
                    size = rows * n * k + experts * n * k * 20
                    if kernel not in found or size < found[kernel][0]:
                        found[kernel] = (size, rows, n, k, experts)
    return {kernel: v[1:] for kernel, v in found.items()}


@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_every_kernel_is_some_calls(dtype, by_expert):
    wanted = {"matmul_" + f for f in FORMS if not (dtype == "float32" and "x256" in f)}
    missing = wanted - set(sizes_of_kernels(dtype, by_expert))
    assert not missing, missing


# ------------------------------------------------------------ numbers and handles of a call

def test_numbers_past_their_types_are_refused():
    import struct

    a, sa, b, sb = Fake((4, 300), F8), Fake((4, 3), "float32"), Fake((5, 200, 300), F8), Fake((5, 2, 3), "float32")
    off, o = Fake((6,), "int32"), Fake((4, 200), "float16")
    for n in (1 << 31, -(1 << 31) - 1, 1 << 63):
        with pytest.raises(struct.error):
            decoder.matmul_f8_experts(a, sa, b, sb, off, o, per_token=n)
    with pytest.raises(struct.error):
        decoder.sort_tokens(Fake((1, 1 << 31), "int32"), off, Fake((1 << 31,), "int32"), Fake((1, 1 << 31), "int32"))
    with pytest.raises(struct.error):
        decoder.quantize_f8(Fake((1, 8), "float32", strides=(1 << 63, 1)), Fake((1, 8), F8), Fake((1, 1), "float32"))
    for per_token in (1.5, "1", None):
        with pytest.raises(TypeError):
            decoder.matmul_f8_experts(a, sa, b, sb, off, o, per_token=per_token)


@pytest.mark.parametrize("stream", [0, None, np.int64(0), ctypes.c_void_p(None), ctypes.c_void_p(0)])
def test_streams_as_numbers_or_handles(stream):
    """No rows: nothing is launched, so no stream is touched."""
    x, q, s = Fake((0, 300), "float32"), Fake((0, 300), F8), Fake((0, 3), "float32")
    decoder.quantize_f8(x, q, s, stream=stream)
    decoder.dequantize_f8(q, s, x, stream=stream)
    for wrong in ("0", 1.0):
        with pytest.raises((TypeError, AttributeError)):
            decoder.quantize_f8(x, q, s, stream=wrong)


def test_tensors_whose_axes_are_no_tuple():
    """shape and stride() may be any sequence; what raises in them comes through."""
    class Listed(Fake):
        def stride(self):
            return list(self._strides)

    class Broken(Fake):
        def data_ptr(self):
            raise KeyError("no storage")

    x, q, s = Listed((0, 300), "float32"), Listed((0, 300), F8), Listed((0, 3), "float32")
    x.shape, q.shape = [0, 300], [0, 300]
    decoder.quantize_f8(x, q, s)
    with pytest.raises(KeyError):
        decoder.quantize_f8(Broken((0, 300), "float32"), q, s)
    with pytest.raises(ValueError):
        decoder.quantize_f8(Fake((0, 300, 1, 1, 1), "float32"), q, s)  # more axes than any call takes
    x._strides = (300,)
    with pytest.raises(ValueError):
        decoder.quantize_f8(x, q, s)
