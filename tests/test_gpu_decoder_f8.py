"""The decoder layer's positions, 8-bit floats and experts against their formulas
in 64 bits, through spinnv2_amd.decoder, without torch.

Codes, orders and sums of whole numbers have to be equal.  Tolerances elsewhere
count roundings: half a step of the output's type (bf16 2^-8, fp16 2^-11, fp32
2^-24, relative), and what the formula's own steps leave."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from spinnv2_amd import decoder
from spinnv2_amd.decoder import DeviceArray as Array, KvCache, _FLOAT8, to_float8

from .test_decoder_f8 import FORMS, kernel_of, sizes_of_kernels
from .test_gpu_decoder import HALF, SMALLEST, Hip, gaps, rounded, strided

pytestmark = pytest.mark.gpu

F8 = "float8_e4m3fn"
TYPES = ["float32", "float16", "bfloat16"]


def heads_of(values, dtype, pad=0, at=0):
    """A [tokens, heads, dim] array whose tokens lie `pad` elements apart, as strided()."""
    tokens, heads, dim = values.shape
    a = strided(values.reshape(tokens, heads * dim), dtype, pad, at)
    a.shape, a.strides = values.shape, (heads * dim + pad, dim, 1)
    return a


def flat(a):
    return Array((a.shape[0], a.shape[1] * a.shape[2]), a.dtype, buffer=a.buffer, at=a.at, strides=(a.strides[0], 1))


# ----------------------------------------------------------------- rotate

def turned(x, positions, axis, frequencies, interleaved, weight, eps, norm):
    """The heads x [tokens, heads, dim] in 64 bits."""
    pairs = len(frequencies)
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 if weight is None else weight)
    angle = positions.astype(np.float64)[:, axis] * frequencies.astype(np.float64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b, out = x[..., first], x[..., second], x.copy()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    return out


def _rotate_case(tokens, heads, kv_heads, dim, dtype, *, pairs=None, axes=1, interleaved=False, norm=True, wtype=None, pad=0, at=0, in_place=False,
                 cache=False, page=16, seed=1, edit=None, top=100000, eps=1e-6):
    rng = np.random.default_rng(seed)
    pairs = dim // 2 if pairs is None else pairs
    q, k, v = (rounded(rng.standard_normal((tokens, n, dim)), dtype) for n in (heads, kv_heads, kv_heads))
    if edit:
        edit(q, k, v)
    frequencies = (500000.0 ** (-np.arange(pairs) / max(pairs, 1))).astype(np.float32)
    positions = rng.integers(-5, top, (tokens, axes)).astype(np.int32)
    axis = rng.integers(0, axes, pairs).astype(np.int32)
    weights = [None if wtype == "none" else rounded(1 + 0.3 * rng.standard_normal(dim), wtype or dtype) for _ in range(2)]
    dq, dk, dv = (heads_of(x, dtype, pad, at) for x in (q, k, v))
    oq, ok = (dq, dk) if in_place else (heads_of(np.zeros_like(x), dtype, pad, at) for x in (q, k))
    kw = {}
    if cache:
        pages = tokens // page + 2
        kw["cache"] = KvCache.empty(pages, kv_heads, page, dim)
        for b in kw["cache"].buffers:
            b.upload(np.full(b.shape, 3))
        slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
        if tokens > 2:
            slots[1], slots[2] = -1, pages * page
        kw.update(v=dv, slots=Array.of(slots))
    decoder.rotate(dq, dk, strided(positions, "int32", 2 if axes > 1 else 0), Array.of(frequencies), oq, ok, axes=Array.of(axis) if axes > 1 else None,
                   norm=norm, q_weight=None if weights[0] is None else Array.of(weights[0], wtype or dtype),
                   k_weight=None if weights[1] is None else Array.of(weights[1], wtype or dtype), eps=eps, interleaved=interleaved, **kw)
    for x, w, o in ((q, weights[0], oq), (k, weights[1], ok)):
        with np.errstate(invalid="ignore"):
            want = turned(x, positions, axis, frequencies, interleaved, w, eps, norm)
        got = o.download().astype(np.float64)
        size = np.abs(np.nan_to_num(want)).max(initial=0)
        # 64-bit angles are within 2^-53 of themselves, up to 2^17: 2^-36 of the pair
        np.testing.assert_allclose(got, want, rtol=HALF[dtype] * 1.01, atol=size * 2.0 ** -35 + SMALLEST[dtype], equal_nan=True)
        if pad or at:
            assert (gaps(flat(o)) == 77).all()
    if cache:
        # the same bits as the rotated keys written by a call of their own
        other = KvCache.empty(pages, kv_heads, page, dim)
        for b in other.buffers:
            b.upload(np.full(b.shape, 3))
        other.write(ok, dv, kw["slots"])
        for a, b in zip(kw["cache"].buffers, other.buffers):
            np.testing.assert_array_equal(a.download(), b.download())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(1, 1, 1, 16), (3, 4, 2, 64), (5, 7, 3, 80), (2, 32, 8, 128), (9, 3, 1, 256), (70, 5, 5, 96),
                                                       (700, 8, 1, 64), (3000, 2, 1, 32)])
def test_rotate(gpu, tokens, heads, kv_heads, dim, dtype):
    _rotate_case(tokens, heads, kv_heads, dim, dtype)
    _rotate_case(tokens, heads, kv_heads, dim, dtype, cache=True, pad=8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(pairs=0), dict(pairs=1), dict(pairs=5), dict(pairs=8), dict(pairs=16, interleaved=True), dict(pairs=13, interleaved=True),
                                dict(interleaved=True), dict(norm=False), dict(norm=False, pairs=7), dict(wtype="float32"), dict(wtype="none"),
                                dict(axes=3), dict(axes=2, interleaved=True), dict(pad=3, at=1), dict(in_place=True), dict(in_place=True, pairs=11, pad=1),
                                dict(in_place=True, interleaved=True), dict(cache=True, page=64, axes=3, interleaved=True), dict(top=2 ** 31 - 1, pairs=4)])
@pytest.mark.parametrize("dim", [48, 128])
def test_rotate_variants(gpu, kw, dim, dtype):
    _rotate_case(21, 5, 3, dim, dtype, **kw)


def test_rotate_one_side_alone(gpu):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 3, 64))
    p, f = rng.integers(0, 99, (6, 1)).astype(np.int32), np.float32(1.0) / np.arange(1, 33, dtype=np.float32)
    want = turned(x.astype(np.float32).astype(np.float64), p, np.zeros(32, int), f, False, None, 0, False)
    for keys in (False, True):
        out = Array((6, 3, 64), "float32")
        dx = Array.of(x, "float32")
        dp = Array.of(p[:, 0])
        if keys:
            decoder.rotate(None, dx, dp, Array.of(f), None, out)
        else:
            decoder.rotate(dx, None, dp, Array.of(f), out, None)
        np.testing.assert_allclose(out.download(), want, rtol=2.0 ** -24 * 1.01, atol=2.0 ** -45)


@pytest.mark.parametrize("norm", [False, True])
def test_rotate_values_that_are_not_finite_stay_in_their_head(gpu, norm):
    def edit(q, k, v):
        q[1, 0, 3] = np.nan
        q[2, 1, 60] = np.inf  # past the pairs: nothing turns with it
        k[3, 0, 0] = -np.inf
        v[4, 0, 1] = np.nan

    _rotate_case(6, 2, 2, 64, "float32", pairs=16, norm=norm, cache=True, edit=edit)


def test_rotate_zeros_and_axes_out_of_range(gpu):
    """Heads of zeros stay zeros with eps 0 or not a number of a norm of 0 / 0; a pair of no axis is not turned."""
    x = np.zeros((2, 1, 32))
    x[1] = np.arange(32)
    out = Array((2, 1, 32), "float32")
    decoder.rotate(Array.of(x, "float32"), None, Array.of(np.array([[7, 8], [9, 10]], np.int32)), Array.of(np.ones(16, np.float32)), out, None,
                   axes=Array.of(np.array([-1, 2] * 8, np.int32)))
    np.testing.assert_array_equal(out.download(), x)


# ------------------------------------------------------------ 8-bit floats

def coded(v):
    """(values of codes, scales) of the last axis by blocks of 128, in 64 bits; ties to the even code."""
    rows, cols = v.shape
    blocks = -(-cols // 128)
    values, scales = np.zeros((rows, cols)), np.zeros((rows, blocks))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        for b in range(blocks):
            part = v[:, 128 * b:128 * b + 128]
            top = np.abs(part).max(1)
            finite = np.isfinite(top)
            y = np.where((top > 0)[:, None] & finite[:, None], part * 448.0 / top[:, None], 0.0)
            y = np.clip(y, -448, 448)  # a quotient of doubles may round past 448
            values[:, 128 * b:128 * b + 128] = _FLOAT8[to_float8(y)]
            scales[:, b] = np.where(finite, top / 448, np.nan)
    return values, scales


def _rows_case(kind, rows, cols, dtype, *, pad=0, at=0, residual=True, weight=None, in_place=False, seed=1, edit=None, eps=1e-6, size=1.0):
    rng = np.random.default_rng(seed)
    wide = 2 * cols if kind == "gate" else cols
    x = rounded(rng.standard_normal((rows, wide)) * np.where(rng.random(wide) < 0.01, 30.0, 1.0) * size, dtype)
    if edit:
        edit(x)
    dx = strided(x, dtype, pad, at)
    dq, ds = strided(np.zeros((rows, cols)), F8, pad, at), strided(np.zeros((rows, -(-cols // 128))), "float32", pad, at)
    norm = np.ones((rows, 1))
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == "norm":
            r = rounded(rng.standard_normal((rows, cols)) * size, dtype) if residual else None
            wtype = weight or dtype
            w = None if weight == "none" else rounded(1 + 0.3 * rng.standard_normal(cols), wtype)
            dr = None if r is None else strided(r, dtype, pad, at)
            dh = (dx if in_place else strided(np.zeros_like(x), dtype, pad, at)) if residual else None
            decoder.rmsnorm_f8(dx, None if w is None else Array.of(w, wtype), dq, ds, residual=dr, residual_out=dh, eps=eps)
            h = x if r is None else rounded(x.astype(np.float32) + r.astype(np.float32), dtype)
            norm = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
            v = h if w is None else h * w
            if residual:
                np.testing.assert_array_equal(dh.download().astype(np.float64), h)
        elif kind == "gate":
            decoder.gate_f8(dx, dq, ds)
            v = x[:, :cols] / (1 + np.exp(-x[:, :cols])) * x[:, cols:]
        else:
            decoder.quantize_f8(dx, dq, ds)
            v = x
        codes, scale = coded(v)
        scale = np.where(scale == 0, 0.0, scale * norm)
    got, got_scale = dq.download(), ds.download()
    np.testing.assert_array_equal(got, codes)
    # a norm's sum and root in 64 bits, the products with weights (or a gate) and the scale rounded to fp32: two half steps;
    # of a gate its exponential, quotient and product as well, within 2^-21 in all
    rtol = 2.0 ** -20.5 if kind == "gate" else 2.0 ** -23 * 1.01
    np.testing.assert_allclose(got_scale, scale, rtol=rtol, atol=2.0 ** -149, equal_nan=True)
    if pad or at:
        assert (gaps(dq) == _FLOAT8[to_float8(77)]).all() and (gaps(ds) == 77).all()
    # and back
    back = strided(np.zeros((rows, cols)), dtype, pad, at)
    decoder.dequantize_f8(dq, ds, back)
    with np.errstate(over="ignore", invalid="ignore"):
        want = rounded(got * np.repeat(got_scale, 128, 1)[:, :cols], dtype)
    np.testing.assert_array_equal(back.download().astype(np.float64), want)
    if pad or at:
        assert (gaps(back) == 77).all()


LENGTHS = [(1, 1), (3, 7), (5, 64), (4, 128), (9, 130), (3, 512), (2, 1001), (3, 1032), (2, 2056), (3, 4096), (2, 6001), (2, 8192), (2, 9000), (1, 16384),
           (2, 16400), (1, 30001), (200, 136)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["values", "norm", "gate"])
@pytest.mark.parametrize("rows,cols", LENGTHS)
def test_rows(gpu, rows, cols, kind, dtype):
    _rows_case(kind, rows, cols, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(residual=False), dict(weight="float32"), dict(weight="none"), dict(in_place=True), dict(pad=5), dict(pad=3, at=1),
                                dict(in_place=True, pad=16, at=16), dict(eps=0.0)])
@pytest.mark.parametrize("cols", [5, 300, 5000, 17003])
def test_norm_variants(gpu, cols, kw, dtype):
    _rows_case("norm", 4, cols, dtype, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["values", "gate"])
@pytest.mark.parametrize("kw", [dict(pad=5), dict(pad=3, at=1), dict(pad=16, at=16)])
def test_rows_strided(gpu, kind, kw, dtype):
    _rows_case(kind, 7, 333, dtype, **kw)


@pytest.mark.parametrize("kind", ["values", "norm", "gate"])
@pytest.mark.parametrize("dtype,size", [("float32", 1e-38), ("float32", 1e-42), ("float32", 1e37), ("bfloat16", 1e-38), ("bfloat16", 2.0 ** 120),
                                        ("float16", 2e-7), ("float16", 1000.0), ("float32", 1e-30), ("bfloat16", 1e-20), ("float32", 1e25)])
def test_rows_at_the_ends_of_their_range(gpu, kind, dtype, size):
    if kind == "gate" and dtype != "float16":
        size = min(size, 1e18)  # the product of both halves stays in fp32's range
    _rows_case(kind, 3, 700, dtype, size=size, eps=0.0 if kind == "norm" and dtype == "float32" and size < 1e-20 else 1e-6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["values", "norm", "gate"])
def test_rows_that_are_not_finite_or_zero(gpu, kind, dtype):
    def edit(x):
        x[0, 5], x[1, 200], x[1, 3], x[2, 130] = np.nan, np.inf, -np.inf, np.nan
        x[3] = 0
        x[4, 128:256] = 0
        x[5, :300] = -0.0

    _rows_case(kind, 7, 300, dtype, residual=False, edit=edit)


def test_ties_go_to_the_even_code(gpu):
    """Values whose quotients lie on the border of two codes exactly, and next to it by one step of fp32."""
    border = (_FLOAT8[1:127].astype(np.float64) + _FLOAT8[:126]) / 2
    for top in (448.0, 7.0, 448 * 2.0 ** -40):
        x = np.concatenate([border, [448.0, 0.0]]) * (top / 448)
        both = np.stack([x, -x, np.nextafter(x.astype(np.float32), np.float32(0)), np.minimum(np.nextafter(x.astype(np.float32), np.float32(1e9)), np.float32(top))])
        q, s = Array((4, 128), F8), Array((4, 1), "float32")
        decoder.quantize_f8(Array.of(both, "float32"), q, s)
        want, _ = coded(both.astype(np.float64))
        np.testing.assert_array_equal(q.download(), want)


def test_gates_whose_quotients_are_ties(gpu):
    """Elements with the gate of their block's largest: their quotients are those of the factors, ties among them, whatever the
    gate's own 64-bit value was rounded to."""
    rng = np.random.default_rng(8)
    border = (_FLOAT8[1:127].astype(np.float64) + _FLOAT8[:126]) / 2
    u = np.concatenate([border, [448.0, 0.0]])[None] * np.where(rng.random((64, 128)) < 0.5, -1.0, 1.0)
    g = np.repeat(rng.standard_normal((64, 1)) * 3, 128, 1)
    x = np.concatenate([g, u], 1).astype(np.float32)
    q, s = Array((64, 128), F8), Array((64, 1), "float32")
    decoder.gate_f8(Array.of(x), q, s)
    want = _FLOAT8[to_float8(u * np.sign(x[:, :1]))]
    np.testing.assert_array_equal(q.download(), want)


def test_gates_far_below_zero(gpu):
    """Gates whose exponential leaves fp32's range, alone in their block and beside others, with small and large factors."""
    rng = np.random.default_rng(3)
    g = -np.abs(rng.standard_normal((6, 256))) * 40 - 60
    u = rng.standard_normal((6, 256)) * np.array([1.0, 1e10, 1e30, 1e38, 1e-10, 1.0])[:, None]
    g[4:, ::7] = 1.0
    g[5, 128:] = -2000.0
    x = np.concatenate([g, u], 1).astype(np.float32)
    q, s = Array((6, 256), F8), Array((6, 2), "float32")
    decoder.gate_f8(Array.of(x), q, s)
    x = x.astype(np.float64)
    with np.errstate(over="ignore"):
        want, scale = coded(x[:, :256] / (1 + np.exp(-x[:, :256])) * x[:, 256:])
    np.testing.assert_array_equal(q.download(), want)
    np.testing.assert_allclose(s.download(), scale, rtol=2.0 ** -20.5, atol=2.0 ** -149)


# ---------------------------------------------------------------- products

def _whole(rng, shape):
    """Codes of whole numbers up to 8: their products' sums have no rounding on any matrix core."""
    return rng.integers(-8, 9, shape).astype(np.float64)


def _twos(rng, shape):
    return 2.0 ** rng.integers(-1, 2, shape)


def _scaled(a, sa):
    return a * np.repeat(sa, 128, -1)[..., :a.shape[-1]]


def _product(a, sa, b, sb):
    rows = np.repeat(sb, 128, -2)[..., :b.shape[-2], :]
    return _scaled(a, sa) @ np.swapaxes(_scaled(b, rows), -1, -2)


def _blocks(n):
    return -(-n // 128)


def _matmul_case(m, n, k, dtype, *, bias=False, pad=0, at=0, seed=1):
    rng = np.random.default_rng(seed)
    a, b, sa, sb = _whole(rng, (m, k)), _whole(rng, (n, k)), _twos(rng, (m, _blocks(k))), _twos(rng, (_blocks(n), _blocks(k)))
    c = rng.integers(-99, 99, n).astype(np.float64) if bias else None
    out = strided(np.zeros((m, n)), dtype, pad, at)
    decoder.matmul_f8(strided(a, F8, pad, at), strided(sa, "float32", pad, at), strided(b, F8, pad, at), strided(sb, "float32", pad, at), out,
                      bias=None if c is None else Array.of(c, "float32"))
    want = _product(a, sa, b, sb) + (0.0 if c is None else c)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(out.download().astype(np.float64), rounded(want, dtype))
    if pad or at:
        assert (gaps(out) == 77).all()


SIZES = [(1, 1, 1), (1, 16, 128), (2, 5, 7), (3, 17, 15), (4, 64, 16), (5, 100, 129), (16, 130, 255), (17, 16, 256), (33, 65, 300), (64, 200, 1000),
         (77, 128, 383), (129, 257, 640), (200, 300, 1), (1, 1000, 4100), (300, 64, 2000), (256, 512, 384), (513, 260, 130)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(gpu, m, n, k, dtype):
    _matmul_case(m, n, k, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(bias=True), dict(pad=1), dict(pad=16, at=16), dict(pad=3, at=5, bias=True)])
@pytest.mark.parametrize("m,n,k", [(3, 70, 200), (70, 129, 513), (300, 300, 260)])
def test_matmul_variants(gpu, m, n, k, kw, dtype):
    _matmul_case(m, n, k, dtype, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_every_kernel_of_the_product(gpu, form, dtype):
    """Each kernel at the smallest sizes that take it, with rows apart, a bias, a row of NaN and codes behind the rows' ends."""
    sizes = sizes_of_kernels(dtype, False)
    if "matmul_" + form not in sizes:
        assert dtype == "float32" and "x256" in form
        return
    m, n, k, _ = sizes["matmul_" + form]
    _matmul_case(m, n, k, dtype)
    pad = 0 if k % 16 else 16
    if kernel_of(dtype, m, n, k, pad=pad) == "matmul_" + form:
        _matmul_case(m, n, k, dtype, pad=pad, at=pad, bias=True, seed=2)


def test_matmul_of_nothing(gpu):
    """k = 0: the bias alone, or zeros."""
    out = Array.of(np.full((3, 5), 9.0), "float32")
    bias = np.arange(5.0)
    z = lambda shape, t: Array(shape, t)  # noqa: E731
    decoder.matmul_f8(z((3, 0), F8), z((3, 0), "float32"), z((5, 0), F8), z((1, 0), "float32"), out, bias=Array.of(bias, "float32"))
    np.testing.assert_array_equal(out.download(), np.tile(bias, (3, 1)))
    decoder.matmul_f8(z((3, 0), F8), z((3, 0), "float32"), z((5, 0), F8), z((1, 0), "float32"), out)
    assert not out.download().any()


def _limit(a, sa, b, sb, dtype, want):
    """What roundings leave: half a step of the type; of 16-bit types' products, on the 8-bit matrix cores, each of eight
    products may lose what lies 2^-13 below the largest of them, and sums of a block and of blocks fp32's roundings; of
    fp32's, on the fp16 cores, those roundings alone."""
    size = _product(np.abs(a), sa, np.abs(b), sb)
    k = a.shape[1]
    lost = (k + 2) * 2.0 ** -23 * size
    if dtype != "float32":
        pa, pb = (np.pad(np.abs(_scaled(x, s)), ((0, 0), (0, -k % 8))) for x, s in ((a, sa), (b, np.repeat(sb, 128, 0)[:b.shape[0]])))
        for i in range(0, pa.shape[1], 8):
            lost = lost + 8 * 2.0 ** -13 * (pa[:, None, i:i + 8] * pb[None, :, i:i + 8]).max(-1)
    return np.abs(want) * HALF[dtype] * 1.001 + lost + SMALLEST[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 1024), (20, 70, 515), (70, 130, 384), (140, 150, 300)])
def test_matmul_of_any_codes(gpu, m, n, k, dtype):
    rng = np.random.default_rng(7)
    a, b = (_FLOAT8[to_float8(np.clip(rng.standard_normal(s) * 160, -448, 448))].astype(np.float64) for s in ((m, k), (n, k)))
    sa, sb = (rounded(0.01 * rng.random(s) + 0.001, "float32") for s in ((m, _blocks(k)), (_blocks(n), _blocks(k))))
    out = Array((m, n), dtype)
    decoder.matmul_f8(Array.of(a, F8), Array.of(sa, "float32"), Array.of(b, F8), Array.of(sb, "float32"), out)
    want = _product(a, sa, b, sb)
    got = out.download().astype(np.float64)
    assert (np.abs(got - want) <= _limit(a, sa, b, sb, dtype, want)).all()
    # at random rather than in the worst case: 4e-5 of a sum's size, and half a step, in the root mean square
    rms = np.sqrt(np.mean((got - want) ** 2) / np.mean(want ** 2))
    assert rms < (2e-6 if dtype == "float32" else 1e-4 + HALF[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 40, 300), (70, 150, 300), (300, 300, 300)])
def test_matmul_values_that_are_not_finite_stay_in_their_rows(gpu, m, n, k, dtype):
    """A NaN code or scale makes its row or column NaN and no other; what lies behind a row's end is not read as a value."""
    rng = np.random.default_rng(9)
    a, b, sa, sb = _whole(rng, (m, k)), _whole(rng, (n, k)), _twos(rng, (m, 3)), _twos(rng, (_blocks(n), 3))
    a[1, 299], b[n - 1, 0], sa[2, 1] = np.nan, np.nan, np.inf
    out = Array((m, n), dtype)
    # rows lie 20 elements apart, which hold NaN
    da, db = (Array((r, k + 20), F8) for r in (m, n))
    da.upload(np.nan), db.upload(np.nan)
    va, vb = (Array((r, k), F8, buffer=d.buffer, strides=(k + 20, 1)) for r, d in ((m, da), (n, db)))
    va.upload(a), vb.upload(b)
    decoder.matmul_f8(va, Array.of(sa, "float32"), vb, Array.of(sb, "float32"), out)
    with np.errstate(invalid="ignore"):
        want = _product(a, sa, b, sb)
        sums = _product(a[2:3, 128:256], np.ones((1, 1)), b[:, 128:256], np.ones((_blocks(n), 1)))
    want[2] = np.where(sums[0] == 0, np.nan, np.where(sums[0] > 0, np.inf, -np.inf))
    want[2, n - 1] = np.nan
    np.testing.assert_array_equal(out.download().astype(np.float64), rounded(want, dtype))


# ----------------------------------------------------------------- experts

def _order(ids, experts):
    flat_ids = ids.ravel()
    order = np.concatenate([np.flatnonzero(flat_ids == e) for e in range(experts)]).astype(np.int32)
    place = np.full(flat_ids.shape, -1, np.int32)
    place[order] = np.arange(len(order))
    offsets = np.concatenate([[0], np.cumsum([(flat_ids == e).sum() for e in range(experts)])]).astype(np.int32)
    return offsets, order, place.reshape(ids.shape)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("tokens,per_token,experts", [(0, 2, 3), (1, 1, 1), (1, 8, 64), (63, 1, 5), (64, 8, 64), (65, 3, 300), (1000, 4, 7), (1025, 8, 128),
                                                      (9000, 2, 1), (20011, 5, 33), (70, 2, 4096), (4096, 1, 3), (65536, 1, 9), (65537, 1, 9)])
def test_sort_tokens(gpu, tokens, per_token, experts, wide):
    rng = np.random.default_rng(tokens)
    ids = rng.integers(-2 if tokens % 2 else 0, experts + (2 if tokens % 2 else 0), (tokens, per_token)).astype(np.int64 if wide else np.int32)
    if wide and tokens > 10:
        ids[3, 0], ids[5, 0] = 2 ** 40, -2 ** 40  # whose low halves are expert 0
    want_offsets, want_order, want_place = _order(ids, experts)
    offsets, order, place = Array((experts + 1,), "int32"), Array((tokens * per_token,), "int32"), Array((tokens, per_token), "int32")
    order.upload(np.full(order.shape, 12345)), place.upload(np.full(place.shape, 12345)), offsets.upload(np.full(offsets.shape, 12345))
    decoder.sort_tokens(Array.of(ids), offsets, order, place)
    np.testing.assert_array_equal(offsets.download(), want_offsets)
    got = order.download()
    np.testing.assert_array_equal(got[:len(want_order)], want_order)
    assert (got[len(want_order):] == 12345).all()
    np.testing.assert_array_equal(place.download(), want_place)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,per_token,cols,kw", [(1, 1, 1, {}), (3, 2, 7, {}), (5, 3, 64, dict(pad=3, at=1)), (4, 9, 1001, {}), (70, 8, 520, dict(residual=True)),
                                                      (6, 4, 2049, dict(residual=True, in_place=True, pad=1)), (300, 2, 33, dict(residual=True, pad=8, at=8))])
def test_combine(gpu, tokens, per_token, cols, kw, dtype):
    rng = np.random.default_rng(2)
    pad, at = kw.get("pad", 0), kw.get("at", 0)
    rows = tokens * per_token
    y = rounded(rng.standard_normal((rows, cols)), dtype)
    place = rng.permutation(rows).reshape(tokens, per_token).astype(np.int32)
    if tokens > 2:
        place[1, 0], place[2, -1] = -1, rows
        y[[r for r in range(rows) if r not in place][:2]] = np.nan  # rows that no token picks
        place[0] = place[0, 0]  # one row several times
    weights = rng.standard_normal((tokens, per_token)).astype(np.float32)
    r = rounded(rng.standard_normal((tokens, cols)), dtype) if kw.get("residual") else None
    dr = None if r is None else strided(r, dtype, pad, at)
    out = dr if kw.get("in_place") else strided(np.zeros((tokens, cols)), dtype, pad, at)
    decoder.combine(strided(y, dtype, pad, at), Array.of(place), Array.of(weights), out, residual=dr)
    there = (place >= 0) & (place < rows)
    picked = np.where(there[..., None], y[np.where(there, place, 0)], 0.0)
    terms = picked * weights.astype(np.float64)[..., None]
    want = terms.sum(1) + (0.0 if r is None else r)
    size = np.abs(terms).sum(1) + (0.0 if r is None else np.abs(r))
    # a rounding to fp32 for each term, one to the type
    limit = np.abs(want) * HALF[dtype] * 1.001 + (per_token + 1) * 2.0 ** -24 * size * 1.01 + SMALLEST[dtype]
    assert (np.abs(out.download().astype(np.float64) - want) <= limit).all()
    if pad or at:
        assert (gaps(out) == 77).all()


def _experts_case(ids, experts, n, k, dtype, *, by_order=True, bias=False, pad=0, seed=1, spare=0):
    rng = np.random.default_rng(seed)
    tokens, per_token = ids.shape
    offsets, order, _ = _order(ids, experts)
    rows = tokens if by_order else tokens * per_token
    a, b = _whole(rng, (rows, k)), _whole(rng, (experts, n, k))
    sa, sb = _twos(rng, (rows, _blocks(k))), _twos(rng, (experts, _blocks(n), _blocks(k)))
    c = rng.integers(-99, 99, (experts, n)).astype(np.float64) if bias else None
    m = tokens * per_token + spare
    out = strided(np.zeros((m, n)), dtype, pad)
    out.upload(55)
    full = np.full(m, 0, np.int32)
    full[:len(order)] = order
    decoder.matmul_f8_experts(strided(a, F8, pad), strided(sa, "float32", pad), Array.of(b, F8), Array.of(sb, "float32"), Array.of(offsets), out,
                              order=Array.of(full) if by_order else None, per_token=per_token, bias=None if c is None else Array.of(c, "float32"))
    got = out.download().astype(np.float64)
    for e in range(experts):
        low, high = offsets[e], offsets[e + 1]
        row = order[low:high] // per_token if by_order else np.arange(low, high)
        want = _product(a[row], sa[row], b[e], sb[e]) + (0.0 if c is None else c[e])
        with np.errstate(over="ignore"):
            np.testing.assert_array_equal(got[low:high], rounded(want, dtype))
    assert (got[offsets[-1]:] == 55).all()
    if pad:
        assert (gaps(out) == 77).all()


def _ids(rng, tokens, per_token, experts, kind):
    if kind == "one":
        return np.full((tokens, per_token), experts - 1, np.int32)
    if kind == "holes":  # choices of no expert, and experts that no one chooses
        return rng.integers(-1, max(1, experts // 2), (tokens, per_token)).astype(np.int32)
    return rng.integers(0, experts, (tokens, per_token)).astype(np.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["any", "one", "holes"])
@pytest.mark.parametrize("tokens,per_token,experts,n,k", [(1, 1, 1, 16, 128), (1, 4, 9, 100, 130), (7, 2, 70, 33, 260), (64, 8, 16, 64, 256),
                                                          (130, 3, 5, 130, 200), (400, 4, 3, 300, 140), (33, 2, 130, 17, 15)])
def test_experts(gpu, tokens, per_token, experts, n, k, kind, dtype):
    ids = _ids(np.random.default_rng(tokens), tokens, per_token, experts, kind)
    _experts_case(ids, experts, n, k, dtype, spare=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_every_kernel_of_the_experts_product(gpu, form, dtype):
    """Each kernel at the smallest sizes that take it, the experts of ragged counts of rows."""
    sizes = sizes_of_kernels(dtype, True)
    if "matmul_" + form not in sizes:
        assert dtype == "float32" and "x256" in form
        return
    m, n, k, experts = sizes["matmul_" + form]
    rng = np.random.default_rng(m)
    ids = np.minimum(rng.integers(0, experts, (m, 1)), rng.integers(0, experts, (m, 1))).astype(np.int32)
    assert kernel_of(dtype, m, n, k, experts, m) == "matmul_" + form
    _experts_case(ids, experts, n, k, dtype)


def test_experts_rows_of_one_token(gpu):
    """One output row, whose input is not the first of several."""
    rng = np.random.default_rng(4)
    a, b = _whole(rng, (4, 144)), _whole(rng, (2, 20, 144))
    sa, sb = _twos(rng, (4, 2)), _twos(rng, (2, 1, 2))
    out = Array((1, 20), "float32")
    decoder.matmul_f8_experts(Array.of(a, F8), Array.of(sa, "float32"), Array.of(b, F8), Array.of(sb, "float32"),
                              Array.of(np.array([0, 0, 1], np.int32)), out, order=Array.of(np.array([3], np.int32)))
    np.testing.assert_array_equal(out.download(), _product(a[3:], sa[3:], b[1], sb[1]))


@pytest.mark.parametrize("kw", [dict(by_order=False), dict(bias=True), dict(pad=3), dict(pad=16, bias=True, by_order=False)])
@pytest.mark.parametrize("tokens", [5, 300])
def test_experts_variants(gpu, tokens, kw):
    ids = _ids(np.random.default_rng(3), tokens, 2, 6, "any")
    _experts_case(ids, 6, 140, 300, "bfloat16", **kw)


def test_experts_inputs_that_are_not_there(gpu):
    """Order past a's rows, offsets past m or not rising: zeros, or nothing computed, and no read or write out of range."""
    rng = np.random.default_rng(1)
    a, b = _whole(rng, (4, 64)), _whole(rng, (3, 20, 64))
    ones = lambda shape: Array.of(np.ones(shape), "float32")  # noqa: E731
    out = Array((6, 20), "float32")
    out.upload(55)
    order = np.array([0, 3, 4, 2 ** 31 - 1, -1, 1], np.int32)
    decoder.matmul_f8_experts(Array.of(a, F8), ones((4, 1)), Array.of(b, F8), ones((3, 1, 1)), Array.of(np.array([0, 5, 3, 9], np.int32)), out,
                              order=Array.of(order))
    got = out.download()
    want = np.zeros((6, 20))
    want[[0, 1]] = a[[0, 3]] @ b[0].T
    want[5] = a[1] @ b[2].T
    want[3:5] = 0  # expert 2 from row 3 on, whose order is past a's rows
    np.testing.assert_array_equal(got, want)


# -------------------------------------------------------- streams and graphs

def _layer_arrays(rng, tokens, per_token, experts, width, inner):
    """A layer of experts: norm, sort, product, gate, product, combine; all arrays of one call of it."""
    x = rounded(rng.standard_normal((tokens, width)), "bfloat16")
    ids = _ids(rng, tokens, per_token, experts, "any")
    first, second = rng.standard_normal((experts, 2 * inner, width)), rng.standard_normal((experts, width, inner))
    s = dict(x=Array.of(x, "bfloat16"), weight=Array.of(rounded(1 + 0.2 * rng.standard_normal(width), "bfloat16"), "bfloat16"), ids=Array.of(ids),
             choice=Array.of(rng.random((tokens, per_token)).astype(np.float32)))
    for name, w in (("first", first), ("second", second)):
        e, n, k = w.shape
        # weights by blocks of 128 x 128, as their products take them
        pad = np.pad(w, ((0, 0), (0, -n % 128), (0, -k % 128))).reshape(e, _blocks(n), 128, _blocks(k), 128)
        scale = np.abs(pad).max((2, 4)) / 448
        codes = w / np.repeat(np.repeat(scale, 128, 1), 128, 2)[:, :n, :k]
        s[name], s[name + "_scale"] = Array.of(np.clip(codes, -448, 448), F8), Array.of(scale, "float32")
    rows = tokens * per_token
    s.update(q=Array((tokens, width), F8), q_scale=Array((tokens, _blocks(width)), "float32"), offsets=Array((experts + 1,), "int32"),
             order=Array((rows,), "int32"), place=Array((tokens, per_token), "int32"), up=Array((rows, 2 * inner), "bfloat16"),
             mid=Array((rows, inner), F8), mid_scale=Array((rows, _blocks(inner)), "float32"), down=Array((rows, width), "bfloat16"),
             out=Array((tokens, width), "bfloat16"))
    return s


def _layer(s, per_token, stream=0):
    decoder.rmsnorm_f8(s["x"], s["weight"], s["q"], s["q_scale"], stream=stream)
    decoder.sort_tokens(s["ids"], s["offsets"], s["order"], s["place"], stream=stream)
    decoder.matmul_f8_experts(s["q"], s["q_scale"], s["first"], s["first_scale"], s["offsets"], s["up"], order=s["order"], per_token=per_token, stream=stream)
    decoder.gate_f8(s["up"], s["mid"], s["mid_scale"], stream=stream)
    decoder.matmul_f8_experts(s["mid"], s["mid_scale"], s["second"], s["second_scale"], s["offsets"], s["down"], stream=stream)
    decoder.combine(s["down"], s["place"], s["choice"], s["out"], residual=s["x"], stream=stream)


def _layer_wanted(s, per_token):
    """The layer in 64 bits from its inputs and the weights' codes, without rounding activations."""
    d = {k: v.download().astype(np.float64) for k, v in s.items()}
    x, inner, width = d["x"], d["mid"].shape[1], d["x"].shape[1]
    h = x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6) * d["weight"]
    out = x.copy()
    for t in range(len(x)):
        for j in range(per_token):
            e = int(d["ids"][t, j])
            first, second = (w * np.repeat(np.repeat(sc, 128, 0), 128, 1)[:w.shape[0], :w.shape[1]]
                             for w, sc in ((d["first"][e], d["first_scale"][e]), (d["second"][e], d["second_scale"][e])))
            y = first @ h[t]
            out[t] += d["choice"][t, j] * (second @ (y[:inner] / (1 + np.exp(-y[:inner])) * y[inner:]))
    return out


@pytest.mark.parametrize("tokens", [1, 40])
def test_a_layer_of_experts(gpu, tokens):
    """The operators together, as a layer of experts uses them."""
    rng = np.random.default_rng(11)
    s = _layer_arrays(rng, tokens, 2, 5, 200, 150)
    _layer(s, 2)
    got, want = s["out"].download().astype(np.float64), _layer_wanted(s, 2)
    # inputs' and gates' codes are off by up to 2^-4 of themselves, 2^-4 / sqrt(3) at random, products of the gate by two such;
    # the outputs' sums of them by as much, and bf16 roundings of 2^-9 are small beside it
    error = np.sqrt(np.mean((got - want) ** 2) / np.mean(want ** 2))
    assert error < 3 * 2.0 ** -4 / np.sqrt(3), error
    assert error > 0


def test_streams_and_graphs(gpu):
    """The layer and a rotation into a cache on a stream of its own, and captured and replayed with other inputs between."""
    hip = Hip()
    rng = np.random.default_rng(12)
    s = _layer_arrays(rng, 40, 2, 5, 200, 150)
    cache = KvCache.empty(4, 2, 16, 64)
    heads = [Array.of(rng.standard_normal((40, n, 64)), "bfloat16") for n in (4, 2, 2)]
    q_out, positions = Array((40, 4, 64), "bfloat16"), Array.of(rng.integers(0, 999, 40).astype(np.int32))
    frequencies, slots = Array.of(np.float32(1) / np.arange(1, 33, dtype=np.float32)), Array.of(rng.permutation(64)[:40].astype(np.int64))

    def calls(stream):
        _layer(s, 2, stream)
        decoder.rotate(heads[0], heads[1], positions, frequencies, q_out, None, norm=True, cache=cache, v=heads[2], slots=slots, stream=stream)

    def results():
        return [x.download() for x in (s["out"], s["order"], s["place"], q_out, *cache.buffers)]

    for b in cache.buffers:
        b.upload(np.zeros(b.shape))
    calls(0)
    want = results()
    stream = hip.stream()
    s["out"].upload(0)
    calls(stream.value)
    hip("hipStreamSynchronize", stream)
    for a, b in zip(results(), want):
        np.testing.assert_array_equal(a, b)
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", stream, ctypes.c_int(2))
    calls(stream.value)
    hip("hipStreamEndCapture", stream, ctypes.byref(graph))
    hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
    for seed in (20, 21, 22):
        new = np.random.default_rng(seed)
        s["x"].upload(new.standard_normal((40, 200)))
        s["ids"].upload(_ids(new, 40, 2, 5, "holes" if seed == 21 else "any"))
        heads[1].upload(new.standard_normal((40, 2, 64)))
        for x in (s["up"], s["down"]):
            x.upload(np.zeros(x.shape))
        hip("hipGraphLaunch", run, stream)
        hip("hipStreamSynchronize", stream)
        replayed = results()
        s["out"].upload(0), q_out.upload(0)
        calls(0)
        for a, b in zip(results(), replayed):
            np.testing.assert_array_equal(a, b)
    hip("hipGraphExecDestroy", run)
    hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", stream)


# ------------------------------------------------------- rows far apart, calls at once

class Far(Array):
    """Rows of the last axis 2^27 bytes and a page apart in a buffer that arrays share, each from a place of its own in them."""

    ROWS, STEP, AREA = 64, 2 ** 27 + 4096, 2 ** 16

    def __init__(self, buffer, area, shape, dtype):
        size = 2 if dtype in ("bfloat16", "float16") else 1 if dtype == F8 else 4
        inner = shape[1:]
        strides = (self.STEP // size, *(int(np.prod(inner[i + 1:])) for i in range(len(inner))))
        assert shape[0] <= self.ROWS and np.prod(inner) * size <= self.AREA
        super().__init__(shape, dtype, buffer=buffer, at=area * self.AREA // size, strides=strides)

    def _each(self):
        for i in range(self.shape[0]):
            yield i, ctypes.c_void_p(self.data_ptr() + i * self.STEP), int(np.prod(self.shape[1:])) * self.itemsize

    def upload(self, values):
        values = np.broadcast_to(np.asarray(values), self.shape)
        to = {"bfloat16": decoder.to_bfloat16, "float8_e4m3fn": to_float8}.get(self.dtype, lambda v: v.astype(self.dtype))
        lib = self.buffer.lib
        for i, p, n in self._each():
            row = np.ascontiguousarray(to(values[i]))
            assert row.nbytes == n and lib.spkv2_device_memcpy_h2d(p, row.ctypes.data, n) == 0
        return self

    def download(self):
        kind, lib = self._kind(), self.buffer.lib
        raw = np.empty(self.shape, kind)
        for i, p, n in self._each():
            assert lib.spkv2_device_memcpy_d2h(raw[i:].ctypes.data, p, n) == 0
        if self.dtype == F8:
            return _FLOAT8[raw]
        return (raw.astype(np.uint32) << 16).view(np.float32) if self.dtype == "bfloat16" else raw


@pytest.fixture(scope="module")
def far(gpu):
    """Far arrays of one buffer of 8 GiB: far(area, shape, dtype)."""
    from spinnv2_amd.runtime import DeviceBuffer

    buffer = DeviceBuffer(Far.ROWS * Far.STEP)
    yield lambda area, shape, dtype: Far(buffer, area, shape, dtype)
    buffer.free()


@pytest.mark.parametrize("kind", ["values", "norm", "gate"])
def test_rows_far_apart(far, kind):
    """Rows past 2^32 bytes from the first, and back."""
    rows, cols = 50, 1000
    rng = np.random.default_rng(2)
    x = rounded(rng.standard_normal((rows, 2 * cols if kind == "gate" else cols)), "bfloat16")
    dx, q, s, back = far(0, x.shape, "bfloat16").upload(x), far(1, (rows, cols), F8), far(2, (rows, 8), "float32"), far(3, (rows, cols), "bfloat16")
    want_q, want_s, want_back = Array((rows, cols), F8), Array((rows, 8), "float32"), Array((rows, cols), "bfloat16")
    near = Array.of(x, "bfloat16")
    w = Array.of(rounded(1 + 0.3 * rng.standard_normal(cols), "bfloat16"), "bfloat16")
    for a, b, c, d, h in ((dx, q, s, back, far(4, (rows, cols), "bfloat16")), (near, want_q, want_s, want_back, Array((rows, cols), "bfloat16"))):
        if kind == "norm":
            decoder.rmsnorm_f8(a, w, b, c, residual=a, residual_out=h)
            np.testing.assert_array_equal(h.download(), rounded(2 * x, "bfloat16"))
        else:
            (decoder.gate_f8 if kind == "gate" else decoder.quantize_f8)(a, b, c)
        decoder.dequantize_f8(b, c, d)
    for a, b in ((q, want_q), (s, want_s), (back, want_back)):
        np.testing.assert_array_equal(a.download(), b.download())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", ["a", "b", "out"])
def test_matmul_rows_far_apart(far, which, dtype):
    m, n, k = (64, 60, 384) if which == "b" else (60, 300, 384)
    rng = np.random.default_rng(3)
    a, b, sa, sb = _whole(rng, (m, k)), _whole(rng, (n, k)), _twos(rng, (m, 3)), _twos(rng, (_blocks(n), 3))
    put = lambda area, v, t, name: far(area, v.shape, t).upload(v) if which == name else Array.of(v, t)  # noqa: E731
    out = far(4, (m, n), dtype) if which == "out" else Array((m, n), dtype)
    decoder.matmul_f8(put(0, a, F8, "a"), put(1, sa, "float32", "a"), put(2, b, F8, "b"), put(3, sb, "float32", "b"), out)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(out.download().astype(np.float64), rounded(_product(a, sa, b, sb), dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [4, 60, 900])
def test_experts_far_apart(far, tokens, dtype):
    """Experts' weights past 2^32 bytes from the first, and outputs where they are few."""
    n, k, experts = 140, 256, 60
    rng = np.random.default_rng(tokens)
    ids = rng.integers(experts - 5, experts, (tokens, 1)).astype(np.int32)
    offsets, order, _ = _order(ids, experts)
    a, b, sa, sb = _whole(rng, (tokens, k)), _whole(rng, (experts, n, k)), _twos(rng, (tokens, 2)), _twos(rng, (experts, 2, 2))
    out = far(4, (tokens, n), dtype) if tokens <= Far.ROWS else Array((tokens, n), dtype)
    decoder.matmul_f8_experts(Array.of(a, F8), Array.of(sa, "float32"), far(0, b.shape, F8).upload(b), far(1, sb.shape, "float32").upload(sb),
                              Array.of(offsets), out, order=Array.of(order))
    want = np.zeros((tokens, n))
    for e in range(experts):
        row = order[offsets[e]:offsets[e + 1]]
        want[offsets[e]:offsets[e + 1]] = _product(a[row], sa[row], b[e], sb[e])
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(out.download().astype(np.float64), rounded(want, dtype))


def test_combine_and_rotate_far_apart(far):
    rng = np.random.default_rng(6)
    y, r = rounded(rng.standard_normal((60, 520)), "bfloat16"), rounded(rng.standard_normal((50, 520)), "bfloat16")
    place, weights = Array.of(rng.integers(0, 60, (50, 3)).astype(np.int32)), Array.of(rng.standard_normal((50, 3)).astype(np.float32))
    out, want = far(2, (50, 520), "bfloat16"), Array((50, 520), "bfloat16")
    decoder.combine(far(0, y.shape, "bfloat16").upload(y), place, weights, out, residual=far(1, r.shape, "bfloat16").upload(r))
    decoder.combine(Array.of(y, "bfloat16"), place, weights, want, residual=Array.of(r, "bfloat16"))
    np.testing.assert_array_equal(out.download(), want.download())
    heads = [rounded(rng.standard_normal((50, n, 64)), "bfloat16") for n in (4, 2, 2)]
    positions, frequencies = rng.integers(0, 9999, (50, 2)).astype(np.int32), np.float32(1) / np.arange(1, 33, dtype=np.float32)
    axes, slots = Array.of(rng.integers(0, 2, 32).astype(np.int32)), Array.of(rng.permutation(64)[:50].astype(np.int64))
    results = []
    for place_at in (lambda area, v, t: far(area, v.shape, t).upload(v), lambda area, v, t: Array.of(v, t)):
        q, k, v = (place_at(i, x, "bfloat16") for i, x in enumerate(heads))
        cache = KvCache.empty(4, 2, 16, 64)
        for b in cache.buffers:
            b.upload(np.zeros(b.shape))
        decoder.rotate(q, k, place_at(3, positions, "int32"), Array.of(frequencies), q, k, axes=axes, norm=True, cache=cache, v=v, slots=slots)
        results.append([x.download() for x in (q, k, *cache.buffers)])
    for a, b in zip(*results):
        np.testing.assert_array_equal(a, b)


def test_calls_of_two_threads_at_once(gpu):
    """Two threads, each with a layer and a stream of its own: nothing of a call is shared with another."""
    import threading

    hip = Hip()
    layers = [_layer_arrays(np.random.default_rng(30 + i), 30 + 9 * i, 2, 5, 200, 150) for i in range(2)]
    wanted = []
    for s in layers:
        _layer(s, 2)
        wanted.append([s[k].download() for k in ("out", "order", "place", "offsets")])
        s["out"].upload(0)
    streams, failed = [hip.stream() for _ in layers], []

    def work(s, stream):
        try:
            for _ in range(40):
                _layer(s, 2, stream.value)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(layers, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for stream in streams:
        hip("hipStreamSynchronize", stream)
        hip("hipStreamDestroy", stream)
    assert not failed
    for s, want in zip(layers, wanted):
        for name, w in zip(("out", "order", "place", "offsets"), want):
            np.testing.assert_array_equal(s[name].download(), w)


@pytest.mark.parametrize("tokens", [1, 50, 3000])
def test_as_many_experts_as_there_may_be(gpu, tokens):
    rng = np.random.default_rng(tokens)
    _experts_case(_ids(rng, tokens, 2, 4096, "any"), 4096, 9, 48, "float32", spare=3)


# tiles 256 channels wide of which a workgroup takes several: one to nine blocks of k, whole ones and not
@pytest.mark.parametrize("m,n,k", [(4700, 4360, 16), (4700, 4360, 128), (4700, 4360, 400), (4700, 4360, 512), (4700, 4360, 1040), (8300, 4360, 272)])
def test_workgroups_of_several_tiles(gpu, m, n, k):
    assert kernel_of("bfloat16", m, n, k) == "matmul_tiles<256x256,groups=1,direct>"
    _matmul_case(m, n, k, "bfloat16", bias=k > 300)


@pytest.mark.parametrize("kind,kw", [("any", {}), ("holes", dict(bias=True)), ("any", dict(by_order=False, spare=5))])
@pytest.mark.parametrize("k", [112, 384, 656])
def test_workgroups_of_several_experts_tiles(gpu, k, kind, kw):
    for tokens, experts, n in ((3300, 6, 4360), (9000, 70, 1540))[:2 if k == 112 else 1]:
        assert "x256,groups=1,direct" in kernel_of("bfloat16", 2 * tokens, n, k, experts, tokens)
        _experts_case(_ids(np.random.default_rng(k), tokens, 2, experts, kind), experts, n, k, "bfloat16", **kw)
