"""Edges of the decoder layer's positions, 8-bit floats and experts, against their
formulas in 64 bits; tolerances as in test_gpu_decoder_f8."""

from __future__ import annotations

import numpy as np
import pytest

from spinnv2_amd import build, decoder
from spinnv2_amd.decoder import DeviceArray as Array, KvCache, _FLOAT8, to_float8

from .test_decoder_f8 import FORMS, kernel_of
from .test_decoder_f8_edges import sizes_of_steps
from .test_gpu_decoder import gaps, rounded, strided
from .test_gpu_decoder_f8 import F8, _limit, coded

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------- rotate

@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("pairs,interleaved", [(32, False), (32, True), (29, False), (29, True)])
def test_pairs_of_no_axis_are_not_turned(gpu, pairs, interleaved, dtype):
    """... whatever their partners hold; and head norms of 0 / 0 are NaN, with eps zeros stay zeros."""
    rng = np.random.default_rng(1)
    x = rounded(rng.standard_normal((3, 2, 64)), dtype)
    x[0, 0, :12], x[1, 1, 40:50] = np.inf, np.nan
    dx, out = Array.of(x, dtype), Array(x.shape, dtype)
    args = Array.of(np.array([[7, 8], [9, 10], [1, 2]], np.int32)), Array.of(np.ones(pairs, np.float32)), out, None
    kw = dict(axes=Array.of(rng.choice([-1, 2, 2 ** 31 - 1], pairs).astype(np.int32)), interleaved=interleaved)
    decoder.rotate(dx, None, *args, **kw)
    np.testing.assert_array_equal(out.download(), x)
    dx.upload(np.zeros(x.shape))
    decoder.rotate(dx, None, *args, norm=True, eps=1e-6, **kw)
    assert (out.download() == 0).all()
    for axes in (kw["axes"], Array.of(np.zeros(pairs, np.int32))):
        decoder.rotate(dx, None, *args, axes=axes, norm=True, eps=0.0, interleaved=interleaved)
        assert np.isnan(out.download()).all()


# ------------------------------------------------------------ 8-bit floats

def _gate(x, dtype):
    """(codes' values, scales) of gate_f8 for x [rows, 2 cols], and the values in 64 bits."""
    rows, cols = x.shape[0], x.shape[1] // 2
    q, s = Array((rows, cols), F8), Array((rows, -(-cols // 128)), "float32")
    decoder.gate_f8(Array.of(x, dtype), q, s)
    with np.errstate(over="ignore", invalid="ignore"):
        v = x[:, :cols] / (1 + np.exp(-x[:, :cols])) * x[:, cols:]
    return q.download(), s.download(), v


@pytest.mark.parametrize("dtype,least", [("float32", 2.0 ** -149), ("bfloat16", 2.0 ** -133)])
@pytest.mark.parametrize("factor", [2.0 ** 66, 2.0 ** 100, 2.0 ** 123])
def test_gates_below_fp32s_normal_values(gpu, factor, dtype, least):
    """Gates whose half is subnormal, with factors that make it a block's largest, alone and beside ordinary gates."""
    rng = np.random.default_rng(41)
    t = rng.integers(1, 60, (8, 256)) * least
    t[2:4] = rng.uniform(0.5, 8.0, (2, 256)) * 2.0 ** -126  # around the smallest normal value
    u = rng.uniform(1.0, 2.0, t.shape) * factor
    some = rng.random((4, 256)) < 0.5
    u[4:] = np.where(some, rng.uniform(1.0, 8.0, (4, 256)), u[4:])
    t[4:] = np.where(some, rng.uniform(1.0, 8.0, (4, 256)) * least * factor, t[4:])
    t[6, :128] = 0.0
    x = rounded(np.concatenate([t * rng.choice([-1.0, 1.0], t.shape), u * rng.choice([-1.0, 1.0], t.shape)], 1), dtype)
    got, scale, v = _gate(x, dtype)
    want, want_scale = coded(v)
    np.testing.assert_array_equal(got, want)
    np.testing.assert_allclose(scale, want_scale, rtol=2.0 ** -20.5, atol=2.0 ** -149)


def _assert_nearest(got, want):
    """Scales are the nearest fp32 values to `want`; either one where it lies within 2^-45 of the middle of two."""
    with np.errstate(over="ignore", invalid="ignore"):
        low, high = (np.asarray(want * (1 + d), np.float32) for d in (-2.0 ** -45, 2.0 ** -45))
    assert (((got >= low) & (got <= high)) | (np.isnan(got) & np.isnan(low))).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("cols", [5, 128, 300, 1024])
@pytest.mark.parametrize("kind", ["values", "norm", "gate"])
def test_scales_are_those_of_the_largest_value_in_64_bits(gpu, kind, cols, dtype):
    """A scale has one rounding, and no bit of what lies in other blocks."""
    rng = np.random.default_rng(cols)
    rows = 60
    x = rounded(rng.standard_normal((rows, 2 * cols if kind == "gate" else cols)), dtype)
    w = rounded(1 + 0.3 * rng.standard_normal(cols), "float32")

    def call(x):
        q, s = Array((len(x), cols), F8), Array((len(x), -(-cols // 128)), "float32")
        if kind == "norm":
            decoder.rmsnorm_f8(Array.of(x, dtype), Array.of(w, "float32"), q, s, eps=1e-6)
        else:
            (decoder.gate_f8 if kind == "gate" else decoder.quantize_f8)(Array.of(x, dtype), q, s)
        return q.download(), s.download()

    q, s = call(x)
    v, norm = x, 1.0
    if kind == "norm":
        v, norm = x * w, 1 / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6)
    elif kind == "gate":
        v = x[:, :cols] / (1 + np.exp(-x[:, :cols])) * x[:, cols:]
    values, scale = coded(v)
    np.testing.assert_array_equal(q, values)
    _assert_nearest(s, scale * norm)
    # every row by itself, and among others
    other = np.roll(x, 7, 0)
    other[::3] = x[::3]
    for a, b in zip(call(other), (q, s)):
        np.testing.assert_array_equal(a[::3], b[::3])
    for r in (0, 17):
        for a, b in zip(call(x[r:r + 1]), (q, s)):
            np.testing.assert_array_equal(a[0], b[r])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("cols", [300, 2000, 17000])
def test_blocks_beside_ones_that_are_not_finite(gpu, cols, dtype):
    """A row with a NaN has no norm: its scales are NaN in every block, one of zeros too; one with an infinity has norm 0."""
    rng = np.random.default_rng(3)
    x = rounded(rng.standard_normal((5, cols)), dtype)
    x[:, 128:256] = 0.0
    x[1, 3], x[2, 290], x[3, 7], x[4] = np.nan, np.nan, np.inf, 0.0
    q, s = Array((5, cols), F8), Array((5, -(-cols // 128)), "float32")
    decoder.rmsnorm_f8(Array.of(x, dtype), None, q, s, eps=0.0)
    got, values = s.download(), Array((5, cols), "float32")
    assert np.isnan(got[1:3]).all() and np.isnan(got[3, 0]) and (got[3, 1:] == 0).all() and (got[4] == 0).all()
    assert (got[0, [0, 2]] > 0).all() and got[0, 1] == 0
    decoder.dequantize_f8(q, s, values)
    y = values.download()
    assert np.isnan(y[1:3]).all() and (y[3, 128:] == 0).all() and (y[4] == 0).all()


# ------------------------------------------------- the cache without the native calls

def test_the_cache_writes_and_reads_the_same_without_the_native_calls(gpu, monkeypatch, tmp_path):
    rng = np.random.default_rng(9)
    k, v = (Array.of(rng.standard_normal((40, 2, 64)), "bfloat16") for _ in range(2))
    slots = Array.of(rng.permutation(64)[:40].astype(np.int64))
    table, first = Array.of(np.array([[2, 0], [1, 3]], np.int32)), Array.of(np.array([3, 0], np.int32))
    offsets = Array.of(np.array([0, 20, 45], np.int32))

    def results():
        cache = KvCache.empty(4, 2, 16, 64)
        for b in cache.buffers:
            b.upload(np.zeros(b.shape))
        cache.write(k, v, slots)
        out = [Array((45, 2, 64), "bfloat16") for _ in range(4)]
        cache.read(table, first, offsets, *out[:2])
        cache.read(table, None, offsets, *out[2:])
        return [x.download() for x in (*cache.buffers, *out)]

    want = results()
    monkeypatch.setattr(build, "CALLS", tmp_path / "calls.so")
    monkeypatch.setattr(decoder, "_calls", None)
    for a, b in zip(results(), want):
        np.testing.assert_array_equal(a, b)


# ---------------------------------------------------------------- products

_CODE_OF = to_float8(np.arange(-8, 9))  # of whole numbers up to 8


def _codes(codes, pad):
    """An array of these 8-bit codes [.., rows, k], whose rows lie `pad` codes of NaN apart."""
    *outer, k = codes.shape
    raw = np.full((*outer, k + pad), 0x7F, np.uint8)
    raw[..., :k] = codes
    whole = Array(raw.shape, "int8")
    whole.upload(raw.view(np.int8))
    return Array(codes.shape, F8, buffer=whole.buffer, strides=whole.strides)


class Product:
    """A product of rows with weights, by expert where there are some: its arrays, the call, and its values in 64 bits."""

    def __init__(self, m, n, k, experts, dtype, *, seed, any_codes=False, a_rows=None, order=False, bias=False):
        rng = np.random.default_rng(seed)
        self.m, self.n, self.k, self.experts, self.dtype = m, n, k, experts, dtype
        self.blocks, pad = -(-k // 128), 16
        a_rows, e = m if a_rows is None else a_rows, max(experts, 1)
        if any_codes:
            ca, cb = (to_float8(np.clip(rng.standard_normal(4096) * 160, -448, 448))[rng.integers(0, 4096, s)] for s in ((a_rows, k), (e, n, k)))
            self.a_scale, self.b_scale = (rounded(0.01 * rng.random(s) + 0.001, "float32") for s in ((a_rows, self.blocks), (e, -(-n // 128), self.blocks)))
        else:  # whole numbers and powers of two: their sums have no rounding in any order
            ca, cb = (_CODE_OF[rng.integers(0, 17, s, np.int8)] for s in ((a_rows, k), (e, n, k)))
            self.a_scale, self.b_scale = (2.0 ** rng.integers(-1, 2, s) for s in ((a_rows, self.blocks), (e, -(-n // 128), self.blocks)))
        self.ca, self.cb, self.pad = ca, cb, pad
        self.bias = rng.integers(-99, 99, (e, n)).astype(np.float64) if bias else None
        if experts:
            counts = np.bincount(np.minimum(rng.integers(0, experts, m), rng.integers(0, experts, m)), minlength=experts)
            self.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        else:
            self.offsets = np.array([0, m], np.int32)
        self.order = rng.permutation(max(a_rows, m))[:m].astype(np.int32) if order else None

    def inputs(self):
        """Each output row's input; -1: none."""
        row = np.arange(self.m) if self.order is None else self.order.astype(np.int64)
        return np.where((row >= 0) & (row < len(self.ca)), row, -1)

    def __call__(self):
        out = strided(np.zeros((self.m, self.n)), self.dtype, 8)
        sa, sb = Array.of(self.a_scale, "float32"), Array.of(self.b_scale if self.experts else self.b_scale[0], "float32")
        a, b = _codes(self.ca, self.pad), _codes(self.cb if self.experts else self.cb[0], self.pad)
        if self.experts:
            decoder.matmul_f8_experts(a, sa, b, sb, Array.of(self.offsets), out, order=None if self.order is None else Array.of(self.order),
                                      bias=None if self.bias is None else Array.of(self.bias, "float32"))
        else:
            decoder.matmul_f8(a, sa, b, sb, out, bias=None if self.bias is None else Array.of(self.bias[0], "float32"))
        got = out.download().astype(np.float64)
        assert (gaps(out) == 77).all()
        return got

    def rows(self, rows):
        """Those input rows' values."""
        a = _FLOAT8[self.ca[rows]].astype(np.float64) * np.repeat(self.a_scale[rows], 128, 1)[:, :self.k]
        a[np.asarray(rows) < 0] = 0.0
        return a

    def weights(self, e, cols=slice(None)):
        scale = np.repeat(np.repeat(self.b_scale[e], 128, 0)[:self.n], 128, 1)[:, :self.k]
        return _FLOAT8[self.cb[e, cols]].astype(np.float64) * scale[cols]

    def values(self):
        want, rows = np.zeros((self.m, self.n)), self.inputs()
        for e in range(max(self.experts, 1)):
            low, high = self.offsets[e], self.offsets[e + 1]
            if high > low:
                want[low:high] = self.rows(rows[low:high]) @ self.weights(e).T
                if self.bias is not None:
                    want[low:high] += self.bias[e]
        return want

    def kernel(self):
        return kernel_of(self.dtype, self.m, self.n, self.k, self.experts, len(self.ca), self.pad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", FORMS)
def test_experts_whose_offsets_fall(gpu, form, dtype):
    """Values of rows that several experts have are one's of them, in any mixture; nothing else is written, and no more tiles
    are taken than the rows have."""
    size = sizes_of_steps(dtype, True).get(("matmul_" + form, 5))
    if size is None:
        return
    m, n, k, _ = size
    p = Product(m, n, k, 4, dtype, seed=5)
    p.offsets = np.array([0, m, 3, m, 0], np.int32)
    got, a = p(), p.rows(np.arange(m))
    each = [rounded(a @ p.weights(e).T, dtype) for e in range(4)]
    known = np.logical_or.reduce([got == y for y in (*each, np.zeros((m, n)))])
    assert known.all()


def _steps_cases():
    """(form, type, blocks of k, by expert): every kernel over several steps of k."""
    for dtype in ("float32", "float16", "bfloat16"):
        for by_expert in (False, True):
            for kernel, blocks in sorted(sizes_of_steps(dtype, by_expert)):
                if blocks < 70 or dtype != "float16":
                    yield kernel, dtype, blocks, by_expert


@pytest.mark.parametrize("kernel,dtype,blocks,by_expert", _steps_cases())
def test_every_kernel_over_several_steps(gpu, kernel, dtype, blocks, by_expert):
    """k of 5 to 70 blocks, the last one not whole, codes of NaN behind rows' ends, a bias; by expert through an order of which
    a tenth names rows that are not there: below zero, past a's rows, far past them."""
    m, n, k, experts = sizes_of_steps(dtype, by_expert)[kernel, blocks]
    p = Product(m, n, k, experts, dtype, seed=blocks, order=by_expert, bias=blocks != 9)
    if by_expert:
        rng = np.random.default_rng(2)
        absent = rng.random(m) < 0.1
        p.order[absent] = rng.choice([-1, -2 ** 31, m, m + 1, 2 ** 31 - 1], m).astype(np.int32)[absent]
    if p.kernel() != kernel:  # rows that lie apart may take another: then side by side
        p.pad = 0
    assert p.kernel() == kernel
    with np.errstate(over="ignore"):
        want = rounded(p.values(), dtype)
    np.testing.assert_array_equal(p(), want)


@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", FORMS)
def test_every_kernel_with_any_codes(gpu, form, dtype, by_expert):
    """Codes of all sizes and scales that are no powers of two; a NaN code of a row, one of a channel, a scale of infinity and one
    of NaN change their rows and channels and no other; by expert without an order, more rows than a has."""
    sizes = sizes_of_steps(dtype, by_expert)
    size = next((sizes["matmul_" + form, b] for b in (9, 5, 22, 70) if ("matmul_" + form, b) in sizes), None)
    if size is None:
        assert dtype == "float32" and "x256" in form
        return
    m, n, k, experts = size
    p = Product(m, n, k, experts, dtype, seed=7, any_codes=True, a_rows=max(1, m - m // 9) if by_expert else None)
    rng = np.random.default_rng(8)
    rows, channel, e = rng.permutation(len(p.ca))[:3], int(rng.integers(n)), int(np.searchsorted(p.offsets, m // 2, side="right")) - 1
    odd = np.zeros((m, n), bool)
    if len(rows) == 3:
        p.ca[rows[0], k - 1], p.a_scale[rows[1], 1], p.a_scale[rows[2], p.blocks - 1] = 0x7F, np.inf, np.nan
        odd[rows] = True
        p.cb[e, channel, k // 2] = 0xFF
        odd[p.offsets[e]:p.offsets[e + 1], channel] = True
        odd[p.inputs() < 0] = False
    got = p()
    assert (np.isfinite(got) == ~odd).all()
    assert np.isnan(got[rows[[0, 2]]]).all() if len(rows) == 3 else True
    assert (got[p.inputs() < 0] == 0).all()
    # some rows and channels, those of the tiles' ends among them
    some = np.unique(np.concatenate([rng.integers(0, m, 30), [0, m - 1], p.offsets[1:-1]]))
    some = some[some < m]
    some = some[~odd[some].all(1)]
    cols = np.unique(np.concatenate([rng.integers(0, n, 40), [0, n - 1]]))
    for e in range(max(experts, 1)):
        mine = some[(some >= p.offsets[e]) & (some < p.offsets[e + 1])]
        if not len(mine):
            continue
        a, b = p.rows(p.inputs()[mine]), p.weights(e, cols)
        keep = ~odd[np.ix_(mine, cols)]
        b = np.nan_to_num(b, nan=0.0)
        want = a @ b.T
        ones = np.ones((len(a), p.blocks)), np.ones((-(-len(b) // 128), p.blocks))
        limit = _limit(a, ones[0], b, ones[1], dtype, want)
        assert (np.abs(got[np.ix_(mine, cols)] - want) <= limit)[keep].all()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k,experts", [(6600, 4360, 112, 6), (6600, 4360, 656, 6), (18000, 1540, 112, 70), (9000, 4360, 1040, 3), (5000, 3000, 272, 5)])
def test_rows_that_are_not_there_in_workgroups_of_several_tiles(gpu, m, n, k, experts, dtype, bias):
    """Through an order and without one; which rows are there differs from tile to tile."""
    rng = np.random.default_rng(k)
    for order in (True, False):
        p = Product(m, n, k, experts, dtype, seed=m + order, order=order, bias=bias, a_rows=m if order else m - m // 5)
        if order:
            absent = rng.random(m) < np.repeat(rng.choice([0.0, 0.02, 0.5, 1.0], -(-m // 100)), 100)[:m]
            p.order[absent] = rng.choice([-1, -2 ** 31, m, 2 ** 31 - 1], m).astype(np.int32)[absent]
        p.pad = 0
        assert "x256,groups=1,direct" in p.kernel()
        with np.errstate(over="ignore"):
            want = rounded(p.values(), dtype)
        np.testing.assert_array_equal(p(), want)
