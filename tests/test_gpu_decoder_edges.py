"""The decoder layer's operators where ranges end: windows, sizes, scales and
products next to what their types hold, and combinations of masks, splits and
kernels.  References in 64 bits or in whole numbers, as in test_gpu_decoder."""

from __future__ import annotations

from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

from spinnv2_amd import decoder
from spinnv2_amd.decoder import DeviceArray as Array, KvCache

from .test_decoder_edges import PRODUCTS, SPLIT, matmul_kernel
from .test_gpu_decoder import FAR, HALF, _attend_case, _matmul_case, rounded

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- norm

def _exact_codes(p, top):
    """rint(127 p / top) in rationals: round() of a Fraction takes ties to the even one."""
    return 0 if top == 0 else round(127 * Fraction(float(p)) / Fraction(float(top)))


def _norm_exactly(h, w, dtype, weight_dtype, eps=0.0, in_place=False):
    """h [rows, cols] and w [cols] hold values of their types; products of two of them are exact in float64."""
    rows, cols = h.shape
    q, s = Array((rows, cols), "int8"), Array((rows,), "float32")
    x, more = Array.of(h, dtype), {}
    if in_place:
        more = dict(residual=Array.of(np.zeros_like(h), dtype), residual_out=x)
    decoder.rmsnorm_i8(x, Array.of(w, weight_dtype), q, s, eps=eps, **more)
    p = h * w
    top = np.abs(p).max(1)
    codes = np.array([[_exact_codes(v, t) for v in row] for row, t in zip(p, top)])
    np.testing.assert_array_equal(q.download(), codes)
    want = top / 127 / np.sqrt((h * h).sum(1) / cols + eps)
    np.testing.assert_allclose(s.download().astype(np.float64), want, rtol=2.0 ** -24 * 1.001 + cols * 2.0 ** -52, atol=2.0 ** -150)


@pytest.mark.parametrize("dtype,weight_dtype", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("cols", [3, 40, 1003, 2056, 17000])
def test_norm_of_products_past_float32(gpu, cols, dtype, weight_dtype):
    """Rows whose largest product with the weights passes fp32's largest value, or is far below its smallest."""
    rng = np.random.default_rng(cols)
    sizes = np.array([2.0 ** 124, 2.0 ** 120, 2.0 ** -100, 1.0, 2.0 ** 60])[:, None] if dtype != "float16" else np.array([2.0 ** 13, 1.0, 2.0 ** -8])[:, None]
    h = rounded(np.clip(rng.standard_normal((len(sizes), cols)), -7, 7) * sizes, dtype)
    for w_size in (4.0, 2.0 ** -60) if dtype != "float16" else (2.0 ** 120, 2.0 ** -140):
        w = rounded((1 + rng.random(cols)) * w_size, weight_dtype)
        _norm_exactly(h, w, dtype, weight_dtype)
    w = rounded(2.0 ** rng.uniform(-100, 20, cols), weight_dtype)
    _norm_exactly(h, w, dtype, weight_dtype, in_place=True)


# Whole numbers a b and c d whose quotient 127 a b / (c d) is a border of two codes, or less than 2^-52 of itself beside one.
BORDERS = [(8940899, 9729239, 10614406, 10566517), (11295405, 9747045, 9645777, 13871550), (9160570, 12577316, 12957651, 10603233),
           (14745699, 11389702, 14989556, 14745699), (14594146, 7324835, 12089229, 9639527), (12585681, 8392783, 12248134, 10790721)]


@pytest.mark.parametrize("border", BORDERS)
def test_norm_codes_next_to_a_border(gpu, border):
    """127 a b has 55 bits: in float64 it is rounded past the border, or off it."""
    a, b, c, d = border
    h = np.array([[c, a, -a, 0, a, c, 1, 2, 3, 4], [-c, a, -a, 0, a, 0, 1, 2, 3, 4]], np.float64)
    w = np.array([d, b, b, 1, -b, 1, 1, 1, 1, 1], np.float64)
    _norm_exactly(h, w, "float32", "float32")
    _norm_exactly(h * 2.0 ** -60, w * 2.0 ** -40, "float32", "float32")


def test_norm_of_more_rows_than_a_launch_has_waves(gpu):
    """A wave takes a row up to 1024 columns: 2^26 rows are 2^32 threads."""
    rows = (1 << 26) + 5
    x = np.arange(rows, dtype=np.int64) % 7 - 3
    dx, q, s = Array.of(x.astype(np.float16)[:, None]), Array((rows, 1), "int8"), Array((rows,), "float32")
    decoder.quantize_i8(dx, q, s)
    np.testing.assert_array_equal(q.download()[:, 0], np.sign(x) * 127)
    np.testing.assert_array_equal(s.download(), (np.abs(x) / 127).astype(np.float32))


# ---------------------------------------------------------------- product

# each kernel of the product by one of these
@pytest.mark.parametrize("m,n", [(2, 16), (70, 130), (3, 4100), (300, 520), (65, 3001), (129, 4100), (1500, 1300), (2050, 2050), (2050, 4100)])
def test_matmul_of_sums_of_2_to_the_31(gpu, m, n):
    """2^17 products of -128 and -128: one more than int32 holds."""
    k = 1 << 17
    u, v = np.full(m, -128.0), np.full(n, -128.0)
    u[0], v[n // 2] = 127, 127
    a, b = (np.repeat(x.astype(np.int8)[:, None], k, 1) for x in (u, v))
    out = Array((m, n), "float32")
    decoder.matmul_i8(Array.of(a), Array.of(np.ones(m, np.float32)), Array.of(b), Array.of(np.ones(n, np.float32)), out)
    np.testing.assert_array_equal(out.download(), np.outer(u, v) * k)


@pytest.mark.parametrize("kernel,m,n,k,dtype,bias,pads,at", PRODUCTS)
def test_matmul_of_every_kernel(gpu, kernel, m, n, k, dtype, bias, pads, at):
    _matmul_case(m, n, k, dtype, bias, pads, at)


@pytest.mark.parametrize("kernel,m,n,k", [p[:4] for p in PRODUCTS if p[3] in (15, 333, 2111)])
def test_matmul_of_every_kernel_with_extreme_codes(gpu, kernel, m, n, k):
    _matmul_case(m, n, k, "float32", extreme=True)


@pytest.mark.parametrize("kernel,m,n,k", [p[:4] for p in PRODUCTS if p[3] in (15, 200, 2048)])
def test_matmul_of_every_kernel_with_scales_that_are_not_finite(gpu, kernel, m, n, k):
    """A token's NaN is its row's, a channel's infinity its column's, and no other's."""
    a, b = np.ones((m, k), np.int8), np.ones((n, k), np.int8)
    sa, sb = np.ones(m, np.float32), np.ones(n, np.float32)
    sa[m // 2], sb[n - 2] = np.nan, np.inf
    out = Array((m, n), "float32")
    decoder.matmul_i8(Array.of(a), Array.of(sa), Array.of(b), Array.of(sb), out)
    want = np.full((m, n), np.float32(k))
    want[:, n - 2], want[m // 2] = np.inf, np.nan
    np.testing.assert_array_equal(out.download(), want)


def test_matmul_gives_the_same_bits_in_every_kernel(gpu):
    """One row and channel among fewer or more others, 333 and 2111 codes each."""
    rng = np.random.default_rng(6)
    for k, m, n, parts in ((333, 3001, 4100, [(9, 333), (3, 4100), (17, 4100), (65, 3001), (3001, 130), (700, 3001)]), (2111, 700, 4100, [(129, 4100), (9, 333)])):
        a, b = rng.integers(-127, 128, (m, k), dtype=np.int8), rng.integers(-127, 128, (n, k), dtype=np.int8)
        sa, sb, c = rng.random(m).astype(np.float32), rng.random(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)

        def product(m, n):
            out = Array((m, n), "float32")
            decoder.matmul_i8(Array.of(a[:m]), Array.of(sa[:m]), Array.of(b[:n]), Array.of(sb[:n]), out, bias=Array.of(c[:n]))
            return out.download()

        whole = product(m, n)
        kernels = {matmul_kernel(m, n, k, "float32")}
        for rows, cols in parts:
            np.testing.assert_array_equal(product(rows, cols), whole[:rows, :cols])
            kernels.add(matmul_kernel(rows, cols, k, "float32"))
        assert len(kernels) == len(parts) + 1


def test_matmul_of_rows_far_apart(gpu):
    """260 rows of more than 2^23 bytes: the last ones lie past 2^31."""
    rng = np.random.default_rng(8)
    m, n, k, stride = 260, 70, 200, (1 << 23) + 16
    a, b = rng.integers(-127, 128, (m, k), dtype=np.int8), rng.integers(-127, 128, (n, k), dtype=np.int8)
    far = Array((m, k), "int8", strides=(stride, 1))
    for i, row in enumerate(a):
        assert gpu.spkv2_device_memcpy_h2d(far.data_ptr() + i * stride, row.ctypes.data, k) == 0
    sums = a.astype(np.float64) @ b.astype(np.float64).T
    ones = [Array.of(np.ones(x, np.float32)) for x in (m, n)]
    out = Array((m, n), "float32")
    decoder.matmul_i8(far, ones[0], Array.of(b), ones[1], out)
    np.testing.assert_array_equal(out.download(), sums)
    out = Array((n, m), "float32")
    decoder.matmul_i8(Array.of(b), ones[1], far, ones[0], out)
    np.testing.assert_array_equal(out.download(), sums.T)


# -------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
def test_attention_in_a_window_past_every_token(gpu, window, dtype):
    """The widest windows, with queries that lie before the first token: position + 1 - window is below -2^31."""
    for bound in ({}, {"max_length": FAR}):
        _attend_case([1, 40, 9, 70], [5, 12, 41, 70], 4, 2, 64, 16, dtype, window=window, **bound)
    _attend_case([1, 700], [1, 1], 4, 2, 64, 16, dtype, window=window)


def _cached(lengths, kv, dim, page, seed=3):
    rng = np.random.default_rng(seed)
    need = [max(1, -(-n // page)) for n in lengths]
    pages = sum(need) + 1
    codes = [np.clip(np.rint(rng.standard_normal((pages, kv, page, dim)) * 45), -127, 127).astype(np.int8) for _ in range(2)]
    scales = [(0.01 + 0.01 * rng.random((pages, kv, page))).astype(np.float32) for _ in range(2)]
    order = rng.permutation(pages - 1).astype(np.int32) + 1
    table, at = np.zeros((len(lengths), max(need)), np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return codes, scales, table


def _attend(codes, scales, table, lengths, counts, q, dtype, bound, **kw):
    """out [queries, heads, dim] of one call"""
    cache = KvCache(*(Array.of(v) for v in codes + scales))
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    kw |= dict(max_queries=max(counts), max_length=bound or max(lengths))
    size = decoder.attention_workspace(len(lengths), len(q), q.shape[1], cache, max_queries=kw["max_queries"], max_length=kw["max_length"])
    out = Array(q.shape, dtype)
    decoder.attention(Array.of(q, dtype), cache, Array.of(table), Array.of(np.array(lengths, np.int32)), Array.of(offsets), out,
                      workspace=Array((size,), "int8") if size else None, **kw)
    return out.download()


# counts, lengths and max_length (0: the longest): single tokens without and with splits, few and many rows, many rows with splits
FORMS = [([1, 1], [200, 90], 0), ([1, 1], [2000, 1500], 0), ([40, 90], [100, 90], 0), ([40, 90], [100, 90], FAR),
         ([300, 150], [700, 400], 1 << 15)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("counts,lengths,bound", FORMS)
def test_attention_does_not_depend_on_what_is_not_read(gpu, counts, lengths, bound, window, dtype):
    """The same bits whatever the value scales of tokens behind a row's own, or ahead of its window."""
    heads, kv, dim, page = 4, 2, 64, 16
    codes, scales, table = _cached(lengths, kv, dim, page)
    q = rounded(np.random.default_rng(1).standard_normal((sum(counts), heads, dim)), dtype)
    plain = _attend(codes, scales, table, lengths, counts, q, dtype, bound, window=window)
    for size in (2.0 ** 30, 2.0 ** 60):
        changed = [scales[0], scales[1].copy()]
        at = [n - 1 if c > 1 else n // 2 for n, c in zip(lengths, counts)]
        for i, t in enumerate(at):
            changed[1][table[i, t // page], :, t % page] *= np.float32(size)
        got = _attend(codes, changed, table, lengths, counts, q, dtype, bound, window=window)
        row = 0
        for n, c, t in zip(lengths, counts, at):
            place = np.arange(n - c, n)
            reads = (place >= t) & ((place < t + window) if window else True)
            np.testing.assert_array_equal(got[row:row + c][~reads], plain[row:row + c][~reads])
            row += c


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("counts,lengths,bound", FORMS)
def test_attention_with_values_of_very_different_sizes(gpu, counts, lengths, bound, dtype):
    """One token's values are far larger than the others', its weight next to nothing."""
    for size in (2.0 ** 20, 2.0 ** 32):
        def edit(q, codes, scales, table):
            np.abs(q, out=q)
            for i, n in enumerate(lengths):
                p, r = table[i, (n // 3) // 16], (n // 3) % 16
                codes[0][p, :, r] = -127
                scales[0][p, :, r] = 0.25  # scores below -100
                scales[1][p, :, r] *= np.float32(size)

        got, want = _attend_case(lengths, counts, 4, 2, 64, 16, dtype, edit=edit, **({"max_length": bound} if bound else {}))
        # values of the others: 127 times 0.02 at most; weights of 11 or 22 bits (2^-11, 2^-23), their scores (2^-14.4), sums of up to 2000 tokens (2^-12)
        off = 127 * 0.02 * (2.0 ** -11 if dtype == "float32" else 2.0 ** -10) + HALF[dtype] * np.abs(want) + 2.0 ** -24
        assert (np.abs(got - want) <= off).all(), float((np.abs(got - want) / off).max())


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("counts,lengths,bound", FORMS)
def test_attention_with_small_values_first(gpu, counts, lengths, bound, dtype):
    """The first tokens' values are tiny, or zero, and count among the weights all the same."""
    for small, large in ((2.0 ** -80, 2.0 ** 8 if dtype == "float16" else 2.0 ** 55), (0.0, 2.0 ** 8 if dtype == "float16" else 2.0 ** 55), (2.0 ** -80, 1.0)):
        def edit(q, codes, scales, table):
            first = np.zeros(scales[1].shape, bool)
            for i, n in enumerate(lengths):
                for t in range(n // 2):
                    first[table[i, t // 16], :, t % 16] = True
            scales[1][:] = np.where(first, scales[1] * np.float32(small), scales[1] * np.float32(large))

        _attend_case(lengths, counts, 4, 2, 64, 16, dtype, edit=edit, **({"max_length": bound} if bound else {}))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("counts,lengths,bound", FORMS)
def test_attention_with_infinite_scales(gpu, counts, lengths, bound, value, which, dtype):
    """As NaN: the rows that read the token are NaN, also where its score would be -inf, and the others have the bits that they have without it."""
    heads, kv, dim, page = 4, 2, 64, 16
    codes, scales, table = _cached(lengths, kv, dim, page)
    rng = np.random.default_rng(1)
    q = np.abs(rounded(rng.standard_normal((sum(counts), heads, dim)), dtype))
    at = [n // 2 for n in lengths]
    for i, t in enumerate(at):
        codes[0][table[i, t // page], :, t % page] = np.where(np.arange(kv) % 2, 100, -100)[:, None]  # scores of both signs
    plain = _attend(codes, scales, table, lengths, counts, q, dtype, bound)
    got = []
    for v in (np.nan, value):
        changed = [s.copy() for s in scales]
        for i, t in enumerate(at):
            changed[which][table[i, t // page], :, t % page] = v
        got.append(_attend(codes, changed, table, lengths, counts, q, dtype, bound))
    np.testing.assert_array_equal(got[1], got[0])
    row = 0
    for n, c, t in zip(lengths, counts, at):
        reads = np.arange(n - c, n) >= t
        assert np.isnan(got[0][row:row + c][reads]).all()
        np.testing.assert_array_equal(got[0][row:row + c][~reads], plain[row:row + c][~reads])
        row += c


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("counts,lengths,bound", FORMS)
def test_attention_of_infinite_queries(gpu, counts, lengths, bound, dtype):
    """A query with an infinity gives NaN, also where all of its scores are -infinity, and zeros where it reads nothing."""
    heads, kv, dim, page = 4, 2, 64, 16
    codes, scales, table = _cached(lengths, kv, dim, page)
    codes[0][..., 7] = -np.abs(codes[0][..., 7]) - 1
    q = rounded(np.random.default_rng(1).standard_normal((sum(counts), heads, dim)), dtype)
    plain = _attend(codes, scales, table, lengths, counts, q, dtype, bound)
    q[::2, 1, 7] = np.inf
    got = _attend(codes, scales, table, lengths, counts, q, dtype, bound)
    assert np.isnan(got[::2, 1]).all()
    got[::2, 1] = plain[::2, 1]
    np.testing.assert_array_equal(got, plain)
    assert (_attend(codes, scales, table, [0 for n in lengths], counts, q, dtype, bound or max(lengths)) == 0).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -40, 2.0 ** 40, 2.0 ** 64])
@pytest.mark.parametrize("counts,lengths,bound", FORMS)
def test_attention_with_key_scales_of_any_size(gpu, counts, lengths, bound, size, dtype):
    """Large keys and small queries, and the other way round: the same scores."""
    def edit(q, codes, scales, table):
        scales[0][:] = scales[0] * np.float32(size)
        q /= size

    _attend_case(lengths, counts, 4, 2, 64, 16, dtype, edit=edit, **({"max_length": bound} if bound else {}))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("window", [20, 100, 700])
def test_attention_in_a_window_over_splits(gpu, window, dtype):
    """Splits ahead of the window hold nothing for a row."""
    _attend_case([1500, 2600, 90], [1, 1, 1], 4, 1, 128, 64, dtype, window=window)
    _attend_case([1500, 2600], [3, 5], 4, 2, 64, 16, dtype, window=window)
    _attend_case([700, 530], [80, 60], 4, 2, 64, 16, dtype, window=window, max_length=1 << 15)


@pytest.mark.parametrize("counts,lengths,bound,heads,kv,dim,dtype,causal", SPLIT)
def test_attention_of_many_rows_over_splits(gpu, counts, lengths, bound, heads, kv, dim, dtype, causal):
    _attend_case(lengths, counts, heads, kv, dim, 16, dtype, causal=causal, max_length=bound)


def test_attention_of_lengths_below_zero(gpu):
    """As of no tokens."""
    for counts in ([1, 1, 1], [40, 30, 2]):
        for causal in (True, False):
            _attend_case([-3, 40, -2 ** 31], counts, 4, 2, 64, 16, "bfloat16", causal=causal)


# ---------------------------------------------------------------- example

def test_example_goes_on_after_a_refusal(gpu, monkeypatch):
    """Tokens that do not fit are refused and leave the sequences as they were."""
    monkeypatch.syspath_prepend(str(Path(__file__).resolve().parent.parent / "examples"))
    from decode_i8 import Decoder, Sizes

    prompt = np.arange(9)
    plain, refused = Decoder(Sizes(layers=1), 1, 16), Decoder(Sizes(layers=1), 1, 16)
    plain.forward([prompt])
    refused.forward([prompt])
    with pytest.raises(ValueError):
        refused.forward([np.zeros(8, np.int64)])
    np.testing.assert_array_equal(refused.forward([prompt[:2]]), plain.forward([prompt[:2]]))
