"""The decoder layer's operators against their formulas in 64 bits, through
spinnv2_amd.decoder, without torch.

Codes, and what is computed from codes by one product, have to be equal.
Tolerances elsewhere count roundings: half a step of the output's type
(bf16 2^-8, fp16 2^-11, fp32 2^-24, relative) and those of the fp32 steps that
the formula needs, bounded from the sums' absolute values."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from spinnv2_amd import decoder
from spinnv2_amd.decoder import DeviceArray as Array, KvCache, to_bfloat16
from spinnv2_amd.runtime import load_library

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALLEST = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}  # the types' steps at zero

LIMIT = {"float32": np.inf, "float16": 65520.0, "bfloat16": np.inf}  # half a step past the type's largest value


def rounded(x, dtype):
    """Values rounded to the type, as float64."""
    with np.errstate(over="ignore"):
        if dtype == "bfloat16":
            return (to_bfloat16(np.asarray(x, np.float32)).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        return np.asarray(x).astype(dtype).astype(np.float64)


def quantised(x):
    """(codes, scales) of the last axis in 64 bits."""
    top = np.abs(x).max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        codes = np.where(top > 0, np.rint(x * 127.0 / top), 0.0)
        bad = ~np.isfinite(top)
        return np.where(bad, 0.0, codes).astype(np.int8), np.where(bad, np.nan, top / 127.0)[..., 0]


def strided(values, dtype, pad, at=0):
    """A 2-d array whose rows lie `pad` elements apart, `at` elements from its buffer's start; what lies between is 77."""
    rows, cols = values.shape
    whole = Array((at + rows * (cols + pad),), dtype)
    whole.upload(77)
    a = Array(values.shape, dtype, buffer=whole.buffer, at=at, strides=(cols + pad, 1))
    a.upload(values)
    return a


def gaps(a):
    """What lies between a strided array's rows, and ahead of it."""
    whole = Array((a.buffer.nbytes // a.itemsize,), a.dtype, buffer=a.buffer).download()
    mask = np.ones(whole.shape, bool)
    mask[a.at:] = False
    end = a.at + a.shape[0] * a.strides[0]
    body = np.ones((a.shape[0], a.strides[0]), bool)
    body[:, :a.shape[1]] = False
    mask[a.at:end] = body.ravel()
    return whole[mask]


# ------------------------------------------------------------------- norm

def _norm_case(rows, cols, dtype, *, residual=True, weight=None, pad=0, at=0, in_place=False, edit=None, seed=1, eps=1e-6):
    rng = np.random.default_rng(seed)
    x = rounded(rng.standard_normal((rows, cols)) * np.where(rng.random(cols) < 0.01, 30.0, 1.0), dtype)
    r = rounded(rng.standard_normal((rows, cols)), dtype) if residual else None
    if edit:
        edit(x)
    wtype = weight or dtype
    w = None if weight == "none" else rounded(1 + 0.3 * rng.standard_normal(cols), wtype)
    dx, dr = strided(x, dtype, pad, at), None if r is None else strided(r, dtype, pad, at)
    dw = None if w is None else Array.of(w, wtype)
    dh = (dx if in_place else strided(np.zeros_like(x), dtype, pad, at)) if residual else None
    dq, ds = strided(np.zeros((rows, cols), np.int8), "int8", pad, at), Array((rows,), "float32")
    decoder.rmsnorm_i8(dx, dw, dq, ds, residual=dr, residual_out=dh, eps=eps)
    with np.errstate(over="ignore", invalid="ignore"):
        h = x if r is None else rounded((x.astype(np.float32) + r.astype(np.float32)), dtype)
        y = h if w is None else h * w
        codes, scale = quantised(y)
        norm = np.sqrt((h * h).sum(1) / cols + eps)
        want = np.where(np.abs(y).max(1) == 0, 0.0, scale / norm)
    np.testing.assert_array_equal(dq.download(), codes)
    got = ds.download().astype(np.float64)
    # 64-bit sums of `cols` squares, one rounding to fp32
    np.testing.assert_allclose(got, want, rtol=2.0 ** -24 * 1.001 + cols * 2.0 ** -52, atol=2.0 ** -150, equal_nan=True)
    if residual:
        np.testing.assert_array_equal(dh.download().astype(np.float64), h)
    if pad or at:
        assert (gaps(dq) == 77).all()
        if residual:
            assert (gaps(dh) == 77).all()
    return dq, ds, codes, got


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (4, 512), (9, 520), (2, 1001), (3, 1032), (2, 2056), (3, 4096), (2, 4104),
                                       (1, 8191), (2, 8192), (2, 9000), (1, 16384), (2, 16400), (1, 30001)])
def test_norm(gpu, rows, cols, dtype):
    _norm_case(rows, cols, dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("kw", [dict(residual=False), dict(weight="float32"), dict(weight="none"), dict(in_place=True), dict(pad=8),
                                dict(pad=5), dict(pad=3, at=1), dict(pad=16, at=16), dict(weight="float32", in_place=True, pad=1)])
@pytest.mark.parametrize("cols", [24, 1040, 17000])
def test_norm_forms(gpu, cols, kw, dtype):
    _norm_case(5, cols, dtype, **kw)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_norm_of_extreme_rows(gpu, dtype):
    """Zeros, one value, infinities, NaN, the type's largest and smallest values: each row by itself."""
    big = {"float32": 3.0e38, "float16": 65504.0, "bfloat16": 3.0e38}[dtype]

    def edit(x):
        x[1] = 0.0
        x[2] = 0.0
        x[2, 5] = -3.0
        x[3, 7] = np.inf
        x[4, 8] = np.nan
        x[5] = rounded(np.full(x.shape[1], big), dtype)
        x[6] = np.where(np.arange(x.shape[1]) % 3, SMALLEST[dtype], -4 * SMALLEST[dtype])
        x[7] = np.where(np.arange(x.shape[1]) % 2, 1.0, 0.5)  # 63.5: ties

    for cols in (72, 1500):
        _norm_case(9, cols, dtype, residual=False, weight="none", edit=edit)
        _norm_case(9, cols, dtype, residual=False, weight="none", edit=edit, eps=0.0)


def test_norm_of_many_rows(gpu):
    _norm_case(4099, 256, "bfloat16")
    _norm_case(70001, 16, "float16")


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols,pad,at", [(1, 1, 0, 0), (7, 16, 0, 0), (5, 20, 0, 0), (3, 33, 0, 0), (6, 4096, 0, 0), (3, 128, 4, 4),
                                              (2, 50, 3, 1), (300, 2048, 16, 16)])
def test_rows_and_back(gpu, rows, cols, pad, at, dtype):
    rng = np.random.default_rng(3)
    x = rounded(rng.standard_normal((rows, cols)) * 3, dtype)
    dx, dq, ds = strided(x, dtype, pad, at), strided(np.zeros(x.shape, np.int8), "int8", pad, at), Array((rows,), "float32")
    out = strided(np.zeros(x.shape), dtype, pad, at)
    decoder.quantize_i8(dx, dq, ds)
    decoder.dequantize_i8(dq, ds, out)
    codes, scale = quantised(x)
    np.testing.assert_array_equal(dq.download(), codes)
    s = ds.download()
    np.testing.assert_array_equal(s, scale.astype(np.float32))
    np.testing.assert_array_equal(out.download().astype(np.float64), rounded(s[:, None] * codes.astype(np.float32), dtype))
    if pad:
        assert (gaps(dq) == 77).all() and (gaps(out) == 77).all()


# ---------------------------------------------------------------- product

def _matmul_case(m, n, k, dtype, bias=False, pads=(0, 0, 0), at=0, extreme=False, seed=5):
    rng = np.random.default_rng(seed)
    if extreme:
        a, b = np.full((m, k), 127, np.int8), np.full((n, k), 127, np.int8)
        a[m // 2], b[n // 2] = -127, -128
    else:
        a, b = (rng.integers(-127, 128, s, dtype=np.int8) for s in ((m, k), (n, k)))
    sa, sb = (0.02 + 0.01 * rng.random(m)).astype(np.float32), (0.0005 + 0.0005 * rng.random(n)).astype(np.float32)
    c = rng.standard_normal(n).astype(np.float32) if bias else None
    da, db = strided(a, "int8", pads[0], at), strided(b, "int8", pads[1], at)
    out = strided(np.zeros((m, n)), dtype, pads[2], at)
    decoder.matmul_i8(da, Array.of(sa), db, Array.of(sb), out, bias=None if c is None else Array.of(c))
    sums = (a.astype(np.float64) @ b.astype(np.float64).T)  # whole numbers below 2^53
    y = sums * sa[:, None].astype(np.float64) * sb.astype(np.float64)
    want = y if c is None else y + c
    # the sum to fp32, two products, the bias's addition; then the output's type
    tol = 3.01 * 2.0 ** -24 * np.abs(y) + (2.0 ** -24 * np.abs(want) if bias else 0)
    tol += HALF[dtype] * (np.abs(want) + tol) + SMALLEST[dtype]
    got = out.download().astype(np.float64)
    assert (np.abs(got - want) <= tol).all(), (m, n, k, float((np.abs(got - want) - tol).max()))
    if any(pads) or at:
        assert (gaps(out) == 77).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 64), (1, 1000, 2048), (1, 4096, 512), (2, 100, 48), (3, 77, 1023), (4, 513, 256),
                                   (5, 33, 4096), (7, 300, 160), (8, 1024, 128), (9, 65, 100), (16, 256, 1040), (17, 129, 512),
                                   (31, 1000, 96), (33, 64, 2048), (64, 1000, 2048), (65, 127, 333), (100, 257, 512), (128, 256, 256),
                                   (129, 384, 64), (255, 512, 128), (256, 256, 1), (257, 513, 200), (300, 1111, 640), (513, 770, 192)])
def test_matmul(gpu, m, n, k, dtype):
    _matmul_case(m, n, k, dtype, bias=(m + n) % 2 == 1)


@pytest.mark.parametrize("m,n,k", [(1, 200, 272), (6, 96, 80), (40, 130, 144), (300, 500, 352), (520, 520, 1024)])
@pytest.mark.parametrize("pads,at", [((16, 32, 8), 16), ((3, 5, 1), 1), ((0, 16, 3), 0), ((4, 4, 4), 4)])
def test_matmul_of_strided_rows(gpu, m, n, k, pads, at):
    _matmul_case(m, n, k, "float32", True, pads, at)
    _matmul_case(m, n, k, "bfloat16", False, pads, at)


@pytest.mark.parametrize("m,n,k", [(1, 64, 1 << 17), (3, 40, (1 << 17) - 16), (70, 130, 1 << 17), (260, 300, 1 << 14)])
def test_matmul_of_the_largest_sums(gpu, m, n, k):
    """127 127 2^17 = 2114060288, just inside int32."""
    _matmul_case(m, n, k, "float32", extreme=True)


def test_matmul_tall_and_wide(gpu):
    _matmul_case(2049, 515, 320, "float16")
    _matmul_case(130, 20001, 64, "bfloat16")
    _matmul_case(1300, 1290, 4096, "float16")


def test_matmul_of_nothing(gpu):
    """k = 0: the bias, or zeros."""
    out = Array.of(np.full((3, 5), 9.0, np.float32))
    a, b = Array((3, 0), "int8"), Array((5, 0), "int8")
    sa, sb, c = Array.of(np.ones(3, np.float32)), Array.of(np.ones(5, np.float32)), Array.of(np.arange(5, dtype=np.float32))
    decoder.matmul_i8(a, sa, b, sb, out, bias=c)
    np.testing.assert_array_equal(out.download(), np.tile(np.arange(5, dtype=np.float32), (3, 1)))
    decoder.matmul_i8(a, sa, b, sb, out)
    assert (out.download() == 0).all()


def test_matmul_carries_what_is_not_finite(gpu):
    """A NaN scale (a row that held a NaN) gives a NaN row, and only that."""
    for m, n, k in ((3, 40, 64), (200, 300, 64)):
        a, b = np.ones((m, k), np.int8), np.ones((n, k), np.int8)
        sa, sb = np.ones(m, np.float32), np.ones(n, np.float32)
        sa[1], sb[n - 2] = np.nan, np.inf
        out = Array((m, n), "float16")
        decoder.matmul_i8(Array.of(a), Array.of(sa), Array.of(b), Array.of(sb), out)
        got = out.download()
        assert np.isnan(got[1]).all() and np.isinf(got[0, n - 2])
        rest = np.delete(np.delete(got, 1, 0), n - 2, 1)
        assert (rest == k).all()


# ------------------------------------------------------------------ cache

def _cache(rng, pages, heads, page, dim, fill=True):
    c = KvCache.empty(pages, heads, page, dim)
    codes = [rng.integers(-127, 128, (pages, heads, page, dim), dtype=np.int8) for _ in range(2)]
    scales = [(0.01 + 0.01 * rng.random((pages, heads, page))).astype(np.float32) for _ in range(2)]
    if fill:
        for b, v in zip(c.buffers, codes + scales):
            b.upload(v)
    return c, codes, scales


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,page,dim,tokens,pad", [(1, 16, 16, 1, 0), (2, 32, 64, 40, 0), (8, 16, 128, 33, 8), (3, 48, 80, 70, 1), (12, 64, 64, 5, 0),
                                                       (1, 256, 256, 300, 0), (5, 16, 112, 19, 3), (4, 32, 192, 21, 0)])
def test_cache_write_and_read(gpu, heads, page, dim, tokens, pad, dtype):
    rng = np.random.default_rng(heads * 100 + dim)
    pages = -(-tokens // page) + 3
    c, codes, scales = _cache(rng, pages, heads, page, dim)
    width = heads * dim
    new = [rounded(rng.standard_normal((tokens, width)) * 2, dtype) for _ in range(2)]
    new[0].reshape(tokens, heads, dim)[0, 0] = 0.0
    if tokens > 4:
        new[1].reshape(tokens, heads, dim)[2, 0, 3] = np.nan
        new[0].reshape(tokens, heads, dim)[3, heads - 1, 1] = -np.inf
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 2:
        slots[1], slots[2 if tokens < 5 else 4] = -1, pages * page  # neither is in the cache
    arrays = [strided(x, dtype, pad) for x in new]
    views = [Array((tokens, heads, dim), dtype, buffer=a.buffer, strides=(width + pad, dim, 1)) for a in arrays]
    c.write(views[0], views[1], Array.of(slots))
    for x, code, scale in zip(new, codes, scales):
        q, s = quantised(x.reshape(tokens, heads, dim))
        for t, slot in enumerate(slots):
            if 0 <= slot < pages * page:
                code[slot // page, :, slot % page] = q[t]
                scale[slot // page, :, slot % page] = s[t]
    got = [b.download() for b in c.buffers]
    for i in range(2):
        np.testing.assert_array_equal(got[i], codes[i])
        np.testing.assert_array_equal(got[2 + i], scales[i])
    # read back: two sequences, one table of them with pages that are not there
    width_t = pages + 2
    table = np.full((3, width_t), -5, np.int32)
    table[0, :pages] = rng.permutation(pages)
    table[2, :pages] = rng.permutation(pages)
    table[2, 1] = pages  # past the cache
    counts = [page + 3, 0, min(2 * page, pages * page) + 1]
    first = np.array([5, 2, page - 1], np.int32)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = int(offsets[-1]) + 2
    outs = [strided(np.full((total, width), 7.0), dtype, pad) for _ in range(2)]
    out_views = [Array((total, heads, dim), dtype, buffer=a.buffer, strides=(width + pad, dim, 1)) for a in outs]
    c.read(Array.of(table), Array.of(first), Array.of(offsets), *out_views)
    for i in range(2):
        want = np.full((total, heads, dim), 7.0)
        for s in range(3):
            for j in range(counts[s]):
                place = int(first[s]) + j
                p = table[s, place // page] if place // page < width_t else -1
                ok = 0 <= p < pages
                want[offsets[s] + j] = (rounded(scales[i][p, :, place % page, None] * codes[i][p, :, place % page].astype(np.float32), dtype) if ok else 0.0)
        np.testing.assert_array_equal(out_views[i].download().astype(np.float64), want)
        if pad:
            assert (gaps(outs[i]) == 77).all()


def test_cache_of_many_tokens(gpu):
    """More vectors than one launch has lanes for at a time, and a read of all of them."""
    rng = np.random.default_rng(9)
    heads, page, dim, tokens = 8, 64, 128, 5000
    pages = -(-tokens // page)
    c = KvCache.empty(pages, heads, page, dim)
    x = rounded(rng.standard_normal((tokens, heads, dim)), "bfloat16")
    a = Array.of(x, "bfloat16")
    table = rng.permutation(pages).astype(np.int32)[None]
    place = np.arange(tokens)
    c.write(a, a, Array.of((table[0, place // page].astype(np.int64) * page + place % page)))
    out = [Array((tokens, heads, dim), "bfloat16") for _ in range(2)]
    c.read(Array.of(table), None, Array.of(np.array([0, tokens], np.int32)), *out)
    q, s = quantised(x)
    want = rounded(s.astype(np.float32)[..., None] * q.astype(np.float32), "bfloat16")
    for o in out:
        np.testing.assert_array_equal(o.download().astype(np.float64), want)


# -------------------------------------------------------------- attention

def _attend_case(lengths, counts, heads, kv, dim, page, dtype, *, causal=True, window=0, pad=0, edit=None, max_length=None, max_queries=None,
                 extra_rows=0, q_size=1.5, seed=11, scale=None):
    rng = np.random.default_rng(seed)
    b = len(lengths)
    need = [max(1, -(-max(n, 0) // page)) for n in lengths]
    width, pages = max(need), sum(need) + 1
    c, codes, scales = _cache(rng, pages, kv, page, dim, fill=False)
    codes = [np.clip(np.rint(rng.standard_normal((pages, kv, page, dim)) * 45), -127, 127).astype(np.int8) for _ in range(2)]
    order = rng.permutation(pages - 1).astype(np.int32) + 1
    table, at = np.zeros((b, width), np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    # what no sequence holds may be anything
    held = np.zeros((pages, page), bool)
    for i, n in enumerate(lengths):
        for t in range(max(n, 0)):
            held[table[i, t // page], t % page] = True
    for s in scales:
        s[~held[:, None].repeat(kv, 1)] = np.nan
    total = int(sum(counts)) + extra_rows
    q = rounded(q_size * rng.standard_normal((total, heads, dim)), dtype)
    if edit:
        edit(q, codes, scales, table)
    for buf, v in zip(c.buffers, codes + scales):
        buf.upload(v)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    qa, oa = strided(q.reshape(total, -1), dtype, pad), strided(np.full((total, heads * dim), 5.0), dtype, pad)
    qv, ov = (Array((total, heads, dim), dtype, buffer=x.buffer, strides=(heads * dim + pad, dim, 1)) for x in (qa, oa))
    kw = dict(max_queries=max(counts) if max_queries is None else max_queries, max_length=max(lengths) if max_length is None else max_length)
    size = decoder.attention_workspace(b, total, heads, c, **kw)
    work = Array((max(size, 1),), "int8")
    work.upload(-1)  # as floats: NaN
    decoder.attention(qv, c, Array.of(table), Array.of(np.array(lengths, np.int32)), Array.of(offsets), ov, causal=causal, window=window,
                      workspace=work if size else None, scale=scale, **kw)
    got = ov.download().astype(np.float64)
    want, tol = np.full((total, heads, dim), 5.0), np.zeros((total, heads, dim))
    factor = dim ** -0.5 if scale is None else scale
    group = heads // kv
    with np.errstate(invalid="ignore"):
        for i, (n, count) in enumerate(zip(lengths, counts)):
            seen = max(0, min(n, kw["max_length"], width * page))
            place = np.arange(seen)
            pg = table[i, place // page] if seen else np.zeros(0, int)
            there = (pg >= 0) & (pg < pages)
            safe = np.where(there, pg, 0)
            for j in range(min(count, kw["max_queries"])):
                last = n - count + j if causal else n - 1
                keep = there & (place <= last) & ((place > last - window) if window else True)
                row = offsets[i] + j
                for h in range(heads):
                    want[row, h] = 0.0
                    if not keep.any():
                        continue
                    kk, vv = (codes[x][safe[keep], h // group, place[keep] % page].astype(np.float64) for x in range(2))
                    ks, vs = (scales[x][safe[keep], h // group, place[keep] % page].astype(np.float64) for x in range(2))
                    s = (kk @ q[row, h]) * ks * factor
                    p = np.exp(s - s.max())
                    v = vv * vs[:, None]
                    want[row, h] = p @ v / p.sum()
                    # a score: its query's rounding, the sum over dim, four products and the exponential's argument
                    wide = dtype == "float32"
                    delta = (np.abs(kk) @ np.abs(q[row, h])) * ks * abs(factor) * ((dim + 8) * 2.0 ** -24 + (2.0 ** -22 if wide else 2.0 ** -36))
                    delta = (delta + np.abs(s) * 6 * 2.0 ** -24).max() + np.abs(s - s.max()).max() * 2.0 ** -23
                    # a weight: its scores, its own rounding to 11 or 22 bits, the exponential's; the sums over the tokens, their joining
                    e = 2.1 * delta + (2.0 ** -22 if wide else 2.0 ** -11) + 2.0 ** -21 + 2 * (len(p) + 64) * 2.0 ** -24
                    a = p @ np.abs(v) / p.sum()
                    tol[row, h] = a * e + np.abs(v).max() * 2.0 ** -30
    tol += HALF[dtype] * (np.abs(want) + tol) + SMALLEST[dtype]
    tol[want == 5.0] = 0.0
    past = np.isinf(got) & (got * want > 0) & (np.abs(want) + tol >= LIMIT[dtype])  # rounds to infinity
    bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | past)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], tol[bad][:4])
    if pad:
        assert (gaps(oa) == 77).all()
    return got, want


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(32, 8, 128, 16), (4, 4, 64, 32), (8, 1, 80, 64), (5, 1, 16, 16), (6, 2, 256, 48), (16, 2, 112, 128), (3, 3, 192, 16)])
def test_attention_of_single_tokens(gpu, heads, kv, dim, page, dtype):
    _attend_case([1, 0, 17, 333, 130, 64], [1, 1, 1, 1, 0, 1], heads, kv, dim, page, dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 64), (12, 12, 64, 32), (8, 1, 80, 16), (2, 1, 256, 16), (5, 1, 48, 16)])
def test_attention_of_prompts(gpu, heads, kv, dim, page, dtype):
    """Whole prompts, one behind an earlier part, one of one token, an idle one, one whose first queries lie before its tokens."""
    _attend_case([70, 200, 1, 33, 9], [70, 37, 1, 0, 12], heads, kv, dim, page, dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim,page,counts,lengths", [(12, 12, 64, 32, [77, 5, 1], [150, 64, 0]), (4, 2, 128, 16, [1, 1, 1], [300, 31, 1]),
                                                              (8, 8, 256, 16, [20, 40, 3], [17, 49, 129]), (6, 3, 80, 64, [130, 2, 0], [100, 1, 7])])
def test_attention_to_an_encoder(gpu, heads, kv, dim, page, counts, lengths, dtype):
    _attend_case(lengths, counts, heads, kv, dim, page, dtype, causal=False)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 1000])
@pytest.mark.parametrize("lengths,counts", [([300, 40, 7], [1, 1, 1]), ([300, 40, 7], [150, 40, 3]), ([200, 3], [4, 7])])
def test_attention_in_a_window(gpu, lengths, counts, window):
    for dtype, dim in (("bfloat16", 128), ("float16", 64), ("float32", 80)):
        _attend_case(lengths, counts, 4, 2, dim, 16, dtype, window=window)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("lengths,counts", [([1500, 2600], [1, 1]), ([900, 2100], [2, 7]), ([1100, 600], [300, 129])])
def test_attention_over_many_tokens(gpu, lengths, counts, dtype):
    """Lengths that are split over workgroups, and joined."""
    _attend_case(lengths, counts, 4, 1, 128, 64, dtype)
    _attend_case(lengths, counts, 2, 2, 64, 32, dtype, causal=False)


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 17, 80]])
def test_attention_of_strided_rows(gpu, counts):
    for dtype, pad in (("bfloat16", 8), ("float16", 3), ("float32", 1)):
        _attend_case([100, 90, 80], counts, 4, 2, 64, 16, dtype, pad=pad, extra_rows=3)


@pytest.mark.parametrize("counts", [[1, 1], [50, 90], [3, 2]])
def test_attention_with_bounds_below_the_sequences(gpu, counts):
    """max_length and max_queries cut what sequences have beyond them."""
    _attend_case([200, 90], counts, 4, 2, 128, 16, "float16", max_length=128)
    _attend_case([200, 90], counts, 4, 2, 128, 16, "float16", max_length=70, causal=False)
    _attend_case([200, 90], counts, 4, 2, 128, 16, "float16", max_queries=max(1, min(counts) - 1))


@pytest.mark.parametrize("counts", [[1, 1, 1], [30, 70, 2]])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_past_bad_pages(gpu, counts, dtype):
    """Pages that the cache does not have are as masked, wherever in the table they are."""
    def edit(q, codes, scales, table):
        table[0, 1], table[0, 3], table[1, 0], table[2, :] = -1, 2 ** 31 - 1, 10 ** 6, -7

    _attend_case([120, 90, 20], counts, 4, 2, 64, 16, dtype, edit=edit)
    _attend_case([120, 90, 20], counts, 4, 2, 64, 16, dtype, edit=edit, causal=False)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_attention_with_nan_in_the_cache(gpu, dtype):
    """Queries ahead of a token whose scales are NaN do not see it; those behind are NaN."""
    def edit(q, codes, scales, table):
        scales[0][table[0, 45 // 16], :, 45 % 16] = np.nan
        scales[1][table[1, 30 // 16], 0, 30 % 16] = np.nan

    got, want = _attend_case([70, 60], [70, 60], 4, 2, 64, 16, dtype, edit=edit)
    assert np.isnan(want[45:70]).all() and np.isfinite(want[:45]).all() and np.isnan(want[100:130, :2]).all()
    _attend_case([70, 60], [1, 1], 4, 2, 64, 16, dtype, edit=edit)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_attention_with_wide_values(gpu, dtype):
    """Scores that grow along the sequence, queries and scales of very different sizes, rows of zeros."""
    def grow(q, codes, scales, table):
        scales[0][:] = scales[0] * (1 + np.arange(scales[0].shape[2]) / 8).astype(np.float32)
        scales[1][:, 0] *= np.float32(1e-6)
        scales[1][:, 1] *= np.float32(3e4)
        q[1] *= 0.0
        q[2] *= 2.0 ** -12
        q[3, 1] = rounded(q[3, 1] * 100, dtype)

    _attend_case([256, 100], [4, 60], 4, 2, 64, 64, dtype, edit=grow)
    _attend_case([256, 100], [200, 60], 4, 2, 128, 64, dtype, edit=grow)
    _attend_case([256, 100], [200, 60], 4, 2, 64, 64, dtype, edit=grow, causal=False, scale=0.5)


@pytest.mark.parametrize("size", [1e-25, 1e-12, 1e20])
def test_attention_with_value_scales_of_any_size(gpu, size):
    def edit(q, codes, scales, table):
        scales[1][:] = scales[1] * np.float32(size)

    _attend_case([100, 300], [1, 1], 4, 2, 64, 16, "float32", edit=edit)
    _attend_case([100, 300], [1, 1], 4, 2, 128, 16, "bfloat16", edit=edit)
    _attend_case([100, 300], [80, 50], 4, 2, 64, 16, "float32", edit=edit)
    _attend_case([100, 300], [80, 50], 4, 2, 128, 16, "bfloat16", edit=edit)


@pytest.mark.parametrize("counts", [[1, 1], [90, 60]])
def test_attention_with_other_scales_of_scores(gpu, counts):
    """Negative, zero, and large enough that one token takes almost all."""
    for scale in (-0.2, 0.0, 2.0):
        _attend_case([100, 300], counts, 4, 2, 64, 16, "float32", scale=scale)
        _attend_case([100, 300], counts, 4, 2, 80, 16, "float16", scale=scale)


# A bound far above the lengths makes calls of many rows take the kernel for
# long ones, 128 rows a workgroup, at sizes that a plain implementation holds.
FAR = 1 << 20


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 64), (12, 12, 64, 32), (8, 1, 80, 16), (2, 1, 256, 16), (10, 2, 48, 16), (4, 2, 96, 48), (3, 3, 192, 16)])
def test_attention_of_many_rows(gpu, heads, kv, dim, page, dtype):
    _attend_case([70, 200, 1, 33, 9], [70, 37, 1, 0, 12], heads, kv, dim, page, dtype, max_length=FAR)
    _attend_case([150, 64, 0], [77, 5, 1], heads, kv, dim, page, dtype, max_length=FAR, causal=False)


@pytest.mark.parametrize("window", [1, 16, 100, 1000])
def test_attention_of_many_rows_in_a_window(gpu, window):
    for dtype, dim in (("bfloat16", 128), ("float16", 64), ("float32", 80)):
        _attend_case([300, 40, 7], [150, 40, 3], 4, 2, dim, 16, dtype, window=window, max_length=FAR)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_attention_of_many_rows_past_what_is_not_finite(gpu, dtype):
    def bad(q, codes, scales, table):
        table[0, 1], table[0, 3], table[1, 0], table[2, :] = -1, 2 ** 31 - 1, 10 ** 6, -7

    def nan(q, codes, scales, table):
        scales[0][table[0, 45 // 16], :, 45 % 16] = np.nan
        scales[1][table[1, 30 // 16], 0, 30 % 16] = np.nan

    def grow(q, codes, scales, table):
        scales[0][:] = scales[0] * (1 + np.arange(scales[0].shape[2]) / 8).astype(np.float32)
        scales[1][:, 0] *= np.float32(1e-6)
        scales[1][:, 1] *= np.float32(3e4)
        q[1] *= 0.0
        q[2] *= 2.0 ** -12
        q[3, 1] = rounded(q[3, 1] * 100, dtype)

    for causal in (True, False):
        _attend_case([120, 90, 20], [30, 70, 2], 4, 2, 64, 16, dtype, edit=bad, causal=causal, max_length=FAR)
    got, want = _attend_case([70, 60], [70, 60], 4, 2, 64, 16, dtype, edit=nan, max_length=FAR)
    assert np.isnan(want[45:70]).all() and np.isfinite(want[:45]).all() and np.isnan(want[100:130, :2]).all()
    _attend_case([256, 100], [200, 60], 4, 2, 128, 64, dtype, edit=grow, max_length=FAR)
    _attend_case([256, 100], [200, 60], 4, 2, 64, 64, dtype, edit=grow, causal=False, scale=0.5, max_length=FAR)
    for scale in (-0.2, 0.0, 2.0):
        _attend_case([100, 300], [90, 60], 4, 2, 80, 16, dtype, scale=scale, max_length=FAR)
    for size in (1e-25, 1e-12, 1e20):
        _attend_case([100, 300], [80, 50], 4, 2, 64, 16, "float32", max_length=FAR,
                     edit=lambda q, c, s, t: s[1].__imul__(np.float32(size)))


def test_attention_of_many_rows_strided_and_bounded(gpu):
    for dtype, pad in (("bfloat16", 8), ("float16", 3), ("float32", 1)):
        _attend_case([100, 90, 80], [40, 17, 80], 4, 2, 64, 16, dtype, pad=pad, extra_rows=3, max_length=FAR)
    _attend_case([200, 90], [50, 90], 4, 2, 128, 16, "float16", max_queries=49, max_length=FAR)
    # long enough by themselves, and cut by the bound
    _attend_case([2600, 2100], [300, 290], 8, 2, 64, 64, "float16", max_length=2000)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_of_many_rows_without_a_join(gpu, dtype):
    """Enough sequences and heads that no split is made: rows leave through LDS."""
    _attend_case([20 + 31 * i for i in range(8)], [20 + 25 * i for i in range(8)], 32, 32, 64, 16, dtype, max_length=FAR)


def test_attention_in_far_slots(gpu):
    """Pages whose bytes lie past 2^32: a cache of 4.5 GiB of keys."""
    heads, page, dim = 1, 256, 256
    pages = (9 << 29) // (heads * page * dim)
    c = KvCache.empty(pages, heads, page, dim)
    rng = np.random.default_rng(2)
    n = 700
    x = rounded(rng.standard_normal((2, n, heads, dim)), "float16")
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    place = np.arange(n)
    slots = Array.of(table[0, place // page].astype(np.int64) * page + place % page)
    k, v = Array.of(x[0], "float16"), Array.of(x[1], "float16")
    c.write(k, v, slots)
    one = Array.of(np.array([0, n], np.int32))
    back = [Array((n, heads, dim), "float32") for _ in range(2)]
    c.read(Array.of(table), None, one, *back)
    kv = []
    for i in range(2):
        q, s = quantised(x[i])
        kv.append(s.astype(np.float32)[..., None] * q.astype(np.float32))
        np.testing.assert_array_equal(back[i].download(), kv[i])
    for count in (1, 40):
        q = rounded(rng.standard_normal((count, 2, dim)), "float16")
        out = Array((count, 2, dim), "float16")
        kw = dict(max_queries=count, max_length=n)
        size = decoder.attention_workspace(1, count, 2, c, **kw)
        decoder.attention(Array.of(q, "float16"), c, Array.of(table), Array.of(np.array([n], np.int32)), Array.of(np.array([0, count], np.int32)),
                          out, workspace=Array((size,), "int8") if size else None, causal=False, **kw)
        s = np.einsum("qhd,td->qht", q, kv[0][:, 0].astype(np.float64)) * dim ** -0.5
        p = np.exp(s - s.max(-1, keepdims=True))
        want = np.einsum("qht,td->qhd", p, kv[1][:, 0].astype(np.float64)) / p.sum(-1, keepdims=True)
        # weights of 11 bits, values below 4; the rest is far smaller
        assert np.abs(out.download().astype(np.float64) - want).max() <= 2.0 ** -10 * 4


# -------------------------------------------------- streams, graphs, repeats

class Hip:
    """The HIP runtime that the library is linked to: another one may be loaded beside it."""

    def __init__(self):
        self.lib = load_library()  # a symbol that it lacks is looked for in its dependencies

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = ctypes.c_void_p()
        self("hipStreamCreateWithFlags", ctypes.byref(s), ctypes.c_uint(1))
        return s


def _layer(seed):
    """The calls of one step on a few sequences, and what they write."""
    rng = np.random.default_rng(seed)
    heads, kv, dim, page, cols, seqs = 4, 2, 64, 16, 256, 3
    x = Array.of(rng.standard_normal((seqs, cols)), "bfloat16")
    w = Array.of(1 + 0.1 * rng.standard_normal(cols), "bfloat16")
    wide = (heads + 2 * kv) * dim
    b, sb = Array.of(rng.integers(-127, 128, (wide, cols), dtype=np.int8)), Array.of((0.001 * rng.random(wide)).astype(np.float32))
    q8, s8 = Array((seqs, cols), "int8"), Array((seqs,), "float32")
    qkv = Array((seqs, wide), "bfloat16")
    parts = [Array((seqs, n, dim), "bfloat16", buffer=qkv.buffer, at=at * dim, strides=(wide, dim, 1)) for n, at in ((heads, 0), (kv, heads), (kv, heads + kv))]
    cache, codes, scales = _cache(rng, 1 + seqs * 80, kv, page, dim)
    lengths = np.array([1200, 77, 3], np.int32)
    table = (1 + np.arange(seqs * 80, dtype=np.int32)).reshape(seqs, 80)
    slots = Array.of(np.array([table[i, (n - 1) // page] * page + (n - 1) % page for i, n in enumerate(lengths)], np.int64))
    table, lengths, offsets = Array.of(table), Array.of(lengths), Array.of(np.arange(seqs + 1, dtype=np.int32))
    kw = dict(max_queries=1, max_length=1200)
    work = Array((max(16, decoder.attention_workspace(seqs, seqs, heads, cache, **kw)),), "int8")
    out = Array((seqs, heads, dim), "bfloat16")

    def step(stream=0):
        decoder.rmsnorm_i8(x, w, q8, s8, stream=stream)
        decoder.matmul_i8(q8, s8, b, sb, qkv, stream=stream)
        cache.write(parts[1], parts[2], slots, stream=stream)
        decoder.attention(parts[0], cache, table, lengths, offsets, out, workspace=work, stream=stream, **kw)

    return x, step, out, rng


def test_calls_run_on_the_stream_they_are_given_and_in_a_graph(gpu):
    hip = Hip()
    x, step, out, rng = _layer(21)
    inputs = [rng.standard_normal(x.shape) for _ in range(4)]
    want = []
    for v in inputs:
        x.upload(v)
        step()
        want.append(out.download())
    assert not np.array_equal(want[0], want[1])
    s = hip.stream()
    for v, w in zip(inputs, want):
        x.upload(v)
        step(s.value)
        hip("hipStreamSynchronize", s)
        np.testing.assert_array_equal(out.download(), w)
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", s, ctypes.c_int(2))
    step(s.value)
    hip("hipStreamEndCapture", s, ctypes.byref(graph))
    hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
    for k in (0, 2, 1, 3, 0):
        x.upload(inputs[k])
        out.upload(0)
        hip("hipGraphLaunch", run, s)
        hip("hipStreamSynchronize", s)
        np.testing.assert_array_equal(out.download(), want[k])
        x.upload(inputs[(k + 1) % 4])
        step()  # eager work between the replays
        np.testing.assert_array_equal(out.download(), want[(k + 1) % 4])
    hip("hipGraphExecDestroy", run)
    hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", s)


def test_results_repeat_bit_by_bit(gpu):
    x, step, out, rng = _layer(23)
    step()
    first = out.download()
    for _ in range(5):
        step()
        np.testing.assert_array_equal(out.download(), first)
    for counts, lengths in (([300, 200], [900, 1000]), ([1, 1], [2000, 2500])):
        runs = [_attend_case(lengths, counts, 4, 2, 64, 16, "bfloat16")[0] for _ in range(2)]
        np.testing.assert_array_equal(*runs)
