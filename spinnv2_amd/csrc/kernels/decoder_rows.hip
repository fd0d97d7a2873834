// Rows of a decoder layer in 8 bits: the residual's addition with a
// root-mean-square norm and int8 codes, and codes back to values.
//
//   h = x + r,  y = h w / sqrt(mean(h^2) + eps),  top = max|y|,
//   q = rint(127 y / top),  scale = top / 127
//
// The norm is one factor of the whole row, so it cancels out of q: the codes
// are those of p = h w, and only the scale needs the sum of squares.  Codes
// are therefore exact: of 16-bit rows p has at most 22 bits and is held in
// fp32, with an fp32 factor in it at most 48, held in fp64.  A product of two
// bf16 may leave fp32's range: a row whose largest does, or is so small that
// others would lose bits that their codes need, is multiplied again in fp64, an
// element at a time, so that the other rows pay no registers for it (1596 x 9233
// and back 44.5 us, 48.4 with runs of 8 in registers there too; 8190 x 4096
// 66.6, 68.8 with fp64 for every row).
//
// One pass: a thread keeps its part of the row in registers between the
// statistics and the codes, so each input is read once and each output
// written once.  Bound by HBM: 8190 x 4096 of bf16 with a residual, 235 MB, in
// 47 us (5.0 TB/s), its codes back to values, 101 MB, in 20 (5.1 TB/s; 16.8
// right behind the norm, whose codes the cache still holds); a few rows by the
// launch (4 x 2048: 3.3 us and 1.8).  Rows of odd lengths lie at any alignment
// and are read 16 bytes a lane all the same, the row's end moved into place:
// 1596 x 9233 without a residual 19 us, and back 9.  Rows of more than 16384
// elements are read twice (1000 x 17000 with a residual 44.5 us, 28 of 16384).
#include <type_traits>

#include "decoder.hpp"

namespace spk::dec {

namespace {

struct RowArgs {
    const void *x, *residual, *weight;
    void *h;
    int8_t *q;
    float *scale;
    int64_t rows, x_stride, r_stride, h_stride, q_stride;
    int cols;
    int norm;
    float eps;
};

template <typename T, typename W>
struct Product {
    using type = float;
};
template <typename W>
struct Product<float, W> {
    using type = double;
};
template <>
struct Product<_Float16, float> {
    using type = double;
};
template <>
struct Product<__bf16, float> {
    using type = double;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
template <typename U>
__device__ __forceinline__ U wave_max(U v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const U o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}

// THREADS threads a row (a wave: several rows a workgroup), each with CHUNKS
// runs of VEC neighbouring elements in registers; CHUNKS = 0: rows of any
// length, read again for the codes.  TAIL: cols is no multiple of VEC.
template <typename T, typename W, int THREADS, int VEC, int CHUNKS, bool TAIL>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) rmsnorm_rows(RowArgs a) {
    using P = typename Product<T, W>::type;
    using U = decltype(abs_bits(P{}));
    constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
    const int64_t row = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kRows + (kRows > 1 ? threadIdx.x / THREADS : 0);
    if (row >= a.rows) return;  // whole waves, or workgroups
    const int tid = kRows > 1 ? threadIdx.x % THREADS : threadIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.r_stride : nullptr;
    T *h = a.h ? static_cast<T *>(a.h) + row * a.h_stride : nullptr;
    const W *w = static_cast<const W *>(a.weight);
    int8_t *q = a.q + row * a.q_stride;
    const int chunks = (a.cols + THREADS * VEC - 1) / (THREADS * VEC);

    float hv[CHUNKS ? CHUNKS : 1][VEC];
    double sum = 0.0;
    U top = 0;
    auto from = [&](int c) { return min((c * THREADS + tid) * VEC, a.cols - VEC); };
    struct Raw {
        Vec<T, VEC> x, r;
    };
    auto fetch = [&](int c, Raw &v) {
        v.x = load_vec<T, VEC>(x + from(c));
        if (r) v.r = load_vec<T, VEC>(r + from(c));
    };
    auto sum_up = [&](int c, const Raw &v, float(&f)[VEC]) {
        const int i = (c * THREADS + tid) * VEC;
        widen(v.x, f);
        if (r) {
            float g[VEC];
            widen(v.r, g);
#pragma unroll
            for (int j = 0; j < VEC; j++) f[j] = static_cast<float>(static_cast<T>(f[j] + g[j]));
        }
        settle<VEC, TAIL>(i, a.cols, f);
    };
    auto keep = [&](int c, const float(&f)[VEC]) {
        const int i = (c * THREADS + tid) * VEC;
        if (h && i < a.cols) store_some<VEC>(h + i, TAIL ? a.cols - i : VEC, f);
    };
    auto products = [&](int c, const float(&f)[VEC], P(&p)[VEC]) {
        float g[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) g[j] = 1.0f;
        if (w) {
            widen(load_vec<W, VEC>(w + from(c)), g);
            settle<VEC, TAIL>((c * THREADS + tid) * VEC, a.cols, g);
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) p[j] = static_cast<P>(f[j]) * static_cast<P>(g[j]);
    };
    auto statistics = [&](int c, const float(&f)[VEC]) {
        P p[VEC];
        products(c, f, p);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            // squares in 64 bits: no row of fp32 or bf16 overflows them
            sum = __builtin_fma(static_cast<double>(f[j]), static_cast<double>(f[j]), sum);
            const U b = abs_bits(p[j]);  // ordered as the values are, NaN above infinity
            top = b > top ? b : top;
        }
    };
    if constexpr (CHUNKS > 0) {
        Raw raw[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) fetch(c, raw[c]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) sum_up(c, raw[c], hv[c]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) keep(c, hv[c]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) statistics(c, hv[c]);
    } else {
        for (int c = 0; c < chunks; c++) {
            Raw raw;
            fetch(c, raw);
            sum_up(c, raw, hv[0]);
            keep(c, hv[0]);
            statistics(c, hv[0]);
        }
    }
    sum = wave_sum(sum);
    top = wave_max(top);
    if constexpr (THREADS > kWave) {
        __shared__ double sums[THREADS / kWave];
        __shared__ U tops[THREADS / kWave];
        if ((tid & (kWave - 1)) == 0) {
            sums[tid / kWave] = sum;
            tops[tid / kWave] = top;
        }
        __syncthreads();
        sum = 0.0;
        top = 0;
#pragma unroll
        for (int i = 0; i < THREADS / kWave; i++) {
            sum += sums[i];
            top = tops[i] > top ? tops[i] : top;
        }
    }
    auto put_scale = [&](double amax) {  // infinite or NaN: the row is
        double s = amax / 127.0;
        if (a.norm) s /= sqrt(sum / a.cols + static_cast<double>(a.eps));
        // 0 of a row of zeros, whose norm may be 0 / 0
        a.scale[row] = !(amax < __builtin_inf()) ? __builtin_nanf("") : amax == 0.0 ? 0.0f : static_cast<float>(s);
    };
    if constexpr (std::is_same_v<P, float> && std::is_same_v<T, __bf16>) {
        // Products below 2^-126 lose bits: next to a top of 2^-90 their codes are 0 all the same.  The row's
        // threads have one top, and turn here together.
        if (w && (top < __builtin_bit_cast(unsigned, 0x1p-90f) || top >= kInfBits)) {
            // h as it was stored, if it was: x may have been overwritten by it
            auto product = [&](int i) {
                const float f = h ? static_cast<float>(h[i]) : r ? static_cast<float>(static_cast<T>(static_cast<float>(x[i]) + static_cast<float>(r[i]))) : static_cast<float>(x[i]);
                return static_cast<double>(f) * static_cast<double>(static_cast<float>(w[i]));
            };
            // this thread's own elements: others may not have stored theirs yet
            auto over_own = [&](auto &&work) {
#pragma unroll 1
                for (int e = 0; e < chunks * VEC; e++) {
                    const int i = (e / VEC * THREADS + tid) * VEC + e % VEC;
                    if (i < a.cols) work(i);
                }
            };
            uint64_t bits = 0;
            over_own([&](int i) { bits = max(bits, abs_bits(product(i))); });
            bits = wave_max(bits);
            if constexpr (THREADS > kWave) {
                __shared__ uint64_t wides[THREADS / kWave];
                if ((tid & (kWave - 1)) == 0) wides[tid / kWave] = bits;
                __syncthreads();
#pragma unroll 1
                for (int i = 0; i < THREADS / kWave; i++) bits = max(bits, wides[i]);
            }
            const double wide = __builtin_bit_cast(double, bits);
            if (tid == 0) put_scale(wide);
            over_own([&](int i) {
                const double p[1] = {product(i)};
                int8_t code[1] = {0};
                if (wide < __builtin_inf() && wide != 0.0) quantise<1>(p, wide, code);
                q[i] = code[0];
            });
            return;
        }
    }
    constexpr U kInf = sizeof(U) == 8 ? static_cast<U>(0x7ff0000000000000ull) : static_cast<U>(kInfBits);
    const bool finite = top < kInf;
    const P amax = __builtin_bit_cast(P, top);
    if (tid == 0) put_scale(static_cast<double>(amax));
    auto codes = [&](int c, const float(&f)[VEC]) {
        const int i = (c * THREADS + tid) * VEC;
        P p[VEC];
        products(c, f, p);
        Vec<int8_t, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; j++) out.v[j] = 0;
        if (finite && top != 0) quantise<VEC>(p, amax, out.v);
        if (i + VEC <= a.cols) {
            __builtin_memcpy(q + i, out.v, VEC);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (i + j < a.cols) q[i + j] = out.v[j];
        }
    };
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) codes(c, hv[c]);
    } else {
        for (int c = 0; c < chunks; c++) {
            // h is read back where it was stored: x may have been overwritten by it
            Raw raw;
            if (h) {
                const int i = (c * THREADS + tid) * VEC;
                // this thread's own elements: past them others may not have stored yet
#pragma unroll
                for (int j = 0; j < VEC; j++) hv[0][j] = i + j < a.cols ? static_cast<float>(h[i + j]) : 0.0f;
            } else {
                fetch(c, raw);
                sum_up(c, raw, hv[0]);
            }
            codes(c, hv[0]);
        }
    }
}

template <typename T, typename W>
int launch_rows(const RowArgs &a, void *stream) {
    const char *what = "rmsnorm_i8";
    auto go = [&](auto kernel, int threads) {
        const int rows = threads < 256 ? 256 / threads : 1;
        // a launch has fewer than 2^32 threads along an axis: up to 2^21 workgroups, then as many again
        const int64_t blocks = (a.rows + rows - 1) / rows, x = std::min<int64_t>(blocks, 1 << 21);
        return launch(what, kernel, dim3(static_cast<unsigned>(x), static_cast<unsigned>((blocks + x - 1) / x)),
                      dim3(threads < 256 ? 256 : threads), stream, a);
    };
    // a wave a row up to 1024 elements: no barrier; then as few threads as hold
    // the row in three runs of 8, since the statistics' join grows with them and
    // threads past the row's end take their part of the CU (1596 x 9233: 26 us
    // with 512 threads, 40 with 1024 and two runs)
    if (a.cols < 8) return go(rmsnorm_rows<T, W, 64, 1, 1, false>, 64);
    auto by_length = [&](auto tail) {
        constexpr bool TAIL = decltype(tail)::value;
        if (a.cols <= 64 * 8) return go(rmsnorm_rows<T, W, 64, 8, 1, TAIL>, 64);
        if (a.cols <= 64 * 16) return go(rmsnorm_rows<T, W, 64, 8, 2, TAIL>, 64);
        if (a.cols <= 256 * 8) return go(rmsnorm_rows<T, W, 256, 8, 1, TAIL>, 256);
        if (a.cols <= 256 * 16) return go(rmsnorm_rows<T, W, 256, 8, 2, TAIL>, 256);
        if (a.cols <= 256 * 24) return go(rmsnorm_rows<T, W, 256, 8, 3, TAIL>, 256);
        if (a.cols <= 512 * 16) return go(rmsnorm_rows<T, W, 512, 8, 2, TAIL>, 512);
        if (a.cols <= 512 * 24) return go(rmsnorm_rows<T, W, 512, 8, 3, TAIL>, 512);
        if (a.cols <= 1024 * 16) return go(rmsnorm_rows<T, W, 1024, 8, 2, TAIL>, 1024);
        return go(rmsnorm_rows<T, W, 1024, 8, 0, TAIL>, 1024);
    };
    return a.cols % 8 ? by_length(std::true_type{}) : by_length(std::false_type{});
}

struct DequantArgs {
    const int8_t *q;
    const float *scale;
    void *out;
    int64_t q_stride, out_stride, rows;
    int cols, runs;  // runs of VEC elements a row
};

// A workgroup takes 256 runs of VEC elements, one row's after the other's.
// TAIL: cols is no multiple of VEC; it is VEC at least.
template <typename T, int VEC, bool TAIL>
__global__ void __launch_bounds__(256) dequantize_rows(DequantArgs a) {
    const int64_t total = a.rows * a.runs;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total;
         t += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = t / a.runs;
        const int i = static_cast<int>(t - row * a.runs) * VEC;
        const float s = a.scale[row];
        float f[VEC];
        widen(load_vec<int8_t, VEC>(a.q + row * a.q_stride + min(i, a.cols - VEC)), f);
        if constexpr (TAIL) settle<VEC, true>(i, a.cols, f);
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] *= s;
        store_some<VEC>(static_cast<T *>(a.out) + row * a.out_stride + i, TAIL ? a.cols - i : VEC, f);
    }
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_rmsnorm_i8(const Spkv2RmsNormI8 *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("rmsnorm_i8: no arguments");
        if (!is_dtype(g->dtype)) return bad("rmsnorm_i8: unknown dtype");
        if (g->weight && g->weight_dtype != g->dtype && g->weight_dtype != SPKV2_DTYPE_FP32)
            return bad("rmsnorm_i8: weight_dtype is neither the rows' nor fp32");
        if (g->rows < 0 || g->cols < 0) return bad("rmsnorm_i8: negative size");
        if (!(g->eps >= 0.0f)) return bad("rmsnorm_i8: eps is negative or NaN");
        if (g->rows == 0) return 0;
        if (g->cols == 0) return bad("rmsnorm_i8: rows without columns");
        if (!g->x || !g->q || !g->scale) return bad("rmsnorm_i8: x, q or scale is NULL");
        if (g->rows > 1) {
            if (g->x_stride < g->cols || g->q_stride < g->cols || (g->residual && g->residual_stride < g->cols) ||
                (g->residual_out && g->residual_out_stride < g->cols))
                return bad("rmsnorm_i8: a stride is below cols");
        }
        if (g->cols > (1 << 24) || g->rows > INT32_MAX) return unsupported("rmsnorm_i8: more than 2^24 columns or 2^31 rows");
        const RowArgs a{g->x, g->residual, g->weight, g->residual_out, g->q, g->scale, g->rows, g->x_stride,
                        g->residual_stride, g->residual_out_stride, g->q_stride, static_cast<int>(g->cols), g->norm, g->eps};
        const bool wide = g->weight && g->weight_dtype == SPKV2_DTYPE_FP32;
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            return wide ? launch_rows<T, float>(a, stream) : launch_rows<T, T>(a, stream);
        });
    });
}

extern "C" int spkv2_mi355x_dequantize_i8(const Spkv2DequantizeI8 *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("dequantize_i8: no arguments");
        if (!is_dtype(g->dtype)) return bad("dequantize_i8: unknown dtype");
        if (g->rows < 0 || g->cols < 0) return bad("dequantize_i8: negative size");
        if (g->rows == 0 || g->cols == 0) return 0;
        if (!g->q || !g->scale || !g->out) return bad("dequantize_i8: q, scale or out is NULL");
        if (g->rows > 1 && (g->q_stride < g->cols || g->out_stride < g->cols)) return bad("dequantize_i8: a stride is below cols");
        if (g->cols > INT32_MAX || g->rows > INT32_MAX) return unsupported("dequantize_i8: more than 2^31 rows or columns");
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel, int run) {
                const DequantArgs a{g->q, g->scale, g->out, g->q_stride, g->out_stride, g->rows, static_cast<int>(g->cols),
                                    static_cast<int>((g->cols + run - 1) / run)};
                const int64_t blocks = (a.rows * a.runs + 255) / 256;
                return launch("dequantize_i8", kernel, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(256), stream, a);
            };
            // one 16-byte store a lane, neighbours' side by side
            constexpr int kRun = 16 / static_cast<int>(sizeof(T));
            if (g->cols < kRun) return go(dequantize_rows<T, 1, false>, 1);
            return g->cols % kRun ? go(dequantize_rows<T, kRun, true>, kRun) : go(dequantize_rows<T, kRun, false>, kRun);
        });
    });
}
