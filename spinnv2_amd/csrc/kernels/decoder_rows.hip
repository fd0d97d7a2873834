// Rows of a decoder layer in 8 bits: the residual's addition with a
// root-mean-square norm and int8 codes, and codes back to values.
//
//   h = x + r,  y = h w / sqrt(mean(h^2) + eps),  top = max|y|,
//   q = rint(127 y / top),  scale = top / 127
//
// The norm is one factor of the whole row, so it cancels out of q: the codes
// are those of p = h w, and only the scale needs the sum of squares.  Codes
// are therefore exact: of 16-bit rows p has at most 22 bits and is held in
// fp32, with an fp32 factor in it at most 48, held in fp64.
//
// One pass: a thread keeps its part of the row in registers between the
// statistics and the codes, so each input is read once and each output
// written once.  Bound by HBM.
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
// length, read again for the codes.
template <typename T, typename W, int THREADS, int VEC, int CHUNKS>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) rmsnorm_rows(RowArgs a) {
    using P = typename Product<T, W>::type;
    using U = decltype(abs_bits(P{}));
    constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (kRows > 1 ? threadIdx.x / THREADS : 0);
    if (kRows > 1 && row >= a.rows) return;
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
    auto load = [&](int c, float(&f)[VEC], bool store) {
        const int i = (c * THREADS + tid) * VEC;
        if (i >= a.cols) {
#pragma unroll
            for (int j = 0; j < VEC; j++) f[j] = 0.0f;
            return;
        }
        load_floats<VEC>(x + i, f);
        if (r) {
            float g[VEC];
            load_floats<VEC>(r + i, g);
#pragma unroll
            for (int j = 0; j < VEC; j++) f[j] = static_cast<float>(static_cast<T>(f[j] + g[j]));
        }
        if (h && store) store_floats<VEC>(h + i, f);
    };
    auto products = [&](int c, const float(&f)[VEC], P(&p)[VEC]) {
        const int i = (c * THREADS + tid) * VEC;
        float g[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) g[j] = 1.0f;
        if (w && i < a.cols) load_floats<VEC>(w + i, g);
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
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) load(c, hv[c], true);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) statistics(c, hv[c]);
    } else {
        for (int c = 0; c < chunks; c++) {
            load(c, hv[0], true);
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
    constexpr U kInf = sizeof(U) == 8 ? static_cast<U>(0x7ff0000000000000ull) : static_cast<U>(kInfBits);
    const bool finite = top < kInf;
    const P amax = __builtin_bit_cast(P, top);
    if (tid == 0) {
        double s = static_cast<double>(amax) / 127.0;
        if (a.norm) s /= sqrt(sum / a.cols + static_cast<double>(a.eps));
        // 0 of a row of zeros, whose norm may be 0 / 0
        a.scale[row] = !finite ? __builtin_nanf("") : top == 0 ? 0.0f : static_cast<float>(s);
    }
    auto codes = [&](int c, const float(&f)[VEC]) {
        const int i = (c * THREADS + tid) * VEC;
        P p[VEC];
        products(c, f, p);
        Vec<int8_t, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; j++) out.v[j] = 0;
        if (finite && top != 0) quantise<VEC>(p, amax, out.v);
        if (i < a.cols) *reinterpret_cast<Vec<int8_t, VEC> *>(q + i) = out;
    };
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) codes(c, hv[c]);
    } else {
        for (int c = 0; c < chunks; c++) {
            // h is read back where it was stored: x may have been overwritten by it
            const int i = (c * THREADS + tid) * VEC;
            if (!h) load(c, hv[0], false);
            else if (i < a.cols) load_floats<VEC>(h + i, hv[0]);
            codes(c, hv[0]);
        }
    }
}

template <typename T, typename W, int VEC>
int launch_rows(const RowArgs &a, void *stream) {
    const char *what = "rmsnorm_i8";
    auto go = [&](auto kernel, int threads) {
        const int rows = threads < 256 ? 256 / threads : 1;
        return launch(what, kernel, dim3(static_cast<unsigned>((a.rows + rows - 1) / rows)), dim3(threads < 256 ? 256 : threads),
                      stream, a);
    };
    constexpr int kOne = VEC == 1 ? 8 : 1;  // runs that hold as much as one of 8
    // a wave a row up to 1024 elements: no barrier; then as few threads as
    // hold the row in 8 runs of 8, since the statistics' join grows with them
    if (a.cols <= 64 * 8) return go(rmsnorm_rows<T, W, 64, VEC, kOne>, 64);
    if (a.cols <= 64 * 16) return go(rmsnorm_rows<T, W, 64, VEC, 2 * kOne>, 64);
    if (a.cols <= 256 * 8) return go(rmsnorm_rows<T, W, 256, VEC, kOne>, 256);
    if (a.cols <= 256 * 16) return go(rmsnorm_rows<T, W, 256, VEC, 2 * kOne>, 256);
    if (a.cols <= 512 * 16) return go(rmsnorm_rows<T, W, 512, VEC, 2 * kOne>, 512);
    if (a.cols <= 1024 * 16) return go(rmsnorm_rows<T, W, 1024, VEC, 2 * kOne>, 1024);
    return go(rmsnorm_rows<T, W, 1024, VEC, 0>, 1024);
}

struct DequantArgs {
    const int8_t *q;
    const float *scale;
    void *out;
    int64_t q_stride, out_stride, rows;
    int cols, runs;  // runs of VEC elements a row
};

// A workgroup takes 256 runs of VEC elements of one row after the other's.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) dequantize_rows(DequantArgs a) {
    const int64_t total = a.rows * a.runs;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total;
         t += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = t / a.runs;
        const int i = static_cast<int>(t - row * a.runs) * VEC;
        const float s = a.scale[row];
        const Vec<int8_t, VEC> c = *reinterpret_cast<const Vec<int8_t, VEC> *>(a.q + row * a.q_stride + i);
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = s * static_cast<float>(c.v[j]);
        store_floats<VEC>(static_cast<T *>(a.out) + row * a.out_stride + i, f);
    }
}

bool vec_rows(const void *p, int64_t stride, size_t size, int vec) {
    const size_t to = size * vec < 16 ? size * vec : 16;
    return aligned(p, to) && (stride * size) % to == 0;
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
        const size_t size = dtype_size(g->dtype);
        const RowArgs a{g->x, g->residual, g->weight, g->residual_out, g->q, g->scale, g->rows, g->x_stride,
                        g->residual_stride, g->residual_out_stride, g->q_stride, static_cast<int>(g->cols), g->norm, g->eps};
        const bool vec = g->cols % 8 == 0 && vec_rows(g->x, g->x_stride, size, 8) &&
                         (!g->residual || vec_rows(g->residual, g->residual_stride, size, 8)) &&
                         (!g->residual_out || vec_rows(g->residual_out, g->residual_out_stride, size, 8)) &&
                         (!g->weight || aligned(g->weight, 16)) && vec_rows(g->q, g->q_stride, 1, 8);
        const bool wide = g->weight && g->weight_dtype == SPKV2_DTYPE_FP32;
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            if (wide) return vec ? launch_rows<T, float, 8>(a, stream) : launch_rows<T, float, 1>(a, stream);
            return vec ? launch_rows<T, T, 8>(a, stream) : launch_rows<T, T, 1>(a, stream);
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
        const size_t size = dtype_size(g->dtype);
        auto vec = [&](int n) {
            return g->cols % n == 0 && vec_rows(g->q, g->q_stride, 1, n) && vec_rows(g->out, g->out_stride, size, n);
        };
        DequantArgs a{g->q, g->scale, g->out, g->q_stride, g->out_stride, g->rows, static_cast<int>(g->cols), 0};
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel, int n) {
                a.runs = a.cols / n;
                const int64_t blocks = (a.rows * a.runs + 255) / 256;
                return launch("dequantize_i8", kernel, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(256),
                              stream, a);
            };
            if (vec(16)) return go(dequantize_rows<T, 16>, 16);
            if (vec(4)) return go(dequantize_rows<T, 4>, 4);
            return go(dequantize_rows<T, 1>, 1);
        });
    });
}
