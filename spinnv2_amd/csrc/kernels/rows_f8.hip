// Rows in 8-bit floats (e4m3) with a scale for each block of 128 columns: of
// values, of a residual's addition with a root-mean-square norm, of a gated
// activation; and codes back to values.
//
//   q = e4m3(448 v / max|v|),  scale = max|v| / 448   over a block
//
// Eight elements a lane, so a block is 16 lanes, whose maximum is joined by lane
// moves.  The norm is one factor of the whole row and cancels out of q: codes
// are those of h w.  fp32 quotients beside a border of two codes are taken again
// in 64 bits, one in thirty thousand (of the gate, whose exponential is within
// 2^-21 in fp32, one in eight thousand), and so is the largest element of a block,
// for its scale, where fp32 does not hold values exactly.  One pass, bound by HBM and, of 16-bit rows, by their
// instructions: 8190 x 8192 of gates in bf16, 337 MB, in 75 to 79 us (4.3 to 4.5
// TB/s; 92 at the clocks that calls one behind the other leave, 88 with fp32 scales,
// off by a bit), of a norm with a residual, 470 MB, in 97 (4.9 TB/s), of values, 203
// MB, in 55, and back to values in 33 (the codes still cached); fp32 rows at 5.5 to
// 5.7 TB/s.
#include "decoder.hpp"

namespace spk::dec {

namespace {

struct RowsArgs {
    const void *x, *residual, *weight;
    void *h;
    uint8_t *q;
    float *scale;
    int64_t rows, x_stride, r_stride, h_stride, q_stride, s_stride;
    int cols, blocks;
    float eps;
    unsigned block_mul;  // n / blocks, by multiplication
    int block_shift;
};

enum Tail { kWhole, kPart, kShort };  // cols is a multiple of 8; is not; is below 8

// Elements i .. i + 8 of a row, zeros past its end
template <typename T, Tail TAIL>
__device__ __forceinline__ void run8(const T *row, int i, int cols, float (&f)[8]) {
    if constexpr (TAIL == kShort) {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = i + j < cols ? static_cast<float>(row[i + j]) : 0.0f;
    } else if constexpr (TAIL == kPart) {
        widen(load_vec<T, 8>(row + min(i, cols - 8)), f);
        settle<8, true>(i, cols, f);
    } else {
        unsigned words[2 * sizeof(T)];
        Vec<T, 8> x = load_vec<T, 8>(row + min(i, cols - 8));
        __builtin_memcpy(words, x.v, sizeof(words));
#pragma unroll
        for (unsigned &w : words) w = i < cols ? w : 0u;
        __builtin_memcpy(x.v, words, sizeof(words));
        widen(x, f);
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ double silu(double g) { return g / (1.0 + exp(-g)); }
// Within 2^-21: exp(-g) as 2^p (1 + rest ln 2) with p = -g log2 e rounded and what the rounding left, the hardware's
// power and reciprocal (a step of fp32 each).  Not below -80, where the power overflows.
__device__ __forceinline__ float silu(float g) {
    const float p = g * -1.44269504f, rest = __builtin_fmaf(g, -1.44269504f, -p) - g * 1.92596300e-8f;
    const float e = __builtin_amdgcn_exp2f(p);
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e * rest, 0.693147182f, e));
}

// What fp32 holds of a value: itself, its nearest, or what is within 2^-21 of it
enum Narrow { kSame, kNearest, kClose };

// f(index, a's, b's) of those of eight elements that `mask` has, one after the other
template <typename F>
__device__ __forceinline__ void each_of(unsigned mask, const float (&a)[8], const float (&b)[8], F &&f) {
    while (__any(mask != 0)) {
        if (mask) {
            const int at = __builtin_ctz(mask);
            mask &= mask - 1;
            float x = a[0], y = b[0];
#pragma unroll
            for (int j = 1; j < 8; j++) x = at == j ? a[j] : x, y = at == j ? b[j] : y;
            f(at, x, y);
        }
    }
}

// The codes and the scale (times `norm`) of a block's 16 lanes with values v, which
// wide(a[j], b[j]) gives in 64 bits (and which may not be 0 where v is, unless a or b
// is).  The scale is the largest value's in 64 bits: the element that fp32 says is the
// largest, and those so near it that fp32 may be wrong, are taken again, the first
// such of each lane by all lanes at once.  All lanes of a wave come here together;
// `left` of the lane's elements are there, `first` lanes write their block's scale.
template <Narrow NARROW, typename Wide>
__device__ __forceinline__ void put_block(const float (&v)[8], const float (&a)[8], const float (&b)[8], Wide &&wide, double norm, uint8_t *q, int left, float *scale,
                                          bool first) {
    using F = F8<NARROW == kClose ? 18 : 20>;
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, abs_bits(v[j]));
    top = max_over<16>(top);
    unsigned code[2] = {0, 0};
    const float amax = __uint_as_float(top);
    const bool plain = F::plain(amax);
    bool near = false;
    if (top) {
        near = F::quantise(v, amax, code);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) near |= a[j] != 0.0f && b[j] != 0.0f;
    }
    double most = NARROW == kSame ? amax : 0.0;  // of this lane
    const auto raise = [&](int, float x, float y) {
        const double f = fabs(wide(x, y));
        most = f > most ? f : f == f ? most : __builtin_inf();
    };
    if constexpr (NARROW != kSame) {
        // in fp32 the largest is within 2^-20, 16 steps at most, of what fp32 says is the largest
        const float bound = __uint_as_float(NARROW == kClose ? top - 32 : top);
        float x = 0.0f, y = 0.0f;
        int count = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const bool is = fabsf(v[j]) >= bound;
            x = is ? a[j] : x, y = is ? b[j] : y;
            count += is;
        }
        if (plain && count) raise(0, x, y);
        if (__any(plain && count > 1)) {
            unsigned mask = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) mask |= plain && fabsf(v[j]) >= bound ? 1u << j : 0u;
            each_of(mask, a, b, raise);
        }
    }
    if (__any(!plain)) {
        unsigned mask = 0;
        if (!plain) {
            most = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j++) mask |= v[j] != 0.0f || (a[j] != 0.0f && b[j] != 0.0f) ? 1u << j : 0u;
        }
        each_of(mask, a, b, raise);
    }
    if (__any(near)) {
        const double all = max_over16(most);
        unsigned mask = 0;
        if (near) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (F::beside(v[j], amax)) mask |= 1u << j;
        }
        each_of(mask, a, b, [&](int at, float x, float y) {
            const double f = wide(x, y);
            unsigned c = 0;
            if (all < __builtin_inf() && all > 0.0) c = exact_code_f8<NARROW != kClose>(fabs(f), all) | (__builtin_signbit(f) ? 0x80u : 0u);
            const int shift = 8 * (at % 4);
            const unsigned is = at < 4 ? code[0] : code[1], put = (is & ~(0xffu << shift)) | c << shift;
            code[0] = at < 4 ? put : code[0];
            code[1] = at < 4 ? code[1] : put;
        });
    }
    if (left >= 8) {
        __builtin_memcpy(q, code, 8);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < left) q[j] = static_cast<uint8_t>(code[j / 4] >> (8 * (j % 4)));
    }
    // The largest of the lanes' scales, as bits: none is below 0, and NaN is above all.  0 of a block of zeros, also where its
    // norm is infinite, but not where its row holds a NaN and so has no norm.
    const float own = !(most < __builtin_inf()) || norm != norm ? __builtin_nanf("") : most == 0.0 ? 0.0f : static_cast<float>(most * (norm * (1.0 / 448.0)));
    const unsigned bits = max_over<16>(abs_bits(own));
    if (first) *scale = __uint_as_float(bits);
}

// Blocks of values or gates, 16 of them a workgroup, one row's after the other's
template <typename T, bool GATE, Tail TAIL>
__global__ void __launch_bounds__(256) quantise_blocks(RowsArgs a) {
    const unsigned at = blockIdx.x * 16 + threadIdx.x / 16;
    const unsigned row = static_cast<unsigned>((static_cast<uint64_t>(at) * a.block_mul) >> a.block_shift);
    const bool in = row < a.rows;
    const int64_t r = in ? row : a.rows - 1;
    const int block = in ? static_cast<int>(at - row * a.blocks) : 0, i = block * 128 + threadIdx.x % 16 * 8;
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
    float v[8];
    run8<T, TAIL>(x, i, a.cols, v);
    const auto put = [&](const float(&t)[8], const float(&up)[8], auto &&wide) {
        put_block<GATE ? kClose : kSame>(v, t, up, wide, 1.0, a.q + r * a.q_stride + i, in ? a.cols - i : 0, a.scale + r * a.s_stride + block,
                                         in && threadIdx.x % 16 == 0);
    };
    if constexpr (GATE) {
        float t[8], up[8], s[8], lowest = 0.0f;
        unsigned most = 0, least = ~0u;
        run8<T, TAIL>(x + a.cols, i, a.cols, up);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            t[j] = v[j];
            s[j] = silu(t[j]);
            v[j] = s[j] * up[j];
            most = max(most, abs_bits(v[j]));
            least = min(least, abs_bits(s[j]));
            lowest = fminf(lowest, t[j]);
        }
        // where fp32's exponential, quotient (whose bits a large factor would show) or product leaves its range, 64 bits
        // say what the value is
        if (most >= __float_as_uint(0x1p120f) || least < __float_as_uint(0x1p-125f) || lowest < -80.0f) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (!(fabsf(v[j]) < 0x1p120f) || t[j] < -80.0f || (fabsf(s[j]) < 0x1p-125f && t[j] != 0.0f && up[j] != 0.0f)) v[j] = __builtin_inff();
        }
        put(t, up, [](float t, float up) { return silu(static_cast<double>(t)) * static_cast<double>(up); });
    } else {
        put(v, v, [](float x, float) { return static_cast<double>(x); });
    }
}

// THREADS threads a row (a wave: several rows a workgroup), each with CHUNKS
// runs of 8 neighbouring elements in registers; CHUNKS = 0: rows of any length,
// read again for the codes.
template <typename T, typename W, int THREADS, int CHUNKS, Tail TAIL>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) norm_blocks(RowsArgs a) {
    constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
    const int64_t row = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kRows + (kRows > 1 ? threadIdx.x / THREADS : 0);
    if (row >= a.rows) return;  // whole waves, or workgroups
    const int tid = kRows > 1 ? threadIdx.x % THREADS : threadIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.r_stride : nullptr;
    T *h = a.h ? static_cast<T *>(a.h) + row * a.h_stride : nullptr;
    const W *w = static_cast<const W *>(a.weight);
    const int chunks = (a.cols + THREADS * 8 - 1) / (THREADS * 8);
    double sum = 0.0;
    const auto run = [&](int c, float(&f)[8]) {
        const int i = (c * THREADS + tid) * 8;
        run8<T, TAIL>(x, i, a.cols, f);
        if (r) {
            float g[8];
            run8<T, TAIL>(r, i, a.cols, g);
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = static_cast<float>(static_cast<T>(f[j] + g[j]));
        }
    };
    const auto keep = [&](int c, const float(&f)[8]) {
        const int i = (c * THREADS + tid) * 8;
        if (h && i < a.cols) store_some<8>(h + i, a.cols - i, f);
    };
    const auto squares = [&](const float(&f)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) sum = __builtin_fma(static_cast<double>(f[j]), static_cast<double>(f[j]), sum);
    };
    float hv[CHUNKS ? CHUNKS : 1][8];
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) run(c, hv[c]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) keep(c, hv[c]);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) squares(hv[c]);
    } else {
        for (int c = 0; c < chunks; c++) {
            run(c, hv[0]);
            keep(c, hv[0]);
            squares(hv[0]);
        }
    }
    sum = wave_sum(sum);
    if constexpr (THREADS > kWave) {
        __shared__ double sums[THREADS / kWave];
        if ((tid & (kWave - 1)) == 0) sums[tid / kWave] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < THREADS / kWave; i++) sum += sums[i];
    }
    const double norm = 1.0 / sqrt(sum / a.cols + static_cast<double>(a.eps));
    const auto codes = [&](int c, const float(&f)[8]) {
        const int i = (c * THREADS + tid) * 8;
        float g[8], v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) g[j] = 1.0f;
        if (w) run8<W, TAIL>(w, i, a.cols, g);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = f[j] * g[j];
        // products of two 16-bit values are exact in fp32
        constexpr Narrow kNarrow = sizeof(T) == 2 && sizeof(W) == 2 ? kSame : kNearest;
        put_block<kNarrow>(v, f, g, [](float x, float y) { return static_cast<double>(x) * static_cast<double>(y); }, norm, a.q + row * a.q_stride + i, a.cols - i,
                           a.scale + row * a.s_stride + i / 128, tid % 16 == 0 && i < a.cols);
    };
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) codes(c, hv[c]);
    } else {
        for (int c = 0; c < chunks; c++) {
            // h is read back where it was stored: x may have been overwritten by it
            if (h) {
                const int i = (c * THREADS + tid) * 8;
                // this thread's own elements: past them others may not have stored yet
#pragma unroll
                for (int j = 0; j < 8; j++) hv[0][j] = i + j < a.cols ? static_cast<float>(h[i + j]) : 0.0f;
            } else {
                run(c, hv[0]);
            }
            codes(c, hv[0]);
        }
    }
}

template <typename T, typename W>
int launch_norm(const RowsArgs &a, void *stream) {
    auto go = [&](auto kernel, int threads) {
        const int rows = threads < 256 ? 256 / threads : 1;
        // a launch has fewer than 2^32 threads along an axis: up to 2^21 workgroups, then as many again
        const int64_t blocks = (a.rows + rows - 1) / rows, x = std::min<int64_t>(blocks, 1 << 21);
        return launch("rmsnorm_f8", kernel, dim3(static_cast<unsigned>(x), static_cast<unsigned>((blocks + x - 1) / x)),
                      dim3(threads < 256 ? 256 : threads), stream, a);
    };
    if (a.cols < 8) return go(norm_blocks<T, W, 64, 1, kShort>, 64);
    auto by_length = [&](auto tail) {
        constexpr Tail TAIL = decltype(tail)::value ? kPart : kWhole;
        // as in the int8 rows: a wave a row up to 1024 elements, then as few threads as hold it in three runs of 8
        if (a.cols <= 64 * 8) return go(norm_blocks<T, W, 64, 1, TAIL>, 64);
        if (a.cols <= 64 * 16) return go(norm_blocks<T, W, 64, 2, TAIL>, 64);
        if (a.cols <= 256 * 8) return go(norm_blocks<T, W, 256, 1, TAIL>, 256);
        if (a.cols <= 256 * 16) return go(norm_blocks<T, W, 256, 2, TAIL>, 256);
        if (a.cols <= 256 * 24) return go(norm_blocks<T, W, 256, 3, TAIL>, 256);
        if (a.cols <= 512 * 16) return go(norm_blocks<T, W, 512, 2, TAIL>, 512);
        if (a.cols <= 512 * 24) return go(norm_blocks<T, W, 512, 3, TAIL>, 512);
        if (a.cols <= 1024 * 16) return go(norm_blocks<T, W, 1024, 2, TAIL>, 1024);
        return go(norm_blocks<T, W, 1024, 0, TAIL>, 1024);
    };
    return a.cols % 8 ? by_length(std::true_type{}) : by_length(std::false_type{});
}

template <typename T, bool GATE>
int launch_blocks(const RowsArgs &a, void *stream) {
    const unsigned grid = static_cast<unsigned>((a.rows * a.blocks + 15) / 16);
    auto go = [&](auto kernel) { return launch(GATE ? "gate_f8" : "quantize_f8", kernel, dim3(grid), dim3(256), stream, a); };
    if (a.cols < 8) return go(quantise_blocks<T, GATE, kShort>);
    return a.cols % 8 ? go(quantise_blocks<T, GATE, kPart>) : go(quantise_blocks<T, GATE, kWhole>);
}

struct DequantArgs {
    const uint8_t *q;
    const float *scale;
    void *out;
    int64_t q_stride, s_stride, out_stride, rows;
    int cols, runs;  // runs of VEC elements a row
};

// N (4 or 8) codes as floats
template <int N>
__device__ __forceinline__ void from_f8(const Vec<uint8_t, N> &x, float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        const int u = static_cast<int>(x.v[j] | x.v[j + 1] << 8 | x.v[j + 2] << 16 | static_cast<unsigned>(x.v[j + 3]) << 24);
        f[j] = __builtin_amdgcn_cvt_f32_fp8(u, 0);
        f[j + 1] = __builtin_amdgcn_cvt_f32_fp8(u, 1);
        f[j + 2] = __builtin_amdgcn_cvt_f32_fp8(u, 2);
        f[j + 3] = __builtin_amdgcn_cvt_f32_fp8(u, 3);
    }
}

// A workgroup takes 256 runs of VEC elements, one row's after the other's.
// TAIL: cols is no multiple of VEC; it is VEC at least.
template <typename T, int VEC, bool TAIL>
__global__ void __launch_bounds__(256) dequantise_blocks(DequantArgs a) {
    const int64_t total = a.rows * a.runs;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total; t += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = t / a.runs;
        const int i = static_cast<int>(t - row * a.runs) * VEC;
        const float s = a.scale[row * a.s_stride + i / 128];
        const uint8_t *q = a.q + row * a.q_stride + min(i, a.cols - VEC);
        float f[VEC];
        if constexpr (VEC == 1) {
            f[0] = __builtin_amdgcn_cvt_f32_fp8(*q, 0);
        } else {
            from_f8(load_vec<uint8_t, VEC>(q), f);
            if constexpr (TAIL) settle<VEC, true>(i, a.cols, f);
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] *= s;
        store_some<VEC>(static_cast<T *>(a.out) + row * a.out_stride + i, TAIL ? a.cols - i : VEC, f);
    }
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_rows_f8(const Spkv2RowsF8 *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("rows_f8: no arguments");
        if (!is_dtype(g->dtype)) return bad("rows_f8: unknown dtype");
        if (g->kind < SPKV2_F8_VALUES || g->kind > SPKV2_F8_GATE) return bad("rows_f8: unknown kind");
        const bool norm = g->kind == SPKV2_F8_NORM;
        if (!norm && (g->residual || g->weight || g->residual_out)) return bad("rows_f8: a residual or weight without the norm");
        if (g->weight && g->weight_dtype != g->dtype && g->weight_dtype != SPKV2_DTYPE_FP32)
            return bad("rows_f8: weight_dtype is neither the rows' nor fp32");
        if (g->rows < 0 || g->cols < 0) return bad("rows_f8: negative size");
        if (norm && !(g->eps >= 0.0f)) return bad("rows_f8: eps is negative or NaN");
        if (g->rows == 0) return 0;
        if (g->cols == 0) return bad("rows_f8: rows without columns");
        if (!g->x || !g->q || !g->scale) return bad("rows_f8: x, q or scale is NULL");
        const int64_t blocks = (g->cols + SPKV2_F8_BLOCK - 1) / SPKV2_F8_BLOCK;
        if (g->rows > 1) {
            if (g->x_stride < (g->kind == SPKV2_F8_GATE ? 2 : 1) * g->cols || g->q_stride < g->cols || (g->residual && g->residual_stride < g->cols) ||
                (g->residual_out && g->residual_out_stride < g->cols))
                return bad("rows_f8: a stride is below cols");
            if (g->scale_stride < blocks) return bad("rows_f8: the scales' stride is below their count");
        }
        if (g->cols > (1 << 24) || g->rows > INT32_MAX) return unsupported("rows_f8: more than 2^24 columns or 2^31 rows");
        // 16 blocks a workgroup of 256; a launch has fewer than 2^32 threads along an axis
        if (!norm && (g->rows * blocks + 15) / 16 >= 1 << 24) return unsupported("rows_f8: more than 2^28 - 16 blocks");
        RowsArgs a{g->x, g->residual, g->weight, g->residual_out, g->q, g->scale, g->rows, g->x_stride, g->residual_stride,
                   g->residual_out_stride, g->q_stride, g->scale_stride, static_cast<int>(g->cols), static_cast<int>(blocks), g->eps, 0, 0};
        div_magic(static_cast<unsigned>(blocks), &a.block_mul, &a.block_shift);
        const bool wide = g->weight && g->weight_dtype == SPKV2_DTYPE_FP32;
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            if (norm) return wide ? launch_norm<T, float>(a, stream) : launch_norm<T, T>(a, stream);
            return g->kind == SPKV2_F8_GATE ? launch_blocks<T, true>(a, stream) : launch_blocks<T, false>(a, stream);
        });
    });
}

extern "C" int spkv2_mi355x_dequantize_f8(const Spkv2DequantizeF8 *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("dequantize_f8: no arguments");
        if (!is_dtype(g->dtype)) return bad("dequantize_f8: unknown dtype");
        if (g->rows < 0 || g->cols < 0) return bad("dequantize_f8: negative size");
        if (g->rows == 0 || g->cols == 0) return 0;
        if (!g->q || !g->scale || !g->out) return bad("dequantize_f8: q, scale or out is NULL");
        if (g->rows > 1 && (g->q_stride < g->cols || g->out_stride < g->cols)) return bad("dequantize_f8: a stride is below cols");
        if (g->rows > 1 && g->scale_stride < (g->cols + SPKV2_F8_BLOCK - 1) / SPKV2_F8_BLOCK)
            return bad("dequantize_f8: the scales' stride is below their count");
        if (g->cols > (1 << 24) || g->rows > INT32_MAX) return unsupported("dequantize_f8: more than 2^24 columns or 2^31 rows");
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel, int run) {
                const DequantArgs a{g->q, g->scale, g->out, g->q_stride, g->scale_stride, g->out_stride, g->rows, static_cast<int>(g->cols),
                                    static_cast<int>((g->cols + run - 1) / run)};
                const int64_t blocks = (a.rows * a.runs + 255) / 256;
                return launch("dequantize_f8", kernel, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(256), stream, a);
            };
            // one 16-byte store a lane, neighbours' side by side
            constexpr int kRun = 16 / static_cast<int>(sizeof(T));
            if (g->cols < kRun) return go(dequantise_blocks<T, 1, false>, 1);
            return g->cols % kRun ? go(dequantise_blocks<T, kRun, true>, kRun) : go(dequantise_blocks<T, kRun, false>, kRun);
        });
    });
}
