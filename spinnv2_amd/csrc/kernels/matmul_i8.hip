// Product of int8 rows and int8 weights with a scale for each token and each
// output channel:
//
//   out[m, n] = sa[m] sb[n] sum_k a[m, k] b[n, k] + bias[n]
//
// int32 sums on the int8 matrix cores, exact whatever their order (127^2 2^17
// < 2^31), scaled in fp32 and rounded once.
#include "decoder.hpp"

namespace spk::dec {

namespace {

typedef int intx16 __attribute__((ext_vector_type(16)));

struct MatmulArgs {
    const int8_t *a, *b;
    const float *a_scale, *b_scale, *bias;
    void *out;
    int64_t a_stride, b_stride, out_stride;
    int m, n, k;
};

// 16 bytes at p, of which `left` are inside the row: zeros past them
__device__ __forceinline__ intx4 load16(const int8_t *p, int left) {
    intx4 v = {0, 0, 0, 0};
    if (left >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (left > 0) {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < left) v[i / 4] |= static_cast<int>(static_cast<unsigned>(static_cast<uint8_t>(p[i])) << (8 * (i % 4)));
    }
    return v;
}

// BM tokens x BN channels a workgroup of four waves (2 x 2), BK bytes of k a
// step through LDS, the next step's in registers meanwhile.
template <typename T, int BM, int BN, int BK>
__global__ void __launch_bounds__(256) matmul_tiles(MatmulArgs a) {
    constexpr int kPitch = BK + 16;  // an odd multiple of 16 bytes: eight rows' 16-byte pieces on different banks
    constexpr int TM = BM / 64, TN = BN / 64;
    constexpr int kRowChunks = BK / 16;
    constexpr int kA = BM * kRowChunks / 256, kB = BN * kRowChunks / 256;
    __shared__ __align__(16) int8_t lds[(BM + BN) * kPitch];
    int8_t *la = lds, *lb = lds + BM * kPitch;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    intx16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0;
    intx4 ra[kA], rb[kB];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int c = 0; c < kA; c++) {
            const int p = c * 256 + tid, row = m0 + p / kRowChunks, k = k0 + (p % kRowChunks) * 16;
            ra[c] = load16(a.a + static_cast<int64_t>(row) * a.a_stride + k, row < a.m ? a.k - k : 0);
        }
#pragma unroll
        for (int c = 0; c < kB; c++) {
            const int p = c * 256 + tid, row = n0 + p / kRowChunks, k = k0 + (p % kRowChunks) * 16;
            rb[c] = load16(a.b + static_cast<int64_t>(row) * a.b_stride + k, row < a.n ? a.k - k : 0);
        }
    };
    fetch(0);
    for (int k0 = 0; k0 < a.k; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kA; c++) {
            const int p = c * 256 + tid;
            *reinterpret_cast<intx4 *>(la + (p / kRowChunks) * kPitch + (p % kRowChunks) * 16) = ra[c];
        }
#pragma unroll
        for (int c = 0; c < kB; c++) {
            const int p = c * 256 + tid;
            *reinterpret_cast<intx4 *>(lb + (p / kRowChunks) * kPitch + (p % kRowChunks) * 16) = rb[c];
        }
        __syncthreads();
        if (k0 + BK < a.k) fetch(k0 + BK);
#pragma unroll
        for (int kk = 0; kk < BK; kk += 32) {
            intx4 fa[TM], fb[TN];
#pragma unroll
            for (int j = 0; j < TM; j++)
                fa[j] = *reinterpret_cast<const intx4 *>(la + (wm + j * 32 + lane % 32) * kPitch + kk + lane / 32 * 16);
#pragma unroll
            for (int i = 0; i < TN; i++)
                fb[i] = *reinterpret_cast<const intx4 *>(lb + (wn + i * 32 + lane % 32) * kPitch + kk + lane / 32 * 16);
#pragma unroll
            for (int i = 0; i < TN; i++)
#pragma unroll
                for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[i], fa[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < TM; j++) {
        const int m = m0 + wm + j * 32 + lane % 32;
        if (m >= a.m) continue;
        const float sa = a.a_scale[m];
        T *out = static_cast<T *>(a.out) + static_cast<int64_t>(m) * a.out_stride;
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int n = n0 + wn + i * 32 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
                if (n >= a.n) continue;
                float v = static_cast<float>(acc[i][j][r]) * sa * a.b_scale[n];
                if (a.bias) v += a.bias[n];
                out[n] = static_cast<T>(v);
            }
    }
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_matmul_i8(const Spkv2MatmulI8 *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("matmul_i8: no arguments");
        if (!is_dtype(g->dtype)) return bad("matmul_i8: unknown dtype");
        if (g->m < 0 || g->n < 0 || g->k < 0) return bad("matmul_i8: negative size");
        if (g->m == 0 || g->n == 0) return 0;
        if (!g->out || !g->a_scale || !g->b_scale || (g->k && (!g->a || !g->b))) return bad("matmul_i8: a NULL pointer");
        if ((g->m > 1 && (g->a_stride < g->k || g->out_stride < g->n)) || (g->n > 1 && g->b_stride < g->k))
            return bad("matmul_i8: a stride is below its row's length");
        if (g->k > (1 << 17)) return unsupported("matmul_i8: k above 2^17, whose sums may pass 32 bits");
        if (g->m > (1 << 22) || g->n > (1 << 30)) return unsupported("matmul_i8: m above 2^22 or n above 2^30");
        const MatmulArgs a{g->a, g->b, g->a_scale, g->b_scale, g->bias, g->out, g->a_stride, g->b_stride, g->out_stride,
                           static_cast<int>(g->m), static_cast<int>(g->n), static_cast<int>(g->k)};
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            const dim3 grid(static_cast<unsigned>((g->n + 63) / 64), static_cast<unsigned>((g->m + 63) / 64));
            return launch("matmul_i8", matmul_tiles<T, 64, 64, 64>, grid, dim3(256), stream, a);
        });
    });
}
