// Tokens sorted by expert, and their experts' rows weighted and added back.
//
// sort_tokens: the choices of one expert keep their order, so a choice's row is
// the count of choices of lower experts and of earlier ones of its own.  A
// workgroup an expert counts and places its own: every id is read once for each
// expert, from L2, but there is one launch, no atomics and no order that changes
// from run to run (65520 choices of 128 experts 14 us, 17.5 where ids come from
// memory: bound by the instructions for each 64 of them; 512 of 64 3.7 to 4.0 us).
//
// combine: bound by the bytes of the rows picked (8190 tokens of 8 rows of 2048,
// 302 MB: 65 us, 4.7 TB/s).
#include "decoder.hpp"

namespace spk::dec {

namespace {

struct SortArgs {
    const void *ids;
    int32_t *offsets, *order, *place;
    int count, experts;
};

// Four ids at p, of which `left` are there, as 16 bits each: 0xffff for those of no expert
template <typename I>
__device__ __forceinline__ void four_ids(const I *p, int left, unsigned experts, unsigned (&id)[4]) {
    I v[4];
    if (left >= 4) {
        __builtin_memcpy(v, p, sizeof(v));
    } else {
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = u < left ? p[u] : static_cast<I>(-1);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) id[u] = static_cast<uint64_t>(v[u]) < experts ? static_cast<unsigned>(v[u]) : 0xffffu;
}

// WAVES waves, each with a run of the choices, PIECE of them at a time: read four a
// lane, counted, and kept in LDS, which gives them back 64 in a row to be placed.
// An expert's workgroups (along y) count all choices and each place a part of every
// run: what they do for 64 choices, not the bytes, takes the time.
template <typename I, int WAVES, int PIECE>
__global__ void __launch_bounds__(64 * WAVES) sort_choices(SortArgs a) {
    constexpr int kBatches = PIECE / 256, kAhead = kBatches < 8 ? kBatches : 8;
    __shared__ __align__(16) uint16_t held[WAVES][PIECE];
    const unsigned e = blockIdx.x, experts = a.experts;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const I *ids = static_cast<const I *>(a.ids);
    const int batches = (a.count + 256 * WAVES - 1) / (256 * WAVES), per = batches * 256;  // counts up to 2^30
    const int first = min(wave * per, a.count), end = min(first + per, a.count);
    // the part of the run that is placed here
    const int parts = gridDim.y, part = blockIdx.y;
    const int from = min(first + static_cast<int>(static_cast<int64_t>(batches) * part / parts) * 256, end);
    const int to = min(first + static_cast<int>(static_cast<int64_t>(batches) * (part + 1) / parts) * 256, end);
    int lower = 0, own = 0, earlier = 0;  // earlier: of its own, ahead of the part
    const auto take = [&](int c0) {
#pragma unroll 1
        for (int b = 0; b < kBatches && c0 + 256 * b < end; b += kAhead) {
            unsigned id[kAhead][4];
#pragma unroll
            for (int n = 0; n < kAhead; n++) {
                const int c = c0 + 256 * (b + n) + 4 * lane;
                four_ids(ids + min(c, a.count), end - c, experts, id[n]);
            }
#pragma unroll
            for (int n = 0; n < kAhead; n++) {
                int mine = 0;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    lower += __popcll(__ballot(id[n][u] < e));
                    mine += __popcll(__ballot(id[n][u] == e));
                }
                own += mine;
                if (c0 + 256 * (b + n) < from) earlier += mine;
                *reinterpret_cast<uint2 *>(&held[wave][256 * (b + n) + 4 * lane]) = uint2{id[n][0] | id[n][1] << 16, id[n][2] | id[n][3] << 16};
            }
        }
    };
    for (int c0 = first; c0 < end; c0 += PIECE) take(c0);
    __shared__ int lowers[WAVES], owns[WAVES];
    if (lane == 0) {
        lowers[wave] = lower;
        owns[wave] = own;
    }
    __syncthreads();
    int row = earlier, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        row += lowers[w] + (w < wave ? owns[w] : 0);
        all += lowers[w] + owns[w];
    }
    if (threadIdx.x == 0 && part == 0) {
        a.offsets[e] = row;
        if (e == experts - 1) a.offsets[experts] = all;
    }
    if (own == 0 && e != 0) return;
    for (int c0 = first; c0 < end; c0 += PIECE) {
        if (c0 + PIECE <= from || c0 >= to) continue;
        if (per > PIECE) take(c0);  // a piece of several; the counts were used
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int c1 = max(c0, from); c1 < min(c0 + PIECE, to); c1 += 64) {
            const int c = c1 + lane;
            const unsigned id = c < end ? held[wave][c - c0] : 0xfffeu;
            const uint64_t mine = __ballot(id == e);
            if (mine) {  // few of 64 choices are one expert's
                if (id == e) {
                    const int r = row + static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mine >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mine), 0)));
                    a.order[r] = c;
                    a.place[c] = r;
                }
                row += __popcll(mine);
            }
            // the first expert's workgroups also mark the choices of none
            if (e == 0 && id == 0xffffu) a.place[c] = -1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

struct CombineArgs {
    const void *y, *residual;
    const int32_t *place;
    const float *weights;
    void *out;
    int64_t rows, tokens, y_stride, residual_stride, out_stride;
    int cols, per_token, runs;  // runs of VEC elements a row
};

// A run of VEC elements of a token a thread.  TAIL: cols is no multiple of VEC; it is VEC at least.
template <typename T, int VEC, bool TAIL>
__global__ void __launch_bounds__(256) combine_rows(CombineArgs a) {
    const int64_t total = a.tokens * a.runs;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total; t += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t token = t / a.runs;
        const int i = static_cast<int>(t - token * a.runs) * VEC, from = min(i, a.cols - VEC);
        float sum[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) sum[e] = 0.0f;
        if (a.residual) load_floats<VEC>(static_cast<const T *>(a.residual) + token * a.residual_stride + from, sum);
        const int32_t *place = a.place + token * a.per_token;
        const float *weights = a.weights + token * a.per_token;
        for (int j = 0; j < a.per_token; j += 4) {
            Vec<T, VEC> v[4];
            float w[4];
            bool there[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int at = min(j + u, a.per_token - 1);
                const int64_t row = place[at];
                w[u] = weights[at];
                there[u] = j + u < a.per_token && row >= 0 && row < a.rows;
                if (there[u]) v[u] = load_vec<T, VEC>(static_cast<const T *>(a.y) + row * a.y_stride + from);
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (there[u]) {
                    float f[VEC];
                    widen(v[u], f);
#pragma unroll
                    for (int e = 0; e < VEC; e++) sum[e] = __builtin_fmaf(w[u], f[e], sum[e]);
                }
        }
        if constexpr (TAIL) settle<VEC, true>(i, a.cols, sum);
        store_some<VEC>(static_cast<T *>(a.out) + token * a.out_stride + i, TAIL ? a.cols - i : VEC, sum);
    }
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_sort_tokens(const Spkv2SortTokens *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("sort_tokens: no arguments");
        if (g->tokens < 0 || g->per_token < 0 || g->experts < 1) return bad("sort_tokens: a negative size, or no expert");
        if (g->experts > 4096) return unsupported("sort_tokens: more than 4096 experts");
        if (g->per_token && g->tokens > (1 << 30) / g->per_token) return unsupported("sort_tokens: more than 2^30 choices");
        const int64_t count = g->tokens * g->per_token;
        if (!g->offsets || (count && (!g->ids || !g->order || !g->place))) return bad("sort_tokens: a NULL pointer");
        const SortArgs a{g->ids, g->offsets, g->order, g->place, static_cast<int>(count), g->experts};
        auto go = [&](auto kernel, int waves) {
            // as many workgroups as CUs where choices are many: one holds most of a CU's LDS
            const int parts = count <= 16384 ? 1 : std::max(1, std::min(256 / g->experts, 8));
            return launch("sort_tokens", kernel, dim3(g->experts, parts), dim3(64 * waves), stream, a);
        };
        auto by_count = [&](auto i) {
            using I = decltype(i);
            // fewer waves join their counts sooner
            return count <= 4096 ? go(sort_choices<I, 4, 1024>, 4) : count <= 16384 ? go(sort_choices<I, 16, 1024>, 16) : go(sort_choices<I, 16, 4096>, 16);
        };
        return g->wide_ids ? by_count(int64_t{}) : by_count(int32_t{});
    });
}

extern "C" int spkv2_mi355x_combine(const Spkv2Combine *g, void *stream) {
    return entry([&]() -> int {
        if (!g) return bad("combine: no arguments");
        if (!is_dtype(g->dtype)) return bad("combine: unknown dtype");
        if (g->rows < 0 || g->tokens < 0 || g->cols < 0) return bad("combine: negative size");
        if (g->per_token < 1) return bad("combine: per_token is below 1");
        if (g->tokens == 0 || g->cols == 0) return 0;
        if (!g->place || !g->weights || !g->out || (g->rows && !g->y)) return bad("combine: a NULL pointer");
        if ((g->rows > 1 && g->y_stride < g->cols) || (g->tokens > 1 && (g->out_stride < g->cols || (g->residual && g->residual_stride < g->cols))))
            return bad("combine: a stride is below cols");
        if (g->tokens > INT32_MAX || g->cols > INT32_MAX) return unsupported("combine: more than 2^31 tokens or columns");
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel, int run) {
                const CombineArgs a{g->y, g->residual, g->place, g->weights, g->out, g->rows, g->tokens, g->y_stride, g->residual_stride,
                                    g->out_stride, static_cast<int>(g->cols), g->per_token, static_cast<int>((g->cols + run - 1) / run)};
                const int64_t blocks = (a.tokens * a.runs + 255) / 256;
                return launch("combine", kernel, dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(256), stream, a);
            };
            constexpr int kRun = 16 / static_cast<int>(sizeof(T));
            if (g->cols < kRun) return go(combine_rows<T, 1, false>, 1);
            return g->cols % kRun ? go(combine_rows<T, kRun, true>, kRun) : go(combine_rows<T, kRun, false>, kRun);
        });
    });
}
