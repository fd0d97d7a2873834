// Norms of queries and keys head by head, the rotation of their positions, and
// the way of keys and values into a paged int8 cache, in one pass.
//
//   y = x w / sqrt(mean(x^2) + eps),  (y_i, y_j) -> (y_i cos - y_j sin, y_j cos + y_i sin)
//
// A wave takes a token, or some of a token's heads where tokens are few: its 64
// lanes take the sines and cosines of the pairs, which every head of the token
// turns by, and groups of 8, 16 or 32 lanes a head each, 8 elements a lane.
//
// In 64 bits: angles of far positions need it (position 70001 times a frequency
// near 1 keeps 7 bits behind the point in fp32), and a key beside the border of
// two bf16 values or two codes falls on its own side.  The vector units take
// 64-bit products at the rate of 32-bit ones.
#include "decoder.hpp"

namespace spk::dec {

namespace {

struct RotateArgs {
    Spkv2Rotate g;
    Spkv2KvCacheI8 c;  // with no pages: none
    int parts;         // waves a token
    unsigned page_mul;  // slot / page_size, by multiplication; 0: slots pass 2^31
    int page_shift;
};

// sin and cos of an angle below 2^40: the angle less the nearest multiple n of
// pi/2, which is held in two doubles, leaves |r| <= pi/4, whose Taylor series
// are within 2^-52 with the terms up to r^15 and r^16; n mod 4 turns them.
__device__ __forceinline__ void sine_cosine(double angle, double *s, double *c) {
    const double n = rint(angle * 0.63661977236758134308);
    double r = __builtin_fma(n, -1.57079632679489655800, angle);
    r = __builtin_fma(n, -6.12323399573676603587e-17, r);
    const double r2 = r * r;
    double a = -1.0 / 1307674368000.0;
    a = __builtin_fma(a, r2, 1.0 / 6227020800.0);
    a = __builtin_fma(a, r2, -1.0 / 39916800.0);
    a = __builtin_fma(a, r2, 1.0 / 362880.0);
    a = __builtin_fma(a, r2, -1.0 / 5040.0);
    a = __builtin_fma(a, r2, 1.0 / 120.0);
    a = __builtin_fma(a, r2, -1.0 / 6.0);
    const double sine = __builtin_fma(a * r2, r, r);
    double b = 1.0 / 20922789888000.0;
    b = __builtin_fma(b, r2, -1.0 / 87178291200.0);
    b = __builtin_fma(b, r2, 1.0 / 479001600.0);
    b = __builtin_fma(b, r2, -1.0 / 3628800.0);
    b = __builtin_fma(b, r2, 1.0 / 40320.0);
    b = __builtin_fma(b, r2, -1.0 / 720.0);
    b = __builtin_fma(b, r2, 1.0 / 24.0);
    b = __builtin_fma(b, r2, -0.5);
    const double cosine = __builtin_fma(b, r2, 1.0);
    const double turn = n - 4.0 * floor(n * 0.25);  // 0, 1, 2 or 3
    const bool swap = turn == 1.0 || turn == 3.0;
    *s = swap ? cosine : sine;
    *c = swap ? sine : cosine;
    if (turn >= 2.0) *s = -*s;
    if (turn == 1.0 || turn == 2.0) *c = -*c;
}

// A double from the lane that the DPP control names, by two 32-bit moves
template <int CONTROL>
__device__ __forceinline__ double moved(double v) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    const unsigned lo = static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(u), CONTROL, 0xF, 0xF, true));
    const unsigned hi = static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(u >> 32), CONTROL, 0xF, 0xF, true));
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
// The sum over groups of LANES neighbouring lanes, in each of them
template <int LANES>
__device__ __forceinline__ double sum_over(double v) {
    v += moved<0xB1>(v);   // lanes 1 0 3 2
    v += moved<0x4E>(v);   // lanes 2 3 0 1
    v += moved<0x141>(v);  // eight lanes mirrored
    if constexpr (LANES >= 16) v += moved<0x140>(v);  // 16 mirrored
    if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
    return v;
}

// What a lane's 8 elements are multiplied by, and their partners: y = norm (x own + partner other)
struct Turn {
    double own[8], other[8];
};

// PAIRED: a lane's elements have their partners in one lane: pairs side by side, or a multiple of 8 apart
template <typename T, typename W, int LANES, bool PAIRED>
__global__ void __launch_bounds__(256) rotate_heads(RotateArgs a) {
    constexpr int kGroups = 64 / LANES, kDim = LANES * 8;
    __shared__ __align__(16) double table[4][2][128];
    __shared__ __align__(32) float heads[4][kGroups][kDim];
    const Spkv2Rotate &g = a.g;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    const int64_t token = at / a.parts;
    const int part = static_cast<int>(at - token * a.parts);
    if (token >= g.tokens) return;  // a whole wave; no barrier follows
    const int dim = g.head_dim, pairs = g.pairs;
    const int group = lane / LANES, i0 = lane % LANES * 8;
    const bool in = i0 < dim;
    double *sines = table[wave][0], *cosines = table[wave][1];
    for (int p = lane; p < pairs; p += 64) {
        const int axis = g.axis ? g.axis[p] : 0;
        const int position = static_cast<unsigned>(axis) < static_cast<unsigned>(g.axes) ? g.positions[token * g.position_stride + axis] : 0;
        sine_cosine(static_cast<double>(position) * static_cast<double>(g.frequencies[p]), &sines[p], &cosines[p]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();

    // where element i of a head has its partner, and with which factors
    const auto pair_of = [&](int i, bool *second) {
        if (g.interleaved) {
            *second = i & 1;
            return i / 2;
        }
        *second = i >= pairs;
        return *second ? i - pairs : i;
    };
    const auto partner_of = [&](int i) { return i >= 2 * pairs || !in ? i : g.interleaved ? i ^ 1 : i >= pairs ? i - pairs : i + pairs; };
    const auto turn_of = [&](const void *weight) {
        Turn t;
        const W *w = static_cast<const W *>(weight);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j;
            bool second;
            const int p = pair_of(i, &second);
            t.own[j] = 1.0;
            t.other[j] = 0.0;
            if (in && i < 2 * pairs) {
                t.own[j] = cosines[p];
                t.other[j] = second ? sines[p] : -sines[p];
            }
            if (in && w && g.norm) {
                t.own[j] *= static_cast<double>(static_cast<float>(w[i]));
                t.other[j] *= static_cast<double>(static_cast<float>(w[partner_of(i)]));
            }
        }
        return t;
    };
    float *mine = heads[wave][group];
    const auto turned = [&](const Turn &t, const float(&x)[8], float(&y)[8]) {
        double factor = 1.0;
        if (g.norm) {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j++) sum = __builtin_fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum);
            factor = 1.0 / sqrt(sum_over<LANES>(sum) / dim + static_cast<double>(g.eps));
        }
        float other[8];
        if (PAIRED && g.interleaved) {
#pragma unroll
            for (int j = 0; j < 8; j++) other[j] = x[j ^ 1];
        } else {
            put_floats<8>(mine + i0, x);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if constexpr (PAIRED) {
                const Vec<float, 8> v = *reinterpret_cast<const Vec<float, 8> *>(mine + partner_of(i0));
#pragma unroll
                for (int j = 0; j < 8; j++) other[j] = v.v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) other[j] = mine[partner_of(i0 + j)];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            // a partner that is not there, or is not finite where nothing turns, adds nothing
            double v = static_cast<double>(x[j]) * t.own[j];
            if (i0 + j < 2 * pairs) v = __builtin_fma(static_cast<double>(other[j]), t.other[j], v);
            y[j] = static_cast<float>(static_cast<T>(v * factor));
        }
    };
    const auto fetch = [&](const void *x, int64_t stride, int head, float(&f)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = 0.0f;
        if (in) load_floats<8>(static_cast<const T *>(x) + token * stride + static_cast<int64_t>(head) * dim + i0, f);
    };
    const auto put = [&](void *y, int64_t stride, int head, const float(&f)[8]) {
        if (in) store_floats<8>(static_cast<T *>(y) + token * stride + static_cast<int64_t>(head) * dim + i0, f);
    };
    const int first = part * kGroups, step = a.parts * kGroups;
    if (g.heads > first) {
        const Turn t = turn_of(g.q_weight);
        for (int h = first; h < g.heads; h += step) {
            const int head = min(h + group, g.heads - 1);
            float x[8], y[8];
            fetch(g.q, g.q_stride, head, x);
            turned(t, x, y);
            if (h + group < g.heads) put(g.q_out, g.q_out_stride, head, y);
        }
    }
    if (g.kv_heads <= first) return;
    const Turn t = turn_of(g.k_weight);
    int64_t page = -1, row = 0;
    if (a.c.pages) {
        const int64_t slot = g.slots[token];
        if (slot >= 0 && slot < a.c.pages * a.c.page_size) {
            page = a.page_mul ? static_cast<int64_t>((static_cast<uint64_t>(slot) * a.page_mul) >> a.page_shift) : slot / a.c.page_size;
            row = slot - page * a.c.page_size;
        }
    }
    const auto code = [&](const float(&f)[8], int head, int8_t *codes, float *scales) {
        const int64_t at_row = (page * a.c.kv_heads + head) * a.c.page_size + row;
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, abs_bits(f[j]));
        top = max_over<LANES>(top);
        const bool finite = top < kInfBits;
        Vec<int8_t, 8> q;
#pragma unroll
        for (int j = 0; j < 8; j++) q.v[j] = 0;
        if (finite && top) quantise<8>(f, __uint_as_float(top), q.v);
        if (in) *reinterpret_cast<Vec<int8_t, 8> *>(codes + at_row * a.c.head_dim + i0) = q;
        if (lane % LANES == 0) scales[at_row] = finite ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
    };
    for (int h = first; h < g.kv_heads; h += step) {
        const int head = min(h + group, g.kv_heads - 1);
        const bool there = h + group < g.kv_heads;
        float x[8], y[8];
        fetch(g.k, g.k_stride, head, x);
        turned(t, x, y);
        if (there && g.k_out) put(g.k_out, g.k_out_stride, head, y);
        if (page >= 0) {
            float v[8];
            fetch(g.v, g.v_stride, head, v);
            if (there) {
                code(y, head, a.c.k, a.c.k_scale);
                code(v, head, a.c.v, a.c.v_scale);
            }
        }
    }
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_rotate(const Spkv2KvCacheI8 *c, const Spkv2Rotate *g, void *stream) {
    return entry([&]() -> int {
        if (c)
            if (int rc = check_cache(c)) return rc;
        if (!g) return bad("rotate: no arguments");
        if (!is_dtype(g->dtype)) return bad("rotate: unknown dtype");
        if (g->tokens < 0 || g->heads < 0 || g->kv_heads < 0 || g->head_dim < 0 || g->pairs < 0) return bad("rotate: negative size");
        if (g->axes < 1) return bad("rotate: fewer than one axis");
        if (g->pairs > g->head_dim / 2) return bad("rotate: more pairs than a head has");
        if (g->norm && !(g->eps >= 0.0f)) return bad("rotate: eps is negative or NaN");
        if (g->norm && (g->q_weight || g->k_weight) && g->weight_dtype != g->dtype && g->weight_dtype != SPKV2_DTYPE_FP32)
            return bad("rotate: weight_dtype is neither the heads' nor fp32");
        if (c && (c->kv_heads != g->kv_heads || c->head_dim != g->head_dim)) return bad("rotate: the cache has other heads");
        if (g->head_dim % 16 || g->head_dim > 256) return unsupported("rotate: head_dim is not a multiple of 16 up to 256");
        if (g->tokens == 0 || (g->heads == 0 && g->kv_heads == 0) || g->head_dim == 0) return 0;
        if ((g->heads && (!g->q || !g->q_out)) || (g->kv_heads && (!g->k || (!c && !g->k_out)))) return bad("rotate: q, k or an output is NULL");
        if (c && (!g->v || !g->slots)) return bad("rotate: a cache without v or slots");
        if (g->pairs && (!g->positions || !g->frequencies)) return bad("rotate: positions or frequencies is NULL");
        const int64_t q_width = static_cast<int64_t>(g->heads) * g->head_dim, k_width = static_cast<int64_t>(g->kv_heads) * g->head_dim;
        if (g->tokens > 1) {
            if (g->heads && (g->q_stride < q_width || g->q_out_stride < q_width)) return bad("rotate: a stride is below the heads' width");
            if (g->kv_heads && (g->k_stride < k_width || (g->k_out && g->k_out_stride < k_width) || (c && g->v_stride < k_width)))
                return bad("rotate: a stride is below the heads' width");
            if (g->pairs && g->position_stride < g->axes) return bad("rotate: positions' stride is below their axes");
        }
        if (g->tokens > INT32_MAX || g->heads > 65535 || g->kv_heads > 65535) return unsupported("rotate: more than 2^31 tokens or 65535 heads");
        RotateArgs a{*g, c ? *c : Spkv2KvCacheI8{}, 1, 0, 0};
        if (c && c->pages * c->page_size <= INT32_MAX) div_magic(static_cast<unsigned>(c->page_size), &a.page_mul, &a.page_shift);
        const int groups = g->head_dim <= 64 ? 8 : g->head_dim <= 128 ? 4 : 2;
        // as many waves a token as fill 256 CUs with eight, one head at least for each of their groups
        const int64_t most = (std::max(g->heads, g->kv_heads) + groups - 1) / groups;
        a.parts = static_cast<int>(std::min<int64_t>(most, (2048 + g->tokens - 1) / g->tokens));
        const int64_t blocks = (g->tokens * a.parts + 3) / 4;
        if (blocks >= 1 << 24) return unsupported("rotate: too many tokens for one launch");
        const bool paired = g->interleaved || g->pairs % 8 == 0;
        const bool wide = g->norm && (g->q_weight || g->k_weight) && g->weight_dtype == SPKV2_DTYPE_FP32;
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel) { return launch("rotate", kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), stream, a); };
            auto by_weight = [&](auto w) {
                using W = decltype(w);
                if (groups == 8) return paired ? go(rotate_heads<T, W, 8, true>) : go(rotate_heads<T, W, 8, false>);
                if (groups == 4) return paired ? go(rotate_heads<T, W, 16, true>) : go(rotate_heads<T, W, 16, false>);
                return paired ? go(rotate_heads<T, W, 32, true>) : go(rotate_heads<T, W, 32, false>);
            };
            return wide ? by_weight(float{}) : by_weight(T{});
        });
    });
}
