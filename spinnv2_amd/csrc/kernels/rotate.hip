// Norms of queries and keys head by head, the rotation of their positions, and
// the way of keys and values into a paged int8 cache, in one pass.
//
//   y = x w / sqrt(mean(x^2) + eps),  (y_i, y_j) -> (y_i cos - y_j sin, y_j cos + y_i sin)
//
// A wave takes a token, or some of a token's heads where tokens are few: its 64
// lanes take the sines and cosines of the pairs, which every head of the token
// turns by, and groups of 8, 16 or 32 lanes a head each, 8 elements a lane.
//
// Bound by HBM and by its arithmetic, each two thirds of the time: 8190 tokens of
// 32 + 8 heads of 128 in bf16, values too, into the cache in 48 to 57 us (185 MB, 3.3
// to 3.9 TB/s), without a cache in 40 (168 MB, 4.2 TB/s); fp32 without a cache at 5.0
// TB/s.  Lanes read the pairs' doubles 32 bytes apart, which loses 44% of the LDS
// cycles to conflicts.
//
// In 64 bits: angles of far positions need it (position 70001 times a frequency
// near 1 keeps 7 bits behind the point in fp32), and a key beside the border of
// two bf16 values or two codes falls on its own side.  The vector units take
// 64-bit products at the rate of 32-bit ones.
#include <type_traits>

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

// 1 / sqrt(v): the hardware's estimate of 2^-26 and a step of Newton's method, within 2^-51; infinite for 0
__device__ __forceinline__ double inverse_root(double v) {
    const double r = __builtin_amdgcn_rsq(v);
    const double better = __builtin_fma(r * 0.5, __builtin_fma(-v * r, r, 1.0), r);
    return v > 0.0 && v < __builtin_inf() ? better : r;
}

// Eight values rounded to T, as floats.  By way of fp32, rounded twice, unless one
// of them may lie on a tie there, which is then taken straight from 64 bits: one
// in thirty thousand of bf16, one in four thousand of fp16.
template <typename T>
__device__ __forceinline__ void rounded(const double (&v)[8], float (&y)[8]) {
    // bits that are all 0 where a value may lie on a tie
    constexpr unsigned kBelow = __is_same(T, __bf16) ? 0x7fffu : 0xfffu;
    unsigned least = ~0u;
    float smallest = 1.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        y[j] = static_cast<float>(v[j]);
        least = min(least, __float_as_uint(y[j]) & kBelow);
        smallest = fminf(smallest, fabsf(y[j]));
    }
    // fp16 values below 2^-14 have their ties elsewhere
    const bool tie = least == 0 || (__is_same(T, _Float16) && smallest < 0x1p-14f);
    if constexpr (sizeof(T) == 2) {
        if (__any(tie)) {
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = static_cast<float>(static_cast<T>(v[j]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = static_cast<float>(static_cast<T>(y[j]));
        }
    }
}

// What a lane's 8 elements are multiplied by, and their partners: y = norm (x own + partner other); a bit for each that turns
struct Turn {
    double own[8], other[8];
    unsigned turns;
};
// in a cosine's place: the pair has no axis
constexpr double kNoAxis = 2.0;

// A lane's 8 elements of a head: four pairs, side by side (kBeside) or four of each
// half (kApart: a multiple of 4 apart), or eight in a row whose partners other lanes
// have (kAny), which LDS passes on.  Through LDS as well, pairs a multiple of 8 apart
// took 8190 tokens of 32 + 8 heads of 128 to 56 us.
enum Pairing { kBeside, kApart, kAny };

template <typename T, typename W, int LANES, Pairing PAIRING>
__global__ void __launch_bounds__(256) rotate_heads(RotateArgs a) {
    constexpr int kGroups = 64 / LANES, kDim = LANES * 8;
    __shared__ __align__(16) double table[4][2][128];
    __shared__ __align__(32) float heads[PAIRING == kAny ? 4 : 1][kGroups][kDim];
    const Spkv2Rotate &g = a.g;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    const int64_t token = at / a.parts;
    const int part = static_cast<int>(at - token * a.parts);
    if (token >= g.tokens) return;  // a whole wave; no barrier follows
    const int dim = g.head_dim, pairs = g.pairs;
    const int group = lane / LANES, eighth = min(lane % LANES, dim / 8 - 1);
    const bool in = lane % LANES < dim / 8;
    // where the lane's elements 0 .. 4 and 4 .. 8 lie; past the pairs, in a row
    int low = eighth * 8, high = low + 4;
    if constexpr (PAIRING == kApart) {
        const int past = eighth * 4 - pairs;
        low = past < 0 ? eighth * 4 : 2 * (pairs + past);
        high = past < 0 ? low + pairs : low + 4;
    }
    const auto place = [&](int e) { return e < 4 ? low + e : high + e - 4; };
    const int first = part * kGroups, step = a.parts * kGroups;
    // without a branch: lanes and groups past the last load its elements, and store nothing
    const auto fetch8 = [&](auto *p) {
        Vec<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, 8> v;
        if constexpr (PAIRING == kApart) {
            __builtin_memcpy(v.v, p + low, sizeof(v.v) / 2);
            __builtin_memcpy(v.v + 4, p + high, sizeof(v.v) / 2);
        } else {
            __builtin_memcpy(v.v, p + low, sizeof(v.v));
        }
        return v;
    };
    const auto fetch = [&](const void *x, int64_t stride, int head) {
        return fetch8(static_cast<const T *>(x) + token * stride + static_cast<int64_t>(head) * dim);
    };
    // the first head is on its way while the angles are taken
    Vec<T, 8> next;
    if (g.heads > first) next = fetch(g.q, g.q_stride, min(first + group, g.heads - 1));
    double *sines = table[wave][0], *cosines = table[wave][1];
    for (int p = lane; p < pairs; p += 64) {
        const int axis = g.axis ? g.axis[p] : 0;
        const bool there = static_cast<unsigned>(axis) < static_cast<unsigned>(g.axes);
        const int position = there ? g.positions[token * g.position_stride + axis] : 0;
        sine_cosine(static_cast<double>(position) * static_cast<double>(g.frequencies[p]), &sines[p], &cosines[p]);
        if (!there) cosines[p] = kNoAxis;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();

    // where element e of the lane has its partner; itself past the pairs
    const auto partner_of = [&](int e) {
        const int i = place(e);
        return i >= 2 * pairs ? i : PAIRING == kBeside ? i ^ 1 : i >= pairs ? i - pairs : i + pairs;
    };
    constexpr int kOther = PAIRING == kBeside ? 1 : 4;  // partner e ^ kOther of the same lane
    const auto turn_of = [&](const void *weight) {
        Turn t;
        t.turns = 0;
        float own[8], other[8];
#pragma unroll
        for (int e = 0; e < 8; e++) own[e] = other[e] = 1.0f;
        if (weight && g.norm) {
            const W *w = static_cast<const W *>(weight);
            widen(fetch8(w), own);
#pragma unroll
            for (int e = 0; e < 8; e++) other[e] = PAIRING == kAny ? static_cast<float>(w[partner_of(e)]) : own[e ^ kOther];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = place(e);
            const bool second = PAIRING == kBeside ? i & 1 : i >= pairs;
            const int p = i >= 2 * pairs ? 0 : PAIRING == kBeside ? i / 2 : second ? i - pairs : i;
            const double c = cosines[p], s = sines[p];
            const bool turns = i < 2 * pairs && c != kNoAxis;
            t.turns |= turns ? 1u << e : 0u;
            t.own[e] = (turns ? c : 1.0) * static_cast<double>(own[e]);
            t.other[e] = turns ? (second ? s : -s) * static_cast<double>(other[e]) : 0.0;
        }
        return t;
    };
    float *mine = heads[PAIRING == kAny ? wave : 0][group];
    const double per = 1.0 / dim;
    const auto turned = [&](const Turn &t, const Vec<T, 8> &raw, float (&y)[8]) {
        float x[8], other[8];
        widen(raw, x);
        double factor = 1.0;
        if (g.norm) {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j++) sum = __builtin_fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum);
            factor = inverse_root(sum_over<LANES>(in ? sum : 0.0) * per + static_cast<double>(g.eps));
        }
        if constexpr (PAIRING != kAny) {
#pragma unroll
            for (int e = 0; e < 8; e++) other[e] = x[e ^ kOther];
        } else {
            if (in) put_floats<8>(mine + low, x);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int e = 0; e < 8; e++) other[e] = mine[partner_of(e)];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            // to what does not turn nothing is added: 0 times what is not finite would be NaN
            const float o = t.turns >> j & 1 ? other[j] : 0.0f;
            v[j] = __builtin_fma(static_cast<double>(o), t.other[j], static_cast<double>(x[j]) * t.own[j]) * factor;
        }
        rounded<T>(v, y);
    };
    const auto put = [&](void *y, int64_t stride, int head, const float(&f)[8]) {
        T *p = static_cast<T *>(y) + token * stride + static_cast<int64_t>(head) * dim;
        if constexpr (PAIRING == kApart) {
            store_floats<4>(p + low, {f[0], f[1], f[2], f[3]});
            store_floats<4>(p + high, {f[4], f[5], f[6], f[7]});
        } else {
            store_floats<8>(p + low, f);
        }
    };
    if (g.heads > first) {
        const Turn t = turn_of(g.q_weight);
        for (int h = first; h < g.heads; h += step) {
            const Vec<T, 8> now = next;
            next = fetch(g.q, g.q_stride, min(h + step + group, g.heads - 1));
            float y[8];
            turned(t, now, y);
            if (in && h + group < g.heads) put(g.q_out, g.q_out_stride, h + group, y);
        }
    }
    if (g.kv_heads <= first) return;
    int64_t page = -1, row = 0;
    if (a.c.pages) {
        const int64_t slot = g.slots[token];
        if (slot >= 0 && slot < a.c.pages * a.c.page_size) {
            page = a.page_mul ? static_cast<int64_t>((static_cast<uint64_t>(slot) * a.page_mul) >> a.page_shift) : slot / a.c.page_size;
            row = slot - page * a.c.page_size;
        }
    }
    const auto code = [&](const float(&x)[8], bool there, int head, int8_t *codes, float *scales) {
        const int64_t at_row = (page * a.c.kv_heads + head) * a.c.page_size + row;
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, abs_bits(x[j]));
        top = max_over<LANES>(in ? top : 0);
        const bool finite = top < kInfBits;
        Vec<int8_t, 8> q;
#pragma unroll
        for (int j = 0; j < 8; j++) q.v[j] = 0;
        if (finite && top) quantise<8>(x, __uint_as_float(top), q.v);
        if (in && there) {
            int8_t *p = codes + at_row * a.c.head_dim;
            __builtin_memcpy(p + low, q.v, 4);
            __builtin_memcpy(p + high, q.v + 4, 4);
        }
        if (lane % LANES == 0 && there) scales[at_row] = finite ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
    };
    const Turn t = turn_of(g.k_weight);
    for (int h = first; h < g.kv_heads; h += step) {
        const int head = min(h + group, g.kv_heads - 1);
        const bool there = h + group < g.kv_heads;
        const Vec<T, 8> k = fetch(g.k, g.k_stride, head);
        Vec<T, 8> v;
        if (page >= 0) v = fetch(g.v, g.v_stride, head);
        float y[8];
        turned(t, k, y);
        if (in && there && g.k_out) put(g.k_out, g.k_out_stride, head, y);
        if (page >= 0) {  // the whole wave: a token's
            code(y, there, head, a.c.k, a.c.k_scale);
            widen(v, y);
            code(y, there, head, a.c.v, a.c.v_scale);
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
        const bool wide = g->norm && (g->q_weight || g->k_weight) && g->weight_dtype == SPKV2_DTYPE_FP32;
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel) { return launch("rotate", kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), stream, a); };
            auto by_weight = [&](auto w) {
                using W = decltype(w);
                auto by_lanes = [&](auto beside, auto apart, auto any) { return go(g->interleaved ? beside : g->pairs % 4 == 0 ? apart : any); };
                if (groups == 8) return by_lanes(rotate_heads<T, W, 8, kBeside>, rotate_heads<T, W, 8, kApart>, rotate_heads<T, W, 8, kAny>);
                if (groups == 4) return by_lanes(rotate_heads<T, W, 16, kBeside>, rotate_heads<T, W, 16, kApart>, rotate_heads<T, W, 16, kAny>);
                return by_lanes(rotate_heads<T, W, 32, kBeside>, rotate_heads<T, W, 32, kApart>, rotate_heads<T, W, 32, kAny>);
            };
            return wide ? by_weight(float{}) : by_weight(T{});
        });
    });
}
