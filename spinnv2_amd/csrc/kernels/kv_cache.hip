// A paged key/value cache in int8: tokens quantised as they are written, and
// read back.
//
// Write: each head's vector of a token is quantised by its own largest
// absolute value.  One pass, a group of lanes a vector, 8 elements a lane, the
// maximum joined over the group's lanes.  Read: 16 codes a lane, scaled.  Both
// bound by HBM; a call of a few tokens by its launch.
#include "decoder.hpp"

namespace spk::dec {

namespace {

struct WriteArgs {
    Spkv2KvCacheI8 c;
    const void *k, *v;
    const int64_t *slots;
    int64_t tokens, k_stride, v_stride;
};

// LANES lanes (of which head_dim / 8 have elements) a vector; blockIdx.y: k, v
template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(256) kv_write(WriteArgs a) {
    const int64_t vec = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t token = vec / a.c.kv_heads;
    const int head = static_cast<int>(vec - token * a.c.kv_heads);
    if (token >= a.tokens) return;  // whole groups of lanes
    const int64_t slot = a.slots[token];
    const int64_t page = slot / a.c.page_size;
    if (slot < 0 || page >= a.c.pages) return;
    const int at = static_cast<int>(slot - page * a.c.page_size);
    const bool is_v = blockIdx.y != 0;
    const T *x = static_cast<const T *>(is_v ? a.v : a.k) + token * (is_v ? a.v_stride : a.k_stride) +
                 static_cast<int64_t>(head) * a.c.head_dim + lane * 8;
    const int64_t row = (page * a.c.kv_heads + head) * a.c.page_size + at;
    const bool in = lane * 8 < a.c.head_dim;
    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (in) {
        if constexpr (VEC) load_floats<8>(x, f);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = static_cast<float>(x[j]);
        }
    }
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, abs_bits(f[j]));
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), d, LANES)));
    const bool finite = top < kInfBits;
    Vec<int8_t, 8> q;
#pragma unroll
    for (int j = 0; j < 8; j++) q.v[j] = 0;
    if (finite && top) quantise<8>(f, __uint_as_float(top), q.v);
    if (in) *reinterpret_cast<Vec<int8_t, 8> *>((is_v ? a.c.v : a.c.k) + row * a.c.head_dim + lane * 8) = q;
    if (lane == 0) (is_v ? a.c.v_scale : a.c.k_scale)[row] = finite ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
}

struct ReadArgs {
    Spkv2KvCacheI8 c;
    Spkv2KvRead r;
};

// The sequence whose rows hold row t: how many of offsets[1 ..] are <= t.
__device__ __forceinline__ int sequence_of(const int32_t *offsets, int sequences, int64_t t) {
    int low = 0, high = sequences;  // the first s with offsets[s + 1] > t
    while (low < high) {
        const int mid = (low + high) / 2;
        if (offsets[mid + 1] > t) high = mid;
        else low = mid + 1;
    }
    return low;
}

// 16 codes a lane, pieces of the token's heads one after the other
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv_read(ReadArgs a) {
    const int pieces = a.c.kv_heads * (a.c.head_dim / 16);
    const bool is_v = blockIdx.y != 0;
    T *out = static_cast<T *>(is_v ? a.r.v : a.r.k);
    if (!out) return;
    const int64_t total = a.r.tokens * pieces;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t t = i / pieces;
        const int p = static_cast<int>(i - t * pieces);
        const int s = sequence_of(a.r.offsets, a.r.sequences, t);
        if (s >= a.r.sequences || t < a.r.offsets[0]) continue;
        const int64_t place = (a.r.first ? a.r.first[s] : 0) + t - a.r.offsets[s];
        const int head = p / (a.c.head_dim / 16), d = (p % (a.c.head_dim / 16)) * 16;
        const int64_t col = place / a.c.page_size;
        int64_t page = -1;
        if (place >= 0 && col < a.r.table_width) page = a.r.table[static_cast<int64_t>(s) * a.r.table_width + col];
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; j++) f[j] = 0.0f;
        if (page >= 0 && page < a.c.pages) {
            const int64_t row = (page * a.c.kv_heads + head) * a.c.page_size + (place - col * a.c.page_size);
            const float scale = (is_v ? a.c.v_scale : a.c.k_scale)[row];
            const Vec<int8_t, 16> q = *reinterpret_cast<const Vec<int8_t, 16> *>((is_v ? a.c.v : a.c.k) + row * a.c.head_dim + d);
#pragma unroll
            for (int j = 0; j < 16; j++) f[j] = scale * static_cast<float>(q.v[j]);
        }
        T *y = out + t * (is_v ? a.r.v_stride : a.r.k_stride) + static_cast<int64_t>(head) * a.c.head_dim + d;
        if constexpr (VEC) store_floats<16>(y, f);
        else {
#pragma unroll
            for (int j = 0; j < 16; j++) y[j] = static_cast<T>(f[j]);
        }
    }
}

}  // namespace

int check_cache(const Spkv2KvCacheI8 *c) {
    if (!c) return bad("kv cache: no cache");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return bad("kv cache: a buffer is NULL");
    if (c->pages < 1 || c->kv_heads < 1 || c->page_size < 1 || c->head_dim < 1) return bad("kv cache: a size is below 1");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))
        return bad("kv cache: a buffer is not 16-byte aligned");
    if (c->page_size % 16 || c->page_size > (1 << 20)) return unsupported("kv cache: page_size is not a multiple of 16 up to 2^20");
    if (c->head_dim % 16 || c->head_dim > 256) return unsupported("kv cache: head_dim is not a multiple of 16 up to 256");
    if (c->kv_heads > 65535 || c->pages > INT32_MAX) return unsupported("kv cache: more than 65535 heads or 2^31 pages");
    return 0;
}

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_kv_write_i8(const Spkv2KvCacheI8 *c, const Spkv2KvWrite *g, void *stream) {
    return entry([&]() -> int {
        if (int rc = check_cache(c)) return rc;
        if (!g) return bad("kv_write_i8: no arguments");
        if (!is_dtype(g->dtype)) return bad("kv_write_i8: unknown dtype");
        if (g->tokens < 0) return bad("kv_write_i8: negative size");
        if (g->tokens == 0) return 0;
        if (!g->k || !g->v || !g->slots) return bad("kv_write_i8: k, v or slots is NULL");
        const int64_t width = static_cast<int64_t>(c->kv_heads) * c->head_dim;
        if (g->tokens > 1 && (g->k_stride < width || g->v_stride < width)) return bad("kv_write_i8: a stride is below the heads' width");
        if (g->tokens > INT32_MAX) return unsupported("kv_write_i8: more than 2^31 tokens");
        const size_t size = dtype_size(g->dtype);
        const bool vec = aligned(g->k, 16) && aligned(g->v, 16) && (g->k_stride * size) % 16 == 0 && (g->v_stride * size) % 16 == 0;
        const WriteArgs a{*c, g->k, g->v, g->slots, g->tokens, g->k_stride, g->v_stride};
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel, int lanes) {
                const int64_t vecs = g->tokens * c->kv_heads, blocks = (vecs + 256 / lanes - 1) / (256 / lanes);
                if (blocks > INT32_MAX) return unsupported("kv_write_i8: too many tokens for one launch");
                return launch("kv_write_i8", kernel, dim3(static_cast<unsigned>(blocks), 2), dim3(256), stream, a);
            };
            if (c->head_dim <= 64) return vec ? go(kv_write<T, 8, true>, 8) : go(kv_write<T, 8, false>, 8);
            if (c->head_dim <= 128) return vec ? go(kv_write<T, 16, true>, 16) : go(kv_write<T, 16, false>, 16);
            return vec ? go(kv_write<T, 32, true>, 32) : go(kv_write<T, 32, false>, 32);
        });
    });
}

extern "C" int spkv2_mi355x_kv_read_i8(const Spkv2KvCacheI8 *c, const Spkv2KvRead *g, void *stream) {
    return entry([&]() -> int {
        if (int rc = check_cache(c)) return rc;
        if (!g) return bad("kv_read_i8: no arguments");
        if (!is_dtype(g->dtype)) return bad("kv_read_i8: unknown dtype");
        if (g->tokens < 0 || g->sequences < 0 || g->table_width < 0) return bad("kv_read_i8: negative size");
        if (g->tokens == 0 || g->sequences == 0 || (!g->k && !g->v)) return 0;
        if (!g->offsets || (!g->table && g->table_width)) return bad("kv_read_i8: table or offsets is NULL");
        const int64_t width = static_cast<int64_t>(c->kv_heads) * c->head_dim;
        if (g->tokens > 1 && ((g->k && g->k_stride < width) || (g->v && g->v_stride < width)))
            return bad("kv_read_i8: a stride is below the heads' width");
        if (g->tokens > INT32_MAX) return unsupported("kv_read_i8: more than 2^31 tokens");
        const size_t size = dtype_size(g->dtype);
        const bool vec = aligned(g->k, 16) && aligned(g->v, 16) && (g->k_stride * size) % 16 == 0 && (g->v_stride * size) % 16 == 0;
        const ReadArgs a{*c, *g};
        const int64_t blocks = (g->tokens * c->kv_heads * (c->head_dim / 16) + 255) / 256;
        const dim3 grid(static_cast<unsigned>(blocks < 65536 ? blocks : 65536), 2);
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            return vec ? launch("kv_read_i8", kv_read<T, true>, grid, dim3(256), stream, a)
                       : launch("kv_read_i8", kv_read<T, false>, grid, dim3(256), stream, a);
        });
    });
}
