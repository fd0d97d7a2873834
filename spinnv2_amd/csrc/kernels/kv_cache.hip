// A paged key/value cache in int8: tokens quantised as they are written, and
// read back.  Both are bound by HBM, a call of a few tokens by its launch.
//
// Write: each head's vector of a token is quantised by its own largest
// absolute value.  One pass, a group of lanes a vector, 8 elements a lane, the
// maximum joined over the group's lanes.  A workgroup takes one head of
// neighbouring tokens, whose rows and scales lie next to each other in a page:
// with the heads side by side instead, a page's line of scales was written a
// few bytes at a time from several XCDs (3 x 8191 tokens of 8 heads of 128,
// 152 MB: 45 us, 38 so, 4.0 TB/s).  Read: 16 codes a lane, scaled (31 us, 4.9
// TB/s).
#include "decoder.hpp"

namespace spk::dec {

namespace {

struct WriteArgs {
    Spkv2KvCacheI8 c;
    const void *k, *v;
    const int64_t *slots;
    int64_t tokens, k_stride, v_stride;
    unsigned page_mul;  // slot / page_size, by multiplication; 0: slots pass 2^31
    int page_shift;
};

// LANES lanes (of which head_dim / 8 have elements) a vector
template <typename T, int LANES>
__global__ void __launch_bounds__(256) kv_write(WriteArgs a) {
    const int head = blockIdx.x % a.c.kv_heads, lane = threadIdx.x % LANES;
    const int64_t token = static_cast<int64_t>(blockIdx.x / a.c.kv_heads) * (256 / LANES) + threadIdx.x / LANES;
    if (token >= a.tokens) return;  // whole groups of lanes
    const bool in = lane * 8 < a.c.head_dim;
    const int64_t at_head = static_cast<int64_t>(head) * a.c.head_dim + lane * 8;
    float f[2][8];
#pragma unroll
    for (int n = 0; n < 2; n++) {
        const T *x = static_cast<const T *>(n ? a.v : a.k) + token * (n ? a.v_stride : a.k_stride) + at_head;
#pragma unroll
        for (int j = 0; j < 8; j++) f[n][j] = 0.0f;
        if (in) load_floats<8>(x, f[n]);
    }
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= a.c.pages * a.c.page_size) return;  // below 2^51
    const int64_t page = a.page_mul ? static_cast<int64_t>((static_cast<uint64_t>(slot) * a.page_mul) >> a.page_shift) : slot / a.c.page_size;
    const int64_t row = (page * a.c.kv_heads + head) * a.c.page_size + (slot - page * a.c.page_size);
#pragma unroll
    for (int n = 0; n < 2; n++) {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, abs_bits(f[n][j]));
        top = max_over<LANES>(top);
        const bool finite = top < kInfBits;
        Vec<int8_t, 8> q;
#pragma unroll
        for (int j = 0; j < 8; j++) q.v[j] = 0;
        if (finite && top) quantise<8>(f[n], __uint_as_float(top), q.v);
        if (in) *reinterpret_cast<Vec<int8_t, 8> *>((n ? a.c.v : a.c.k) + row * a.c.head_dim + lane * 8) = q;
        if (lane == 0) (n ? a.c.v_scale : a.c.k_scale)[row] = finite ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
    }
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
template <typename T>
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
        store_floats<16>(y, f);
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
        WriteArgs a{*c, g->k, g->v, g->slots, g->tokens, g->k_stride, g->v_stride, 0, 0};
        if (c->pages * c->page_size <= INT32_MAX) div_magic(static_cast<unsigned>(c->page_size), &a.page_mul, &a.page_shift);
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto kernel, int lanes) {
                const int64_t blocks = (g->tokens + 256 / lanes - 1) / (256 / lanes) * c->kv_heads;
                if (blocks >= 1 << 24) return unsupported("kv_write_i8: too many tokens for one launch");
                return launch("kv_write_i8", kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), stream, a);
            };
            if (c->head_dim <= 64) return go(kv_write<T, 8>, 8);
            if (c->head_dim <= 128) return go(kv_write<T, 16>, 16);
            return go(kv_write<T, 32>, 32);
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
        const ReadArgs a{*c, *g};
        const int64_t blocks = (g->tokens * c->kv_heads * (c->head_dim / 16) + 255) / 256;
        const dim3 grid(static_cast<unsigned>(blocks < 65536 ? blocks : 65536), 2);
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            return launch("kv_read_i8", kv_read<T>, grid, dim3(256), stream, a);
        });
    });
}
