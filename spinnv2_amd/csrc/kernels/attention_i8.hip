// Attention of new tokens to a paged int8 cache.
//
//   out[i] = sum_t p[i, t] v[t] / sum_t p[i, t],  p = exp(scale q[i] k[t])
//
// The codes are turned into 16-bit floats, exactly, and multiplied on the
// fp16 matrix cores; a token's key scale multiplies its scores, its value
// scale its weights.
//
// attend_rows takes 16 rows (query, head of the group) of a sequence and kv head
// a workgroup, for single tokens above all: bound by the cache's bytes (64 sequences of
// 3001 to 16384 tokens, 8 kv heads of 128, 1.31 GB: 270 us, 4.9 TB/s), one
// short sequence by its loads' latency (333 tokens 9.7 us).  attend_tiles takes
// 128 rows a workgroup: bound by two waves a SIMD whose arithmetic and matrix
// products hide little of each other (4001 queries of 32 heads on 4001 and 6007
// tokens, 394 GFLOP: 507 to 523 us on three chips, 770 TFLOP/s, half of what a
// large product reaches).
//
// Weights are rounded to fp16's 11 bits for the second product, except of fp32
// rows, where they are two parts: bf16 results do not show it (relative error
// 1.7e-3 with either), of fp16 rows 2.1e-4 becomes 2.9e-4, and a second part
// would double the products that the kernel for many rows is bound by.
#include <cstdio>

#include "decoder.hpp"

namespace spk::dec {

namespace {

struct AttnArgs {
    Spkv2KvCacheI8 c;
    const void *q;
    void *out;
    const int32_t *table, *lengths, *offsets;
    float *part, *stats;  // [row][split][head_dim] sums, [row][split][2] base and total; row = row of q * heads + head
    int64_t queries, q_stride, out_stride;
    int max_queries, max_length, table_width, heads, group, sequences;
    int causal, window;
    float scale;
    int row_blocks, split_tokens, splits;
    unsigned page_mul;  // token / page_size, by multiplication
    int page_shift;
};

constexpr int kChunk = 32;   // tokens a wave takes at a time, as two tiles of 16
// A row's weights are 2^(score - base), and times their tokens' value scales
// (their size) they are fp16.  The base is kLift below the largest size so far,
// and follows it only when one passes it by kSlack more: sizes stay below 2^15,
// and the largest at 2^7 or more (2^3 where it is bounded by a tile's largest
// value scale).  So the base goes by what the row itself reads: neither a token
// that its mask leaves out, nor one of large values and next to no weight, costs
// it bits.
constexpr float kSlack = 8.0f, kLift = 7.0f;
// the least logarithm of a value scale: 2^(score - base) stays a float
constexpr float kLeastLog = -96.0f;

// Two codes of a dword, picked by `sel` into the low bytes of two halves, as
// fp16: 0x6400 + (code + 128) is 1024 + 128 + code.
__device__ __forceinline__ half2_t codes_to_half(unsigned hi, unsigned lo, unsigned sel) {
    const unsigned u = __builtin_amdgcn_perm(hi, lo, sel) ^ 0x64806480u;
    constexpr half2_t kBias = {static_cast<_Float16>(1152), static_cast<_Float16>(1152)};
    return __builtin_bit_cast(half2_t, u) - kBias;
}
__device__ __forceinline__ half8_t join(half2_t a, half2_t b, half2_t c, half2_t d) {
    return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// eight codes in a row
__device__ __forceinline__ half8_t codes8(unsigned a, unsigned b) {
    return join(codes_to_half(0, a, 0x0c010c00u), codes_to_half(0, a, 0x0c030c02u), codes_to_half(0, b, 0x0c010c00u),
                codes_to_half(0, b, 0x0c030c02u));
}

// A value that is split into parts is rounded to fp32 first: a product fused
// into the conversion to its high part, but not into the low part's, would give
// parts of two values, a step of fp16 apart where one lies next to a tie.
__device__ __forceinline__ void once(float &v) { asm("" : "+v"(v)); }

// eight elements at p, of any alignment
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    Vec<T, 8> v;
    __builtin_memcpy(v.v, p, sizeof(v.v));
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = static_cast<float>(v.v[e]);
}

__device__ __forceinline__ float over_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// log2 of a value scale, kLeastLog at least.  Infinity or NaN gives what fmaxf
// passes over beside a masked token's score of -infinity.
__device__ __forceinline__ float log_scale(float scale) { return fmaxf(__builtin_amdgcn_logf(fabsf(scale)), kLeastLog); }

// Sums relative to `from`, now relative to `to`: a factor that is applied twice,
// since 2^(from - to) may be 0 where the totals of tokens with tiny values still
// count.
__device__ __forceinline__ float half_ratio(float from, float to) {
    return from > -__builtin_inff() ? __builtin_amdgcn_exp2f((from - to) * 0.5f) : 0.0f;
}

struct Sequence {
    int64_t row0;   // its first row of q
    int count;      // queries computed
    int position;   // position of its first query
    int length;     // tokens read
    int true_length;
};
__device__ __forceinline__ Sequence sequence(const AttnArgs &a, int b) {
    Sequence s;
    const int o0 = a.offsets[b], o1 = a.offsets[b + 1];
    s.true_length = max(a.lengths[b], 0);
    s.row0 = o0;
    s.count = min(o1 - o0, a.max_queries);
    if (o0 < 0) s.count = 0;
    if (o0 + static_cast<int64_t>(s.count) > a.queries) s.count = static_cast<int>(a.queries - o0);
    s.position = s.true_length - (o1 - o0);
    const int64_t held = static_cast<int64_t>(a.table_width) * a.c.page_size;
    s.length = max(0, min(s.true_length, a.max_length));
    if (s.length > held) s.length = static_cast<int>(held);
    return s;
}

// The first token that the window (causal calls only have one) leaves to the
// query at `position`; 0 without one.  No difference is formed that could pass 32 bits: with a window
// of 2^31 - 1 and a query ahead of the first token it would turn into a token far
// past the table.
__device__ __forceinline__ int window_from(const AttnArgs &a, int position) {
    return a.window && position >= a.window ? position + 1 - a.window : 0;
}

// A split in which rows r0 .. r1 read no token: no sums, and a total of 0.
__device__ __forceinline__ void nothing(const AttnArgs &a, const Sequence &s, int head, int split, int r0, int r1) {
    for (int r = r0 + static_cast<int>(threadIdx.x); r < r1; r += blockDim.x) {
        const int i = r / a.group;
        const int64_t at = ((s.row0 + i) * a.heads + head * a.group + (r - i * a.group)) * a.splits + split;
        a.stats[2 * at] = -__builtin_inff();
        a.stats[2 * at + 1] = 0.0f;
    }
}

// Which rows and tokens are a workgroup's: the first split of every sequence and
// head first, the heaviest rows of a causal mask ahead, so that what runs at the
// end is short.  A sequence's and head's blocks are on one XCD where the pairs
// are a multiple of eight, in an order that turns, since an XCD's workgroups go
// to its four engines in turn too.  With the splits side by side each XCD had
// its own, most of them empty on two of the eight (64 sequences of 3001 to 16384
// tokens: 420 us, 305 in this order); without the turn two sequences of 4001 and
// 6007 tokens kept two engines each (619 us, 530 with it).
struct Place {
    int b, head, split, block;
};
__device__ __forceinline__ Place place(const AttnArgs &a) {
    const unsigned pairs = a.sequences * a.c.kv_heads, rest = blockIdx.x / pairs;
    const int pair = (blockIdx.x + rest / 2 % pairs * 8) % pairs;
    Place p;
    p.b = pair / a.c.kv_heads;
    p.head = pair - p.b * a.c.kv_heads;
    p.split = rest / a.row_blocks;
    p.block = a.row_blocks - 1 - rest % a.row_blocks;
    return p;
}

// One workgroup: 16 rows (query, head of the group) of one sequence and kv
// head, and one split of its tokens.  Scores are taken
// transposed, S^T = K q^T on 16x16 tiles: a lane then holds four tokens'
// scores of one row, which are the weights' operand of O^T = V^T P^T as they
// are, if V's rows are taken in the same order.  So nothing passes through LDS
// until the waves' sums are joined.
//
// Lane l: column l % 16 (a row of q), group g = l / 16.
//   K: token l % 16 of the tile, its codes g DP/4 .. + DP/4 (q in the same
//      order of d, which the product does not see)
//   scores, weights: tokens 4 g .. + 4 of each tile
//   V: those tokens' codes VPL (l % 16) .. + VPL (VPL = DP / 16); product j
//      takes d = VPL r + j as its row r
template <typename T, int DP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, DP * sizeof(T) <= 256 ? 12 / WAVES : 1) attend_rows(AttnArgs a) {
    constexpr bool kWide = sizeof(T) == 4;  // rows of 22 bits: two fp16 parts
    constexpr int kParts = kWide ? 2 : 1;
    constexpr int kPieces = DP / 64;  // 16-byte pieces of K a lane
    constexpr int kVpl = DP / 16;     // V codes a lane
    constexpr int kVw = kVpl / 4;
    __shared__ __align__(16) float joined[WAVES * 64 * 4 * kVpl];
    __shared__ float wave_max[WAVES][16], wave_sum[WAVES][16];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const Place at_block = place(a);
    const int b = at_block.b, head = at_block.head, split = at_block.split, block = at_block.block;
    const int dim = a.c.head_dim;
    const Sequence s = sequence(a, b);
    const int rows = s.count * a.group, r0 = block * 16;
    if (r0 >= rows) return;
    const int first_q = r0 / a.group, last_q = (min(rows, r0 + 16) - 1) / a.group;
    int low = split * a.split_tokens, high = min(s.length, low + a.split_tokens);
    if (a.causal) {
        high = min(high, s.position + last_q + 1);
        low = max(low, window_from(a, s.position + first_q));
    }

    if (a.splits > 1 && low >= high) {
        nothing(a, s, head, split, r0, min(rows, r0 + 16));
        return;
    }

    struct Chunk {
        uintx4 k[2][kPieces];
        unsigned v[8][kVw];
        floatx4 ks[2], vs[2];
        bool ok[2];
    };
    // Pages of the wave's next 32 chunks, two a chunk, one a lane: a chunk's
    // loads wait for no load of its page.
    const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
    int ahead = 0;
    auto look = [&](int at) {
        const int t = at + lane / 2 * (WAVES * kChunk) + lane % 2 * 16;
        ahead = -1;
        if (t < high) ahead = table[(static_cast<uint64_t>(static_cast<unsigned>(t)) * a.page_mul) >> a.page_shift];
    };
    auto fetch = [&](Chunk &x, int at, int n) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int t = at + 16 * h;
            const int page_at = static_cast<int>((static_cast<uint64_t>(static_cast<unsigned>(t)) * a.page_mul) >> a.page_shift);
            const int page = __builtin_amdgcn_readlane(ahead, 2 * (n & 31) + h);
            x.ok[h] = page >= 0 && page < a.c.pages;
            x.ks[h] = x.vs[h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < kPieces; p++) x.k[h][p] = uintx4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int w = 0; w < kVw; w++) x.v[4 * h + u][w] = 0;
            if (!x.ok[h]) continue;
            const int64_t row = (static_cast<int64_t>(page) * a.c.kv_heads + head) * a.c.page_size + (t - page_at * a.c.page_size);
            x.ks[h] = *reinterpret_cast<const floatx4 *>(a.c.k_scale + row + 4 * g);
            x.vs[h] = *reinterpret_cast<const floatx4 *>(a.c.v_scale + row + 4 * g);
            const int8_t *k = a.c.k + (row + col) * dim + g * (DP / 4);
#pragma unroll
            for (int p = 0; p < kPieces; p++)
                if (DP / 4 * g + 16 * p < dim) x.k[h][p] = *reinterpret_cast<const uintx4 *>(k + 16 * p);
            const int8_t *v = a.c.v + (row + 4 * g) * dim + kVpl * col;
            if (kVpl * col < dim) {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const Vec<unsigned, kVw> y = *reinterpret_cast<const Vec<unsigned, kVw> *>(v + u * dim);
#pragma unroll
                    for (int w = 0; w < kVw; w++) x.v[4 * h + u][w] = y.v[w];
                }
            }
        }
    };
    // the first chunk is on its way while the queries are split
    Chunk now;
    int at = low / kChunk * kChunk + wave * kChunk, n = 0;
    if (at < high) {
        look(at);
        fetch(now, at, 0);
    }

    // the rows' masks and queries, scaled by a power of two to 2^14 .. 2^15
    half8_t qf[DP / 32][kParts];
    float factor, m, l;
    int last, start;
    floatx4 acc[kVpl];
    {
        const int r = r0 + col, i = r / a.group;
        const bool in = r < rows;
        last = a.causal ? s.position + i : s.length - 1;
        start = window_from(a, last);
        // without a branch, so that all loads are on their way at once: rows past the last are the last
        const int rq = min(r, rows - 1), iq = rq / a.group;
        const T *q = static_cast<const T *>(a.q) + (s.row0 + iq) * a.q_stride +
                     static_cast<int64_t>(head * a.group + (rq - iq * a.group)) * dim;
        float f[DP / 32][8];
        float top = 0.0f;
#pragma unroll
        for (int x = 0; x < DP / 32; x++) {
            const int d = g * (DP / 4) + 8 * x;
            load8(q + min(d, dim - 8), f[x]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f[x][e] = in && d < dim ? f[x][e] : 0.0f;
                top = fmaxf(top, fabsf(f[x][e]));
            }
        }
        top = over_groups_max(top);
        // an infinite query's scores are not finite whatever the codes, and all of -infinity would read as masked
        if (top == __builtin_inff()) f[0][0] = __builtin_nanf("");
        const int ex = top > 0.0f && top < __builtin_inff() ? ilogbf(top) : 0;
        factor = ldexpf(a.scale * 1.44269504088896340736f, ex - 14);
#pragma unroll
        for (int x = 0; x < DP / 32; x++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = ldexpf(f[x][e], 14 - ex);
                const _Float16 hi = static_cast<_Float16>(v);
                qf[x][0][e] = hi;
                if constexpr (kWide) qf[x][kParts - 1][e] = static_cast<_Float16>(v - static_cast<float>(hi));
            }
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < kVpl; j++) acc[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto use = [&](const Chunk &x, int at) {
        floatx4 sc[2];
        sc[0] = sc[1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int p = 0; p < kPieces; p++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const half8_t kf = codes8(x.k[h][p][2 * e], x.k[h][p][2 * e + 1]);
#pragma unroll
                        for (int w = 0; w < kParts; w++)
                            sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[2 * p + e][w], sc[h], 0, 0, 0);
                }
        half8_t pf[kParts];
        {
            float v[8], most = -__builtin_inff();  // the largest size, as a logarithm
            unsigned widest = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = sc[e / 4][e % 4] * (x.ks[e / 4][e % 4] * factor);
                widest = max(widest, max(abs_bits(x.ks[e / 4][e % 4]), abs_bits(x.vs[e / 4][e % 4])));
            }
            if (__any(widest >= kInfBits)) {  // an infinite key scale may have given -infinity, which stands for masked
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (max(abs_bits(x.ks[e / 4][e % 4]), abs_bits(x.vs[e / 4][e % 4])) >= kInfBits) v[e] = __builtin_nanf("");
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int token = at + 16 * (e / 4) + 4 * g + e % 4;
                const bool keep = token >= low && token < high && x.ok[e / 4] && token <= last && token >= start;
                v[e] = keep ? v[e] : -__builtin_inff();
                most = fmaxf(most, v[e] + log_scale(x.vs[e / 4][e % 4]));
            }
            if (__any(most > m + (kLift + kSlack))) {
                // a row whose own sizes have not passed keeps its base
                most = over_groups_max(most);
                const float now = most > m + (kLift + kSlack) ? most - kLift : m;
                const float half = half_ratio(m, now);
                m = now;
                l = l * half * half;
#pragma unroll
                for (int j = 0; j < kVpl; j++) acc[j] *= half * half;
            }
            const float from = m > -__builtin_inff() ? m : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = __builtin_amdgcn_exp2f(v[e] - from);
                l += p;
                // 0 where the row masks the token, whose scale may be NaN
                float w = v[e] == -__builtin_inff() ? 0.0f : p * x.vs[e / 4][e % 4];
                if constexpr (kWide) once(w);
                const _Float16 hi = static_cast<_Float16>(w);
                pf[0][e] = hi;
                if constexpr (kWide) pf[kParts - 1][e] = static_cast<_Float16>(w - static_cast<float>(hi));
            }
        }
#pragma unroll
        for (int j = 0; j < kVpl; j++) {
            const unsigned sel = 0x0c000c00u | ((4u + j % 4) << 16) | (j % 4);
            const half8_t vf = join(codes_to_half(x.v[1][j / 4], x.v[0][j / 4], sel), codes_to_half(x.v[3][j / 4], x.v[2][j / 4], sel),
                                    codes_to_half(x.v[5][j / 4], x.v[4][j / 4], sel), codes_to_half(x.v[7][j / 4], x.v[6][j / 4], sel));
#pragma unroll
                for (int w = 0; w < kParts; w++)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[w], acc[j], 0, 0, 0);
        }
    };

    while (at < high) {
        use(now, at);
        at += WAVES * kChunk;
        n++;
        if (at >= high) break;
        if ((n & 31) == 0) look(at);
        fetch(now, at, n);
    }

    // the waves' sums, joined in wave order
    {
        l = over_groups_sum(l);
        if (g == 0) {
            wave_max[wave][col] = m;
            wave_sum[wave][col] = l;
        }
    }
    __syncthreads();
    {
        float most = wave_max[0][col];
#pragma unroll
        for (int w = 1; w < WAVES; w++) most = fmaxf(most, wave_max[w][col]);
        const bool none = !(most > -__builtin_inff());
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float half = none ? 1.0f : half_ratio(wave_max[w][col], most);
            total += wave_sum[w][col] * half * half;
        }
        const float mine = none ? 1.0f : __builtin_amdgcn_exp2f(m - most);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < kVpl; j += 4)
                *reinterpret_cast<floatx4 *>(joined + (((wave * 4 + i) * kVw + j / 4) * 64 + lane) * 4) =
                    floatx4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]} * mine;
        __syncthreads();
        if (wave >= 4) return;  // the columns are four waves' quarters
        float o[kVpl];
#pragma unroll
        for (int j = 0; j < kVpl; j += 4) {
            floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WAVES; w++)
                sum += *reinterpret_cast<const floatx4 *>(joined + (((w * 4 + wave) * kVw + j / 4) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; e++) o[j + e] = sum[e];
        }
        // this wave's quarter of the columns: d = VPL (4 g + wave) + j
        const int r = r0 + col, i = r / a.group, d = kVpl * (4 * g + wave);
        if (r >= rows || d >= dim) return;
        const int h = head * a.group + (r - i * a.group);
        if (a.splits > 1) {
            const int64_t at_row = ((s.row0 + i) * a.heads + h) * a.splits + split;
#pragma unroll
            for (int j = 0; j < kVpl; j += 4)
                *reinterpret_cast<floatx4 *>(a.part + at_row * dim + d + j) = floatx4{o[j], o[j + 1], o[j + 2], o[j + 3]};
            if (d == 0) {
                a.stats[2 * at_row] = most;
                a.stats[2 * at_row + 1] = total;
            }
        } else {
            T *y = static_cast<T *>(a.out) + (s.row0 + i) * a.out_stride + static_cast<int64_t>(h) * dim + d;
            const float r_total = total == 0.0f ? 0.0f : 1.0f / total;
            Vec<T, kVpl> v;
#pragma unroll
            for (int j = 0; j < kVpl; j++) v.v[j] = static_cast<T>(o[j] * r_total);
            __builtin_memcpy(y, v.v, sizeof(v.v));
        }
    }
}

// ---- many rows ---------------------------------------------------------------

constexpr int kTile = 64;  // tokens

// One workgroup: 128 rows (query, head of the group) of one sequence and kv
// head, 32 a wave, and one split of its tokens, 64 at a time.  The waves turn a
// tile's codes into fp16 in LDS together, K as [token][d] and V as [d][token],
// while they multiply the tile before.  Scores are taken transposed, S^T = K
// q^T, on 32x32 tiles: a lane holds 16 tokens' scores of one row, and these are
// the weights' operand of O^T = V^T P^T as they are, where V's tokens lie in
// the same order: the 16 tokens of a product as 0-3, 8-11 (lanes 0 .. 31), 4-7,
// 12-15 (lanes 32 .. 63).
template <typename T, int DP>
__global__ void __launch_bounds__(256, DP * sizeof(T) > 256 ? 1 : 2) attend_tiles(AttnArgs a) {
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int kParts = kWide ? 2 : 1;
    // 16 bytes past each row: any 16 rows' pieces of one column lie on different banks
    constexpr int kKPitch = DP * 2 + 16, kVPitch = kTile * 2 + 16;
    constexpr int kK = kTile * kKPitch, kV = DP * kVPitch;  // bytes
    constexpr int kKItems = (DP + 63) / 64, kVItems = (DP / 2 + 63) / 64;
    __shared__ __align__(16) int8_t lds[2 * (kK + kV)];
    __shared__ __align__(16) float scales[2][4][kTile];  // keys', values', what no one reads, log_scale() of the values'
    __shared__ __align__(16) unsigned held[2][4];  // kThere, and a bit for each of 16 tokens
    constexpr unsigned kThere = 1u << 16;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    const Place at_block = place(a);
    const int b = at_block.b, head = at_block.head, split = at_block.split, block = at_block.block;
    const int dim = a.c.head_dim;
    const Sequence s = sequence(a, b);
    const int rows = s.count * a.group, r0 = block * 128;
    if (r0 >= rows) return;
    const int first_q = r0 / a.group, last_q = (min(rows, r0 + 128) - 1) / a.group;
    int low = split * a.split_tokens, high = min(s.length, low + a.split_tokens);
    if (a.causal) {
        high = min(high, s.position + last_q + 1);
        low = max(low, window_from(a, s.position + first_q));
    }

    if (a.splits > 1 && low >= high) {
        nothing(a, s, head, split, r0, min(rows, r0 + 128));
        return;
    }

    // this wave's rows
    const int w0 = r0 + 32 * wave, r = w0 + col, i = r / a.group, q_head = head * a.group + (r - i * a.group);
    const bool in = r < rows;
    const int last = a.causal ? s.position + i : s.length - 1;
    const int start = window_from(a, last);
    const int wave_first = w0 / a.group, wave_last = (min(rows, w0 + 32) - 1) / a.group;  // queries
    // tokens that all of the wave's rows read
    const int all_from = window_from(a, s.position + wave_last);
    const int all_to = a.causal ? s.position + wave_first + 1 : s.length;

    half8_t qf[DP / 16][kParts];
    float factor;
    {
        // without a branch, so that all loads are on their way at once: rows past the last are the last
        const int rq = min(r, rows - 1), iq = rq / a.group;
        const T *q = static_cast<const T *>(a.q) + (s.row0 + iq) * a.q_stride + static_cast<int64_t>(head * a.group + (rq - iq * a.group)) * dim;
        float f[DP / 16][8];
        float top = 0.0f;
#pragma unroll
        for (int x = 0; x < DP / 16; x++) {
            const int d = 16 * x + 8 * h;
            load8(q + min(d, dim - 8), f[x]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f[x][e] = in && d < dim ? f[x][e] : 0.0f;
                top = fmaxf(top, fabsf(f[x][e]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        // an infinite query's scores are not finite whatever the codes, and all of -infinity would read as masked
        if (top == __builtin_inff()) f[0][0] = __builtin_nanf("");
        const int ex = top > 0.0f && top < __builtin_inff() ? ilogbf(top) : 0;
        const bool negative = a.scale < 0.0f;  // q takes the sign, so that the largest score has the largest product
        // above zero, since masked scores are -inf times it
        factor = fmaxf(ldexpf(fabsf(a.scale) * 1.44269504088896340736f, ex - 14), 0x1p-126f);
#pragma unroll
        for (int x = 0; x < DP / 16; x++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = ldexpf(negative ? -f[x][e] : f[x][e], 14 - ex);
                const _Float16 hi = static_cast<_Float16>(v);
                qf[x][0][e] = hi;
                if constexpr (kWide) qf[x][kParts - 1][e] = static_cast<_Float16>(v - static_cast<float>(hi));
            }
    }
    floatx16 acc[DP / 32];
#pragma unroll
    for (int j = 0; j < DP / 32; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[j][e] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;
    // A power of two above the value scales of a tile that every row of the wave reads, and its logarithm: what bounds
    // the sizes of every such tile whose scales lie between a sixteenth of it and itself, without a sum for each score.
    float top_scale = 0.0f, top_log = kLeastLog;

    struct Stage {
        uintx4 k[kKItems];
        unsigned v[kVItems][8];
        float scale;
    };
    const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
    const auto page_of = [&](int tile) {  // as the table has it: looked at when the tile is fetched
        const unsigned t = min(tile * kTile + 16 * wave, high - 1);
        return table[(static_cast<uint64_t>(t) * a.page_mul) >> a.page_shift];
    };
    const unsigned pages = static_cast<unsigned>(a.c.pages);
    const auto there = [&](int page) { return static_cast<unsigned>(page) < pages; };
    // This wave's 16 tokens of a tile.  Where a page is missing (its tokens are
    // masked) page 0 is read; codes past the head's, which meet zeros of q or
    // give columns that are not stored, are other codes of the token.
    unsigned k_at[kKItems], v_at[kVItems];
#pragma unroll
    for (int n = 0; n < kKItems; n++) {
        const int item = n * 64 + lane;
        k_at[n] = min(item / (DP / 16), 15) * dim + min(item % (DP / 16) * 16, dim - 16);
    }
#pragma unroll
    for (int n = 0; n < kVItems; n++) {
        const int item = n * 64 + lane;
        v_at[n] = min(item / (DP / 4), 1) * 4 * dim + min(item % (DP / 4) * 4, dim - 4);
    }
    // a token's row in the cache, in two parts: its page's first row (of this head), and the row in the page
    const int64_t page_rows = static_cast<int64_t>(a.c.kv_heads) * a.c.page_size;
    const int8_t *k_head = a.c.k + static_cast<int64_t>(head) * a.c.page_size * dim, *v_head = a.c.v + static_cast<int64_t>(head) * a.c.page_size * dim;
    const float *k_scale = a.c.k_scale + static_cast<int64_t>(head) * a.c.page_size, *v_scale = a.c.v_scale + static_cast<int64_t>(head) * a.c.page_size;
    const auto row_of = [&](int tile, int page) {
        const int t = tile * kTile + 16 * wave;
        const int page_at = static_cast<int>((static_cast<uint64_t>(static_cast<unsigned>(t)) * a.page_mul) >> a.page_shift);
        page = __builtin_amdgcn_readfirstlane(page);
        return (there(page) ? page : 0) * page_rows + (t - page_at * a.c.page_size);
    };
    // The lanes' offsets are added by the loads: sums made ahead of the loop would take two registers each.
    const auto fetch = [&](Stage &x, int tile, int page) {
        const int64_t row = row_of(tile, page);
        const int8_t *k = k_head + row * dim;
#pragma unroll
        for (int n = 0; n < kKItems; n++) {
            asm("" : "+v"(k_at[n]));
            x.k[n] = *reinterpret_cast<const uintx4 *>(k + k_at[n]);
        }
        // lanes 0 .. 15: key scales, 16 .. 31: value scales; zeros for tokens outside the range
        const int token = tile * kTile + 16 * wave + (lane & 15);
        x.scale = ((lane & 16) == 0 ? k_scale : v_scale)[row + (lane & 15)];
        if (!there(page) || token < low || token >= high) x.scale = 0.0f;
        const int8_t *v = v_head + row * dim;
#pragma unroll
        for (int n = 0; n < kVItems; n++) asm("" : "+v"(v_at[n]));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int8_t *ve = v + (e / 4 * 8 + e % 4) * dim;
#pragma unroll
            for (int n = 0; n < kVItems; n++) x.v[n][e] = *reinterpret_cast<const unsigned *>(ve + v_at[n]);
        }
    };
    // V's rows lie in the order d = 0, 4, 8 .., 1, 5, 9 ..: lanes next to each
    // other write rows next to each other, and a lane's sums are runs of four d.
    const auto put = [&](const Stage &x, int buffer, int page) {
        int8_t *k = lds + buffer * kK, *v = lds + 2 * kK + buffer * kV;
#pragma unroll
        for (int n = 0; n < kKItems; n++) {
            const int item = n * 64 + lane, at = item / (DP / 16), piece = item % (DP / 16) * 2;
            if (DP == 96 && at >= 16) continue;
#pragma unroll
            for (int e = 0; e < 2; e++)
                *reinterpret_cast<half8_t *>(k + (16 * wave + at) * kKPitch + (piece + e) * 16) = codes8(x.k[n][2 * e], x.k[n][2 * e + 1]);
        }
        // a token with a scale that is not finite is one of the bits of `held`, and the scale 0 in the product
        const bool odd = !(fabsf(x.scale) < __builtin_inff());
        const unsigned both = static_cast<unsigned>(__ballot(odd)), odds = (both | both >> 16) & (kThere - 1);
        const float scale = odd ? 0.0f : x.scale;
        scales[buffer][lane / 16][16 * wave + lane % 16] = lane < 48 ? scale : log_scale(scale);
        held[buffer][wave] = there(page) ? kThere | odds : 0;
#pragma unroll
        for (int n = 0; n < kVItems; n++) {
            const int item = n * 64 + lane, dq = item % (DP / 4), half = item / (DP / 4);
            if (DP < 128 && half >= 2) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned sel = 0x0c000c00u | ((4u + e) << 16) | e;
                const half8_t y = join(codes_to_half(x.v[n][1], x.v[n][0], sel), codes_to_half(x.v[n][3], x.v[n][2], sel),
                                       codes_to_half(x.v[n][5], x.v[n][4], sel), codes_to_half(x.v[n][7], x.v[n][6], sel));
                *reinterpret_cast<half8_t *>(v + (e * (DP / 4) + dq) * kVPitch + (2 * wave + half) * 16) = y;
            }
        }
    };
    floatx16 sc[2];
    const auto scores = [&](int buffer) {
        const int8_t *k = lds + buffer * kK;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) sc[t][e] = 0.0f;
#pragma unroll
        for (int x = 0; x < DP / 16; x++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const half8_t kf = *reinterpret_cast<const half8_t *>(k + (32 * t + col) * kKPitch + (2 * x + h) * 16);
#pragma unroll
                for (int w = 0; w < kParts; w++) sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[x][w], sc[t], 0, 0, 0);
            }
    };
    const auto add_values = [&](int buffer, const half8_t (&pf)[4][kParts]) {
        const int8_t *v = lds + 2 * kK + buffer * kV;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int j = 0; j < DP / 32; j++) {
                const half8_t vf = *reinterpret_cast<const half8_t *>(v + (32 * j + col) * kVPitch + (2 * g + h) * 16);
#pragma unroll
                for (int w = 0; w < kParts; w++) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[g][w], acc[j], 0, 0, 0);
            }
    };
    const auto weights = [&](int buffer, int tile, half8_t (&pf)[4][kParts]) {
        const uintx4 bits = *reinterpret_cast<const uintx4 *>(held[buffer]);
        unsigned ok[4];
#pragma unroll
        for (int e = 0; e < 4; e++) ok[e] = __builtin_amdgcn_readfirstlane(bits[e]);
        const bool plain = ok[0] == kThere && ok[1] == kThere && ok[2] == kThere && ok[3] == kThere;
        const int at = tile * kTile;
        // every row of the wave reads every token of the tile
        const bool clear = at >= low && at + kTile <= high && at >= all_from && at + kTile <= all_to && plain;
        float most = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const floatx4 ks = *reinterpret_cast<const floatx4 *>(&scales[buffer][0][32 * t + 2 * e + 4 * h]);
#pragma unroll
                for (int u = 0; u < 4; u++) sc[t][e + u] *= ks[u];
            }
        if (!clear) {
            // this lane's first and last token of the tile, counted from its first one there
            const int from_at = max(low, start) - at - 4 * h, to_at = min(high - 1, last) - at - 4 * h;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int token = 32 * t + 8 * (e / 4) + e % 4;
                    const bool keep = token >= from_at && token <= to_at && (ok[2 * t + e / 8] & kThere);
                    sc[t][e] = keep ? sc[t][e] : -__builtin_inff();
                }
            if ((ok[0] | ok[1] | ok[2] | ok[3]) & (kThere - 1)) {  // NaN for the rows that read such a token, and only those
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if ((ok[2 * t + e / 8] >> (8 * (e / 4 % 2) + 4 * h + e % 4) & 1) && sc[t][e] != -__builtin_inff()) sc[t][e] = __builtin_nanf("");
            }
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) most = fmaxf(most, sc[t][e]);
        const float value = scales[buffer][1][lane];
        const auto fits = [&]() { return value <= top_scale && value * 16.0f >= top_scale; };
        float size = __builtin_fmaf(most, factor, top_log);
        if (!clear || __any(!fits() || size > m + (kLift + kSlack))) {
            bool even = clear && __all(fits());
            if (clear && !even) {
                const unsigned half = max_over<32>(abs_bits(value));
                const unsigned up = max(__builtin_amdgcn_readlane(half, 0), __builtin_amdgcn_readlane(half, 32));
                top_log = ceilf(log_scale(__uint_as_float(up)));
                top_scale = ldexpf(1.0f, static_cast<int>(top_log));
                size = __builtin_fmaf(most, factor, top_log);
                even = __all(fits());
            }
            if (!even) {
                size = -__builtin_inff();
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const floatx4 logs = *reinterpret_cast<const floatx4 *>(&scales[buffer][3][32 * t + 2 * e + 4 * h]);
#pragma unroll
                        for (int u = 0; u < 4; u++) size = fmaxf(size, __builtin_fmaf(sc[t][e + u], factor, logs[u]));
                    }
            }
            // a row whose own sizes have not passed keeps its base
            size = fmaxf(size, __shfl_xor(size, 32));
            const float now = size > m + (kLift + kSlack) ? size - kLift : m;
            const float half = half_ratio(m, now);
            m = now;
            l = l * half * half;
#pragma unroll
            for (int j = 0; j < DP / 32; j++) acc[j] *= half * half;
        }
        const float from = m > -__builtin_inff() ? -m : 0.0f;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const floatx4 vs = *reinterpret_cast<const floatx4 *>(&scales[buffer][1][32 * t + 2 * e + 4 * h]);
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e + u], factor, from));
                    l += p;
                    float w = p * vs[u];
                    if constexpr (kWide) once(w);
                    const _Float16 hi = static_cast<_Float16>(w);
                    pf[2 * t + e / 8][0][e % 8 + u] = hi;
                    if constexpr (kWide) pf[2 * t + e / 8][kParts - 1][e % 8 + u] = static_cast<_Float16>(w - static_cast<float>(hi));
                }
            }
    };

    const int first = max(low, 0) / kTile, end = high > low ? (high + kTile - 1) / kTile : 0;
    if (first < end) {
        Stage x;
        int page = page_of(first), then = page_of(first + 1), later = page_of(first + 2);
        fetch(x, first, page);
        put(x, first & 1, page);
        fetch(x, min(first + 1, end - 1), then);
        __syncthreads();
        // the next tile is turned while this one's scores are multiplied, the one after it is loaded meanwhile
        for (int tile = first; tile < end; tile++) {
            scores(tile & 1);
            put(x, ~tile & 1, then);
            fetch(x, min(tile + 2, end - 1), later);
            then = later;
            later = page_of(tile + 3);
            half8_t pf[4][kParts];
            weights(tile & 1, tile, pf);
            add_values(tile & 1, pf);
            __syncthreads();
        }
    }

    // the sum of d = 32 q + 16 h + 4 u + e
    const auto sum = [&](int q, int u, int e) { return acc[(e * (DP / 32) + q) / 4][(e * (DP / 32) + q) % 4 * 4 + u]; };
    l += __shfl_xor(l, 32);
    if (a.splits > 1) {
        if (!in) return;
        const int64_t at_row = ((s.row0 + i) * a.heads + q_head) * a.splits + split;
#pragma unroll
        for (int q = 0; q < DP / 32; q++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int d = 32 * q + 16 * h + 4 * u;
                if (d < dim) *reinterpret_cast<floatx4 *>(a.part + at_row * dim + d) = floatx4{sum(q, u, 0), sum(q, u, 1), sum(q, u, 2), sum(q, u, 3)};
            }
        if (h == 0) {
            a.stats[2 * at_row] = m;
            a.stats[2 * at_row + 1] = l;
        }
        return;
    }
    // Through this wave's part of LDS, 32 of d at a time, to 16-byte pieces: the
    // part of K, which every wave is past; V's last tile may still be read.
    constexpr int kPitch = 32 + 16 / static_cast<int>(sizeof(T)), kPiece = 16 / static_cast<int>(sizeof(T));
    T *turn = reinterpret_cast<T *>(lds + wave * (kK / 2));
    static_assert(32 * kPitch * sizeof(T) <= kK / 2, "a wave's part of LDS holds 32 rows of 32");
    const float part = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < DP / 32; j++) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float o[4] = {sum(j, u, 0) * part, sum(j, u, 1) * part, sum(j, u, 2) * part, sum(j, u, 3) * part};
            put_floats<4>(turn + col * kPitch + 16 * h + 4 * u, o);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        constexpr int kLanes = 32 / kPiece;
#pragma unroll
        for (int y = 0; y < 32; y += 64 / kLanes) {
            const int row = y + lane / kLanes, c = lane % kLanes * kPiece, d = 32 * j + c;
            const int rr = w0 + row, ii = rr / a.group;
            if (rr < rows && d < dim) {
                const Vec<T, kPiece> o = *reinterpret_cast<const Vec<T, kPiece> *>(turn + row * kPitch + c);
                T *out = static_cast<T *>(a.out) + (s.row0 + ii) * a.out_stride + static_cast<int64_t>(head * a.group + rr - ii * a.group) * dim + d;
                __builtin_memcpy(out, o.v, sizeof(o.v));
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// A wave a row of q and head: its splits' sums, joined in their order.  A lane
// takes one split's base and total, so that these come by one load, and four
// splits' sums at a time.
template <typename T>
__global__ void __launch_bounds__(256) join_splits(AttnArgs a) {
    const int head = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int b = blockIdx.x / a.max_queries, i = blockIdx.x - b * a.max_queries;
    if (head >= a.heads) return;
    const Sequence s = sequence(a, b);
    if (i >= s.count) return;
    const int64_t at = ((s.row0 + i) * a.heads + head) * a.splits;
    const int dim = a.c.head_dim;
    float most = -__builtin_inff();
    for (int p = lane; p < a.splits; p += 64) most = fmaxf(most, a.stats[2 * (at + p)]);
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    const bool none = !(most > -__builtin_inff());
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, total = 0.0f;
    for (int p0 = 0; p0 < a.splits; p0 += 64) {
        float half = 0.0f, sum = 0.0f;
        if (p0 + lane < a.splits) {
            sum = a.stats[2 * (at + p0 + lane) + 1];
            half = none ? 1.0f : half_ratio(a.stats[2 * (at + p0 + lane)], most);
        }
        const int end = min(64, a.splits - p0);
        for (int p = 0; p < end; p += 4) {
            float part[4][4], r[4], c[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                r[u] = __shfl(half, p + u);
                c[u] = __shfl(sum, p + u);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int d = lane + 64 * e;
                    // no sums where a split holds no token of the row's
                    part[u][e] = p + u < end && c[u] != 0.0f && d < dim ? a.part[(at + p0 + p + u) * dim + d] : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (c[u] == 0.0f) continue;
                total += c[u] * r[u] * r[u];
                r[u] *= r[u];
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] += r[u] * part[u][e];
            }
        }
    }
    T *y = static_cast<T *>(a.out) + (s.row0 + i) * a.out_stride + static_cast<int64_t>(head) * dim;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (lane + 64 * e < dim) y[lane + 64 * e] = static_cast<T>(total == 0.0f ? 0.0f : o[e] / total);
}

struct Plan {
    bool wide;  // 128 rows a workgroup (attend_tiles), otherwise 16 (attend_rows)
    int waves;  // of attend_rows
    int64_t row_blocks;  // up to 2^36: queries and heads are bounded
    int split_tokens, splits;
    size_t part, stats;  // bytes
};

Plan plan(const Spkv2KvCacheI8 &c, const Spkv2AttentionI8 &g) {
    Plan p;
    const int64_t rows = std::min(g.max_queries, g.queries) * (g.heads / c.kv_heads);
    // attend_tiles reads a tile of tokens once for 128 rows, attend_rows for 16,
    // but spreads few tokens over more waves.  Where 16 rows do not hold them
    // all, rows times tokens of all sequences and kv heads decide (us, rows'
    // kernel against tiles'): 192 x 32 K 30 and 35, 120 x 64 K 28 and 33, 32 x
    // 256 K 36 and 34, 192 x 48 K 38 and 34, 40 x 1 M 125 and 85.
    p.wide = rows > 16 && static_cast<double>(rows) * g.sequences * c.kv_heads * g.max_length > 8e6;
    p.row_blocks = p.wide ? (rows + 127) / 128 : (rows + 15) / 16;
    // Enough workgroups for eight on each CU (two where they take 128 rows), and
    // no split shorter than four chunks for each of four waves (two tiles): a
    // second kernel costs more than a few steps do.  Fewer workgroups than CUs
    // are of eight waves: one sequence of 333
    // tokens 13.1 us with four, 12.2 with eight.
    const int64_t base = g.sequences * c.kv_heads * p.row_blocks;
    const int64_t step = 128, least = p.wide ? 128 : 512;
    int64_t splits = std::min<int64_t>(p.wide ? 512 / base : (2048 + base - 1) / base, (g.max_length + least - 1) / least);
    splits = std::max<int64_t>(splits, 1);
    int64_t tokens = (g.max_length + splits - 1) / splits;
    tokens = std::max<int64_t>((tokens + step - 1) / step * step, step);
    p.split_tokens = static_cast<int>(tokens);
    p.splits = static_cast<int>(std::max<int64_t>((g.max_length + tokens - 1) / tokens, 1));
    p.waves = base * p.splits <= 256 ? 8 : 4;
    const size_t parts = p.splits > 1 ? static_cast<size_t>(g.queries) * g.heads * p.splits : 0;
    p.part = parts * c.head_dim * sizeof(float);
    p.stats = parts * 2 * sizeof(float);
    return p;
}

int check(const Spkv2KvCacheI8 *c, const Spkv2AttentionI8 *g) {
    if (int rc = check_cache(c)) return rc;
    if (!g) return bad("attention_i8: no arguments");
    if (!is_dtype(g->dtype)) return bad("attention_i8: unknown dtype");
    if (g->queries < 0 || g->sequences < 0 || g->table_width < 0 || g->max_queries < 0 || g->max_length < 0)
        return bad("attention_i8: negative size");
    if (g->heads < 1 || g->heads % c->kv_heads) return bad("attention_i8: heads is not a multiple of kv_heads");
    if (g->window < 0 || (g->window && !g->causal)) return bad("attention_i8: window is negative, or not causal");
    if (std::min(g->max_queries, g->queries) * (g->heads / c->kv_heads) > (1 << 30))
        return unsupported("attention_i8: more than 2^30 rows of one sequence and kv head");
    if (g->queries > (1 << 24) || g->heads > 65535 || g->sequences > 65535 || g->max_length > (1 << 30))
        return unsupported("attention_i8: more than 2^24 queries, 65535 heads or sequences, or 2^30 tokens");
    return 0;
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_attention_i8_workspace(const Spkv2KvCacheI8 *c, const Spkv2AttentionI8 *g, size_t *size) {
    return entry([&]() -> int {
        if (!size) return bad("attention_i8: nowhere to put the size");
        if (int rc = check(c, g)) return rc;
        *size = 0;
        if (g->queries == 0 || g->sequences == 0 || g->max_queries == 0) return 0;
        const Plan p = plan(*c, *g);
        *size = p.part + p.stats;
        return 0;
    });
}

extern "C" int spkv2_mi355x_attention_i8_kernel_name(const Spkv2KvCacheI8 *c, const Spkv2AttentionI8 *g, char *buf, size_t buf_size) {
    return entry([&]() -> int {
        if (!buf || !buf_size) return bad("attention_i8: nowhere to put the name");
        if (int rc = check(c, g)) return rc;
        buf[0] = 0;
        if (g->queries == 0 || g->sequences == 0 || g->max_queries == 0) return 0;
        const Plan p = plan(*c, *g);
        if (p.wide) snprintf(buf, buf_size, "attend_tiles<splits=%d>", p.splits);
        else snprintf(buf, buf_size, "attend_rows<waves=%d,splits=%d>", p.waves, p.splits);
        return 0;
    });
}

extern "C" int spkv2_mi355x_attention_i8(const Spkv2KvCacheI8 *c, const Spkv2AttentionI8 *g, void *stream) {
    return entry([&]() -> int {
        if (int rc = check(c, g)) return rc;
        if (g->queries == 0 || g->sequences == 0 || g->max_queries == 0) return 0;
        if (!g->q || !g->out || !g->lengths || !g->offsets || (!g->table && g->table_width))
            return bad("attention_i8: a NULL pointer");
        const int64_t width = static_cast<int64_t>(g->heads) * c->head_dim;
        if (g->queries > 1 && (g->q_stride < width || g->out_stride < width))
            return bad("attention_i8: a stride is below the heads' width");
        const Plan p = plan(*c, *g);
        if (p.splits > 1 && (!g->workspace || g->workspace_size < p.part + p.stats || !aligned(g->workspace, 16)))
            return bad("attention_i8: the workspace is missing, too small or not 16-byte aligned");
        // a launch has fewer than 2^32 threads
        if (g->sequences * p.row_blocks >= (1 << 23) / c->kv_heads / p.splits ||
            (p.splits > 1 && g->sequences * std::min(g->max_queries, g->queries) >= (1 << 24)))
            return unsupported("attention_i8: too many queries and sequences for one launch");
        unsigned mul;
        int shift;
        div_magic(static_cast<unsigned>(c->page_size), &mul, &shift);
        AttnArgs a{*c, g->q, g->out, g->table, g->lengths, g->offsets, static_cast<float *>(g->workspace),
                   reinterpret_cast<float *>(static_cast<char *>(g->workspace) + p.part), g->queries, g->q_stride, g->out_stride,
                   static_cast<int>(std::min<int64_t>(g->max_queries, g->queries)), static_cast<int>(g->max_length), g->table_width, g->heads,
                   g->heads / c->kv_heads, g->sequences, g->causal, g->window, g->scale, static_cast<int>(p.row_blocks), p.split_tokens, p.splits,
                   mul, shift};
        const unsigned blocks = static_cast<unsigned>(g->sequences * p.row_blocks * p.splits);
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            const char *what = "attention_i8";
            auto many = [&](auto kernel) { return launch(what, kernel, dim3(blocks * c->kv_heads), dim3(256), stream, a); };
            auto few = [&](auto four, auto eight) {
                return launch(what, p.waves == 8 ? eight : four, dim3(blocks * c->kv_heads), dim3(64 * p.waves), stream, a);
            };
            const int dim = c->head_dim;
            int rc;
            if (p.wide) {
                rc = dim <= 64    ? many(attend_tiles<T, 64>)
                     : dim <= 96  ? many(attend_tiles<T, 96>)
                     : dim <= 128 ? many(attend_tiles<T, 128>)
                                  : many(attend_tiles<T, 256>);
            } else {
                rc = dim <= 64    ? few(attend_rows<T, 64, 4>, attend_rows<T, 64, 8>)
                     : dim <= 128 ? few(attend_rows<T, 128, 4>, attend_rows<T, 128, 8>)
                                  : few(attend_rows<T, 256, 4>, attend_rows<T, 256, 8>);
            }
            if (rc || p.splits == 1) return rc;
            const dim3 rows(static_cast<unsigned>(g->sequences * a.max_queries), (g->heads + 3) / 4);
            return launch(what, join_splits<T>, rows, dim3(256), stream, a);
        });
    });
}
