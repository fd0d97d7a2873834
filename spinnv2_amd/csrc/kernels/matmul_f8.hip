// Products of rows and weights in 8-bit floats with a scale for each block of
// 128: of a row's columns, and of 128 x 128 weights.
//
//   out[m, n] = sum_t sa[m, t] sb[n / 128, t] sum_{k in block t} a[m, k] b[n, k] + bias[n]
//
// A block of 128 is one matrix instruction's depth (16 x 16 x 128), so each of
// them starts from zero and its sums are scaled and added in fp32.
//
// The 8-bit float matrix cores add eight products at a time and keep 13 bits
// below the largest of them: a sum may be off by 2^-10 of the largest product of
// every eight, at random by 4e-5 of its size, which 16-bit outputs, with 2^-9 and
// 2^-12 of their own, hardly show.  fp32 outputs would (1.1e-5 relative where fp32
// sums leave 3e-7), so theirs are computed on the fp16 cores, whose operands hold
// 8-bit floats exactly, at half the rate: a caller chooses by the output's type.
//
// Many rows are bound by the matrix cores, at the clock that random operands leave
// them: 8192 x 8192 x 8192 into bf16 408 to 460 us, 2.4 to 2.7 PFLOP/s, the cores at
// work in 61% of the cycles (a library's product, one scale for a whole matrix, 423),
// into fp32 908, 1.2 PFLOP/s.
// Few rows are bound by the bytes of the weights: 1 x 4096 x 4096 4.6 to 5.8 us, a
// launch's own time and 2.9 to 3.6 TB/s; 64 tokens of 8 experts of 64, 2048 x 2048,
// 46 to 55 us, 4.8 to 5.9 TB/s.  32 to 300 rows are bound by a workgroup's walk along k
// and by weights read once for each 16 to 64 rows: 64 x 4096 x 4096 7.9 us, 256 x 4096 x
// 14336 33.  Rows by expert leave part of each expert's last tile empty and look their
// rows up ahead of the loop: 4001 tokens of 4 of 32, 4096 x 2048, 172 to 177 us, where
// the products alone would take 103.
#include <cmath>
#include <cstdio>

#include "decoder.hpp"

namespace spk::dec {

namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));

struct MatmulArgs {
    const uint8_t *a, *b;
    const float *a_scale, *b_scale, *bias;
    void *out;
    int64_t a_stride, b_stride, out_stride, sa_stride, sb_stride;
    int m, n, k, n_tiles;
    // by expert
    const int32_t *offsets, *order;
    int64_t a_rows, b_expert, sb_expert;
    int experts, most_down;  // workgroups along the rows at most
    unsigned token_mul;  // choice / per_token, by multiplication
    int token_shift;
};

// 16 bytes at p, of which `left` are inside the row: zeros past them
__device__ __forceinline__ intx4 part16(const uint8_t *p, int left) {
    intx4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (i < left) v[i / 4] |= static_cast<int>(static_cast<unsigned>(p[i]) << (8 * (i % 4)));
    return v;
}
__device__ __forceinline__ intx4 load16(const uint8_t *p, int64_t at) {
    intx4 v;
    __builtin_memcpy(&v, p + at, 16);
    return v;
}
// a mask of 16 bytes without the first `cut`
__device__ __forceinline__ intx4 behind(int cut) {
    intx4 keep;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int c = min(max(cut - 4 * e, 0), 4);
        keep[e] = c == 4 ? 0 : static_cast<int>(~0u << (8 * c));
    }
    return keep;
}

// LDS of one wave alone: its writes are done before its reads, and the other way round
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 16 rows' operand of the matrix cores: 32 of 128 columns a lane, 16 bytes from
// 16 (lane / 16) and as many from there + 64 (any order will do that both operands
// have).  WIDE: turned into fp16.
template <bool WIDE>
struct Operand {
    intx8 v;
    __device__ __forceinline__ void set(intx4 low, intx4 high) { v = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7); }
};
template <>
struct Operand<true> {
    half8_t v[4];
    __device__ __forceinline__ void set(intx4 low, intx4 high) {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const intx4 &from = p < 2 ? low : high;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(from[2 * (p % 2) + e], 1.0f, false);
                const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(from[2 * (p % 2) + e], 1.0f, true);
                v[p][4 * e] = a.x, v[p][4 * e + 1] = a.y, v[p][4 * e + 2] = b.x, v[p][4 * e + 3] = b.y;
            }
        }
    }
};
// The sums of 16 rows of `x` and 16 of `y` over 128 columns: row e of a lane's
// four is x's row 4 (lane / 16) + e, the column y's row lane % 16.
__device__ __forceinline__ floatx4 product(const Operand<false> &x, const Operand<false> &y) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.v, y.v, floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ floatx4 product(const Operand<true> &x, const Operand<true> &y) {
    floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < 4; p++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v[p], y.v[p], sum, 0, 0, 0);
    return sum;
}

// Sums over a wave's lanes up to each, by lane moves: an LDS shuffle in their place waits for LDS six times
__device__ __forceinline__ int sums_through(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // a row of 16 lanes, 1 lane on
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the last lane of rows 0 and 2 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 to rows 2 and 3
    return v;
}

// Rows first .. end of one expert's that a workgroup of `height` rows takes
struct Rows {
    int expert, first, end;
};
// 64 experts, one a lane: their rows, and workgroups of `height` of them, counted with those of the lanes before
struct Experts {
    int low, high, tiles, through;
};
__device__ __forceinline__ Experts experts_from(const MatmulArgs &a, int e0, int height) {
    const int e = e0 + (threadIdx.x & 63);
    Experts x{0, 0, 0, 0};
    if (e < a.experts) {
        x.low = min(max(a.offsets[e], 0), a.m);
        x.high = min(max(a.offsets[e + 1], x.low), a.m);
    }
    x.tiles = (x.high - x.low + height - 1) / height;
    x.through = sums_through(x.tiles);
    return x;
}
__device__ __forceinline__ int tiles_of(const Experts &x) { return __builtin_amdgcn_readlane(x.through, 63); }
// The workgroups of all experts' rows, one expert's after the other's: which of
// them is number `at`, `x` the first 64 experts; expert -1 where there are fewer.
__device__ __forceinline__ Rows rows_of(const MatmulArgs &a, Experts x, int at, int height) {
    for (int e0 = 0;;) {
        const uint64_t past = __ballot(x.through > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            Rows r;
            r.expert = e0 + l;
            const int before = __builtin_amdgcn_readlane(x.through, l) - __builtin_amdgcn_readlane(x.tiles, l);
            r.first = __builtin_amdgcn_readlane(x.low, l) + (at - before) * height;
            r.end = min(__builtin_amdgcn_readlane(x.high, l), r.first + height);
            return r;
        }
        at -= tiles_of(x);
        e0 += 64;
        if (e0 >= a.experts) return Rows{-1, 0, 0};
        x = experts_from(a, e0, height);
    }
}
// the choice that output row r is, and the row of a that it takes (negative: none, or one that a may not have)
__device__ __forceinline__ int choice_of(const MatmulArgs &a, int r) { return a.order ? a.order[r] : r; }
__device__ __forceinline__ int row_of(const MatmulArgs &a, int choice) {
    if (!a.order) return choice;
    return choice < 0 ? -1 : static_cast<int>((static_cast<uint64_t>(static_cast<unsigned>(choice)) * a.token_mul) >> a.token_shift);
}

// 16 TM tokens x 16 TN channels a workgroup, whose waves deal k out among them,
// a block at a time, and join their sums in LDS.  A wave loads eight rows' 128
// bytes an instruction and turns them in LDS of its own into the matrix cores'
// order (16 rows' 16 bytes): loaded in that order, neighbouring lanes are
// different rows and each is a request of its own.
template <typename T, bool EXPERTS, int TM, int TN>
__global__ void __launch_bounds__(512) matmul_rows(MatmulArgs a) {
    constexpr int WAVES = 8;
    constexpr int kPieces = 2 * (TM + TN);  // loads of eight rows a block: 2 TM of a, then 2 TN of b
    constexpr int kAhead = kPieces <= 4 ? 4 : kPieces <= 8 ? 2 : 1;  // blocks loaded together
    constexpr int kTurn = (kPieces > TM * TN ? kPieces : TM * TN) * 1024;
    __shared__ __align__(16) uint8_t lds[WAVES * kTurn];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * TN;
    int m0 = blockIdx.y * 16 * TM, end_m = a.m, expert = 0;
    if constexpr (EXPERTS) {
        const Rows r = rows_of(a, experts_from(a, 0, 16 * TM), blockIdx.y, 16 * TM);
        if (r.expert < 0) return;
        expert = r.expert;
        m0 = r.first;
        end_m = r.end;
    }
    const uint8_t *b = a.b + expert * a.b_expert;
    // the row of a that output row r takes; -1: none
    const auto input = [&](int r) -> int64_t {
        r = min(r, end_m - 1);
        if constexpr (!EXPERTS) return r;
        const int at = row_of(a, choice_of(a, r));
        return at < a.a_rows ? at : -1;
    };
    const int blocks = (a.k + 127) / 128, per = (blocks + WAVES - 1) / WAVES;
    const int first = wave * per, end = min(first + per, blocks);
    const uint8_t *p[kPieces];
#pragma unroll
    for (int c = 0; c < kPieces; c++)
        p[c] = c < 2 * TM ? a.a + max(input(m0 + 8 * c + lane / 8), int64_t(0)) * a.a_stride : b + min(n0 + 8 * (c - 2 * TM) + lane / 8, a.n - 1) * a.b_stride;
    const float *sa[TM], *sb = a.b_scale + expert * a.sb_expert + n0 / 128 * a.sb_stride;
    bool there[TM];
#pragma unroll
    for (int j = 0; j < TM; j++) {
        const int64_t row = input(m0 + 16 * j + col);
        there[j] = row >= 0;
        sa[j] = a.a_scale + max(row, int64_t(0)) * a.sa_stride;
    }
    uint8_t *turn = lds + wave * kTurn;
    const int put_at = lane / 8 * 128;
    floatx4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    struct Block {
        intx4 v[kPieces];
        float sa[TM], sb;
    };
    auto fetch = [&](Block &x, int s) {
        const int k = s * 128 + lane % 8 * 16;
        if (s * 128 + 128 <= a.k) {
#pragma unroll
            for (int c = 0; c < kPieces; c++) x.v[c] = load16(p[c], k);
        } else if (a.k >= 16) {
            // pieces past the row's end are its last 16 bytes, cleared where another piece has them
            const int at = min(k, a.k - 16);
            const intx4 keep = behind(k - at);
#pragma unroll
            for (int c = 0; c < kPieces; c++) x.v[c] = load16(p[c], at) & keep;
        } else {
#pragma unroll
            for (int c = 0; c < kPieces; c++) x.v[c] = part16(p[c], lane % 8 == 0 ? a.k : 0);
        }
#pragma unroll
        for (int j = 0; j < TM; j++) x.sa[j] = sa[j][s];
        x.sb = sb[s];
    };
    auto multiply = [&](const Block &x) {
        // row r's piece lies at place piece ^ (r / 2 % 8): any 16 rows' pieces of one column are then on different banks
#pragma unroll
        for (int c = 0; c < kPieces; c++)
            *reinterpret_cast<intx4 *>(turn + c * 1024 + put_at + ((lane % 8) ^ ((c * 4 + lane / 16) & 7)) * 16) = x.v[c];
        wait_lds();
        Operand<sizeof(T) == 4> fa[TM], fb[TN];
        const auto read = [&](int c, int kk) { return *reinterpret_cast<const intx4 *>(turn + c * 2048 + col * 128 + ((4 * kk + g) ^ (col / 2)) * 16); };
#pragma unroll
        for (int j = 0; j < TM; j++) fa[j].set(read(j, 0), read(j, 1));
#pragma unroll
        for (int i = 0; i < TN; i++) fb[i].set(read(TM + i, 0), read(TM + i, 1));
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++) {
                const floatx4 sum = product(fb[i], fa[j]);
                const float scale = x.sa[j] * x.sb;
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(scale, sum[e], acc[i][j][e]);
            }
        wait_lds();
    };
    Block now[kAhead], next[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++)
        if (first + u < end) fetch(now[u], first + u);
    for (int s = first; s < end; s += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (s + kAhead + u < end) fetch(next[u], s + kAhead + u);
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (s + u < end) multiply(now[u]);
            now[u] = next[u];
        }
    }
    // where the wave turned its operands
    auto sums = [&](int w, int i, int j) -> floatx4 & { return *reinterpret_cast<floatx4 *>(lds + w * kTurn + ((i * TM + j) * 64 + lane) * 16); };
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) sums(wave, i, j) = there[j] ? acc[i][j] : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
    for (int t = wave; t < TM * TN; t += WAVES) {
        const int i = t / TM, j = t % TM;
        floatx4 total = sums(0, i, j);
#pragma unroll
        for (int w = 1; w < WAVES; w++) total += sums(w, i, j);
        const int m = m0 + 16 * j + col, n = n0 + 16 * i + 4 * g, left = a.n - n;
        if (m >= end_m || left <= 0) continue;
        float v[4] = {total[0], total[1], total[2], total[3]};
        if (a.bias) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += a.bias[static_cast<int64_t>(expert) * a.n + min(n + e, a.n - 1)];
        }
        store_some<4>(static_cast<T *>(a.out) + m * a.out_stride + n, left, v);
    }
}

// 16 bytes a lane from base + offset into LDS, lane after lane from `to` on,
// which is one for the wave.  The builtin for it makes the next read of any LDS
// wait for the load; here wait_all() does, ahead of the reads of what was loaded.
__device__ __forceinline__ unsigned lds_address(const void *p) {
    return static_cast<unsigned>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)p));
}
__device__ __forceinline__ void load_lds16(const void *base, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
// A barrier ahead of which every wave's loads into LDS have arrived.
__device__ __forceinline__ void wait_all() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

constexpr int kCus = 256;
// whether tiles leave room for one workgroup on a CU, which then takes one after the other
constexpr bool goes_on(bool direct, int channels) { return direct && channels == 256; }

// WAVES_M x WAVES_N waves, each TJ x TI tiles of 16 x 16 (rows by channels), take
// a block of k a step; where such tiles are few, WAVES_K groups of them take a
// block each and join their sums in the end.
//
// DIRECT: rows are whole runs of 16 bytes, which are loaded into one of two
// buffers of LDS while the other is multiplied (a third and a fourth gained nothing:
// what a CU can have under way is the limit).  Otherwise they wait in registers
// for a step between memory and LDS, at 1.5 to 1.9 times the time of a step.
//
// Tiles so large that a CU holds one workgroup go on (kGoOn): the next tile's rows
// are looked up ahead of a tile's loop, and its first block is under way while the
// tile leaves, in two halves, through the buffer that the block does not take (4001
// tokens of 4 of 32 experts, 4096 x 2048, 187 -> 175 us, 16384 x 8192 x 128 68 -> 56).
template <typename T, bool EXPERTS, bool DIRECT, int WAVES_M, int WAVES_N, int WAVES_K, int TJ, int TI>
__global__ void __launch_bounds__(64 * WAVES_M *WAVES_N *WAVES_K, TJ *TI >= 16 ? 2 : sizeof(T) == 4 || WAVES_N == 4 ? 3 : 4)
    matmul_tiles(MatmulArgs a) {
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int kWaves = WAVES_M * WAVES_N, kThreads = 64 * kWaves;  // of a group
    constexpr int BM = 16 * TJ * WAVES_M, BN = 16 * TI * WAVES_N, BK = 128;
    constexpr int kA = BM * 8 / kThreads, kB = BN * 8 / kThreads, kPieces = kA + kB;  // 16-byte pieces a thread
    constexpr int kPart = (BM + BN) * BK, kBuffer = kPart * WAVES_K;
    constexpr int kScales = BM < 64 ? 64 : BM;
    __shared__ __align__(16) uint8_t lds[2 * kBuffer];
    __shared__ __align__(16) float row_scales[2][kScales][4];  // of four blocks of k
    constexpr bool kGoOn = goes_on(DIRECT, BN);
    __shared__ bool row_there[kGoOn ? 2 : 1][EXPERTS ? kScales : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWaves;
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads), tid = wave * 64 + lane;
    const int col = lane & 15, g = lane >> 4;
    // Workgroups go to the eight XCDs in turn; each XCD takes a run of tiles,
    // four tiles of rows by the channels one after the other, whose operands
    // its L2 then holds for several of them.
    int m_tiles = (a.m + BM - 1) / BM;
    Experts x;
    if constexpr (EXPERTS) {
        x = experts_from(a, 0, BM);
        m_tiles = tiles_of(x);
        for (int e0 = 64; e0 < a.experts; e0 += 64) m_tiles += tiles_of(experts_from(a, e0, BM));
        // offsets that fall name rows more than once: up to 2^27 tiles of rows, whose product with n_tiles passes 2^31
        m_tiles = min(m_tiles, a.most_down);
    }
    const int tiles = m_tiles * a.n_tiles, per = tiles / 8, rest = tiles % 8;
    const int xcd = blockIdx.x % 8, count = per + (xcd < rest ? 1 : 0);
    int local = blockIdx.x / 8;  // of the XCD's tiles
    if (local >= count) return;
    // A thread's pieces of a step: kA of a, then kB of b, kThreads / 8 rows apart.
    // Row r's piece p lies at place p ^ (r / 2 % 8): any 16 rows' pieces of one
    // column are then on different banks.
    // Rows' scales, four blocks of a row a lane: a row at a time they are a request
    // each, of 4 bytes as of 16.  The last four of a row may be some of those before.
    constexpr int kRuns = kScales / 64;  // waves that load them
    // the tile that is next: its place, and the choices that a thread's pieces of a and its scale are of
    int next_m0, next_n0, next_end = a.m, next_expert = 0, choices[EXPERTS ? kA + 1 : 1];
    const auto choose = [&]() {
        const int at = xcd * per + min(xcd, rest) + local;
        constexpr int kGroup = 4;
        const int grp = at / (kGroup * a.n_tiles), in = at - grp * kGroup * a.n_tiles, height = min(kGroup, m_tiles - grp * kGroup);
        const int mt = grp * kGroup + in % height;
        next_n0 = in / height * BN;
        next_m0 = mt * BM;
        if constexpr (EXPERTS) {
            const Rows r = rows_of(a, x, mt, BM);
            if (r.expert < 0) return false;
            next_expert = r.expert, next_m0 = r.first, next_end = r.end;
            int t = tid;
            if constexpr (BN == 256) asm volatile("" : "+v"(t));
#pragma unroll
            for (int c = 0; c < kA; c++) choices[c] = choice_of(a, min(r.first + t / 8 + c * (kThreads / 8), r.end - 1));
            choices[kA] = choice_of(a, min(r.first + (wave % kRuns * 64 + t % 64) % BM, r.end - 1));
        }
        return true;
    };
    if (!choose()) return;
    const int wm = wave / WAVES_N * (16 * TJ), wn = wave % WAVES_N * (16 * TI);
    const int blocks = (a.k + BK - 1) / BK, steps = (blocks + WAVES_K - 1) / WAVES_K;
    const auto input = [&](int choice) -> unsigned {  // ~0: a row that is not there, for which the first is read
        const int at = row_of(a, choice);
        return at >= 0 && at < a.a_rows ? at : 0xffffffffu;
    };

    int m0, n0, end_m, expert;
    const int place = tid & 7, piece = place ^ (tid / 16 & 7);
    const uint8_t *pa, *pb;
    unsigned offset[kPieces];
    const int scale_row = wave % kRuns * 64 + lane;
    const float *sa;
    unsigned scale_at = 0;
    const bool scaler = part == 0 && wave < kRuns;
    const auto quad_from = [&](int q) { return max(min(4 * q, blocks - 4), 0); };
    // The weights' scales of 64 blocks, one a lane: a scalar load in every step would have each of its reads of LDS
    // wait for it, too.
    const float *sb;
    float sb_ahead = 0.0f;
    // how many steps and runs of four scales the tiles before took, and tiles there were, as far as it says which buffer is next
    int flip = 0, quads = 0, turn = 0;
    const auto start = [&]() {
        int tid = wave * 64 + lane;
        if constexpr (BN == 256) asm volatile("" : "+v"(tid));
        const int scale_row = wave % kRuns * 64 + tid % 64, place = tid & 7, piece = place ^ (tid / 16 & 7);
        m0 = next_m0, n0 = next_n0, end_m = next_end, expert = next_expert;
        pa = a.a, pb = a.b + expert * a.b_expert + n0 * a.b_stride, sa = a.a_scale;
        if constexpr (!EXPERTS) pa += m0 * a.a_stride;
#pragma unroll
        for (int c = 0; c < kPieces; c++) {
            const int r = tid / 8 + (c < kA ? c : c - kA) * (kThreads / 8);
            if (c >= kA) offset[c] = static_cast<unsigned>(min(r, a.n - 1 - n0)) * static_cast<unsigned>(a.b_stride) + piece * 16;
            else if (EXPERTS) offset[c] = (input(choices[EXPERTS ? c % kA : 0]) == 0xffffffffu ? 0 : input(choices[EXPERTS ? c % kA : 0])) * static_cast<unsigned>(a.a_stride) + piece * 16;
            else offset[c] = static_cast<unsigned>(min(r, a.m - 1 - m0)) * static_cast<unsigned>(a.a_stride) + piece * 16;
        }
        if constexpr (EXPERTS) {
            const unsigned row = input(choices[EXPERTS ? kA : 0]);
            scale_at = (row == 0xffffffffu ? 0 : row) * static_cast<unsigned>(a.sa_stride) * 4;
            if (scaler) row_there[turn][EXPERTS ? scale_row : 0] = row != 0xffffffffu;
        } else {
            sa += m0 * a.sa_stride;
            scale_at = static_cast<unsigned>(min(scale_row % BM, a.m - 1 - m0)) * static_cast<unsigned>(a.sa_stride) * 4;
        }
        sb = a.b_scale + expert * a.sb_expert + min(n0 + wn, a.n - 1) / 128 * a.sb_stride;
        if (blocks < 4 && scaler) {
            for (int t = 0; t < blocks; t++)
                row_scales[quads][scale_row][t] = *reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(sa + t) + scale_at);
        }
    };
    start();
    // DIRECT: a step's loads into its buffer
    const auto load = [&](int s) {
        const int t = s * WAVES_K + part;
        // the lanes' offsets are added by the loads: sums made ahead of the loop would take two registers each
        asm("" : "+v"(scale_at));
#pragma unroll
        for (int c = 0; c < kPieces; c++) asm("" : "+v"(offset[c]));
        if (t % 4 == 0 && blocks >= 4 && scaler) load_lds16(sa + quad_from(t / 4), scale_at, lds_address(&row_scales[(t / 4 + quads) & 1][wave * 64]));
        const uint8_t *fa = pa + t * BK, *fb = pb + t * BK;
        uint8_t *to = lds + ((s + flip) & 1) * kBuffer + part * kPart + wave * 1024;
        if (t * BK + BK <= a.k) {
#pragma unroll
            for (int c = 0; c < kPieces; c++) load_lds16(c < kA ? fa : fb, offset[c], lds_address(to) + c * (kThreads * 16));
        } else if (t < blocks) {
            // the last block of a row, not whole: zeros past its end (the row's first bytes are loaded there)
            const int past = t * BK + piece * 16 >= a.k ? t * BK + piece * 16 : 0;
            intx4 last[kPieces];
#pragma unroll
            for (int c = 0; c < kPieces; c++) last[c] = load16((c < kA ? fa : fb) + offset[c], -past);
#pragma unroll
            for (int c = 0; c < kPieces; c++) *reinterpret_cast<intx4 *>(to + lane * 16 + c * (kThreads * 16)) = past ? intx4{0, 0, 0, 0} : last[c];
        }
    };
    // otherwise: into registers, and from there into LDS
    intx4 staged[kPieces];
    floatx4 quad;
    const auto fetch = [&](int s) {
        const int t = s * WAVES_K + part;
#pragma unroll
        for (int c = 0; c < kPieces; c++) asm("" : "+v"(offset[c]));
        if (t % 4 == 0 && t < blocks && blocks >= 4 && scaler)
            __builtin_memcpy(&quad, reinterpret_cast<const uint8_t *>(sa + quad_from(t / 4)) + scale_at, 16);
        const uint8_t *fa = pa + t * BK, *fb = pb + t * BK;
        if (t * BK + BK <= a.k) {
#pragma unroll
            for (int c = 0; c < kPieces; c++) __builtin_memcpy(&staged[c], (c < kA ? fa : fb) + offset[c], 16);
        } else if (t < blocks) {
            // what passes the row's end is its last 16 bytes, cleared where another piece has them
            const int back = max(t * BK + piece * 16 + 16 - a.k, 0);
            const intx4 keep = behind(back);
#pragma unroll
            for (int c = 0; c < kPieces; c++) staged[c] = load16((c < kA ? fa : fb) + offset[c], -static_cast<int64_t>(back)) & keep;
        }
    };
    const auto store = [&](int s) {
        const int t = s * WAVES_K + part;
        uint8_t *to = lds + (s & 1) * kBuffer + part * kPart + tid * 16;
#pragma unroll
        for (int c = 0; c < kPieces; c++) *reinterpret_cast<intx4 *>(to + c * (kThreads * 16)) = staged[c];
        // over those that were last read four blocks ago
        if (t % 4 == 0 && t < blocks && blocks >= 4 && scaler) *reinterpret_cast<floatx4 *>(row_scales[t / 4 & 1][scale_row]) = quad;
    };
    floatx4 acc[TI][TJ];
    const int at0 = col * BK + (g ^ (col / 2)) * 16, at1 = col * BK + ((4 + g) ^ (col / 2)) * 16;
    const auto read = [&](const uint8_t *rows, Operand<kWide> &x) {
        x.set(*reinterpret_cast<const intx4 *>(rows + at0), *reinterpret_cast<const intx4 *>(rows + at1));
    };
    // a wave whose rows or channels are all past the end leaves the matrix cores to the others
    bool active;
    const auto step = [&](int s) {
        const int t = s * WAVES_K + part;
        const uint8_t *now = lds + ((s + flip) & 1) * kBuffer + part * kPart;
        if (t % 64 < WAVES_K) {
            sb_ahead = sb[min(t / 64 * 64 + lane, blocks - 1)];
            asm volatile("" : "+v"(sb_ahead));  // waited for here, not in every step
        }
        const float sb_now = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sb_ahead), t % 64));
        if (active && (WAVES_K == 1 || t < blocks)) {
            Operand<kWide> fa[TJ], fb[2];
            float scale[TJ];
            read(now + (BM + wn) * BK, fb[0]);
#pragma unroll
            for (int j = 0; j < TJ; j++) read(now + (wm + 16 * j) * BK, fa[j]);
#pragma unroll
            for (int j = 0; j < TJ; j++) scale[j] = row_scales[(t / 4 + quads) & 1][wm + 16 * j + col][t - quad_from(t / 4)];
            if constexpr (!kWide) __builtin_amdgcn_sched_barrier(0);
            // a product, and the sums of the one two before it, which has ended
            floatx4 sum[3];
            const auto add = [&](int p) {
#pragma unroll
                for (int e = 0; e < 4; e++) acc[p / TJ][p % TJ][e] = __builtin_fmaf(scale[p % TJ], sum[p % 3][e], acc[p / TJ][p % TJ][e]);
            };
#pragma unroll
            for (int i = 0; i < TI; i++) {
#pragma unroll
                for (int j = 0; j < TJ; j++) {
                    const int p = i * TJ + j;
                    sum[p % 3] = product(fb[i & 1], fa[j]);
                    if constexpr (!kWide) __builtin_amdgcn_sched_barrier(0);
                    if (j == 0 && i + 1 < TI) read(now + (BM + wn + 16 * (i + 1)) * BK, fb[(i + 1) & 1]);
                    if (p < TJ) scale[j] *= sb_now;
                    if (p > 1) add(p - 2);
                    if constexpr (!kWide) __builtin_amdgcn_sched_barrier(0);
                }
            }
            add(TI * TJ - 2);
            add(TI * TJ - 1);
        }
    };
    if constexpr (DIRECT) {
        if (steps > 0) load(0);
    }
    while (true) {
        bool more = false;
        if constexpr (kGoOn) {
            local += kCus / 8;
            more = local < count && choose();
        }
        active = m0 + wm < end_m && n0 + wn < a.n;
#pragma unroll
        for (int i = 0; i < TI; i++)
#pragma unroll
            for (int j = 0; j < TJ; j++) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (DIRECT) {
            for (int s = 0; s < steps; s++) {
                // the barrier also ends the reads of the step before, whose buffer is loaded next
                wait_all();
                if (s + 1 < steps) load(s + 1);
                step(s);
            }
        } else if (steps > 0) {
            fetch(0);
            store(0);
            if (steps > 1) fetch(1);
            for (int s = 0; s < steps; s++) {
                __syncthreads();
                if (s + 1 < steps) store(s + 1);
                if (s + 2 < steps) fetch(s + 2);
                step(s);
            }
        }
        __syncthreads();
        if constexpr (WAVES_K > 1) {
            // the groups' sums, joined in their order
            floatx4 *sums = reinterpret_cast<floatx4 *>(lds);
            static_assert((WAVES_K - 1) * BM * BN * 4 <= 2 * kBuffer, "LDS holds the groups' sums");
            if (part > 0) {
#pragma unroll
                for (int i = 0; i < TI; i++)
#pragma unroll
                    for (int j = 0; j < TJ; j++) sums[((part - 1) * TI * TJ + i * TJ + j) * kThreads + tid] = acc[i][j];
            }
            __syncthreads();
            if (part > 0) return;
#pragma unroll
            for (int i = 0; i < TI; i++)
#pragma unroll
                for (int j = 0; j < TJ; j++)
#pragma unroll
                    for (int w = 1; w < WAVES_K; w++) acc[i][j] += sums[((w - 1) * TI * TJ + i * TJ + j) * kThreads + tid];
            // this group's waves write over others' sums
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }

        // This tile's place, and the buffer that its sums may take
        const int n = n0 + wn, m = m0 + wm, left = a.n - n, rows = end_m - m, was = turn;
        const float *bias_from = a.bias + static_cast<int64_t>(expert) * a.n;
        uint8_t *room = lds;
        if constexpr (kGoOn) {
            room += (steps - 1 + flip & 1) * kBuffer;
            if (more) {
                flip = (flip + steps) & 1, quads = (quads + (steps - 1) / 4 + 1) & 1, turn ^= 1;
                start();
                load(0);
            }
        }

        // Places that are the same for every tile are taken anew: kept, they would take registers that the loop needs.
        int lane = threadIdx.x & 63;
        if constexpr (BN == 256) asm volatile("" : "+v"(lane));
        const int col = lane & 15, g = lane >> 4;

        // Through this wave's own part of LDS (every wave is past its last read of the
        // buffers), so that a row's channels leave as 16-byte pieces one after the other.
        // A row's piece p lies at place p ^ (row / rows of 256 bytes): the accumulators'
        // 8-byte writes and the rows' reads are then on different banks.  Sixteen rows at
        // a time, each asked whether it is inside, this took a tile of 256 x 256 8 us.
        constexpr int kHalves = kGoOn ? 2 : 1, kRoom = kGoOn ? kBuffer : 2 * kBuffer, kHigh = 16 * TJ / kHalves;  // rows at a time
        constexpr int kPiece = 16 / static_cast<int>(sizeof(T)), kLanes = 16 * TI / kPiece;  // elements of a piece, pieces of a row
        constexpr int kRows = 64 / kLanes, kReads = kHigh / kRows, kPitch = kLanes * 16;
        static_assert(kHigh * kPitch <= kRoom / kWaves && TJ % kHalves == 0, "a wave's part of LDS holds its tile");
        uint8_t *mine = room + wave * (kRoom / kWaves);
        const auto spot = [&](int row, int p) { return mine + row * kPitch + ((p ^ (row / (16 / kLanes > 0 ? 16 / kLanes : 1))) & (kLanes - 1)) * 16; };
        if constexpr (EXPERTS) {
#pragma unroll
            for (int j = 0; j < TJ; j++)
                if (!row_there[was][wm + 16 * j + col]) {
#pragma unroll
                    for (int i = 0; i < TI; i++) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                }
        }
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < TI; i++) {
                floatx4 bias;
#pragma unroll
                for (int e = 0; e < 4; e++) bias[e] = bias_from[min(n + 16 * i + 4 * g + e, a.n - 1)];
#pragma unroll
                for (int j = 0; j < TJ; j++) acc[i][j] += bias;
            }
        }
        const int c = lane % kLanes * kPiece, r0 = lane / kLanes;
        const auto piece_of = [&](int r) { return *reinterpret_cast<const Vec<T, kPiece> *>(spot(r + r0, lane % kLanes)); };
#pragma unroll
        for (int h = 0; h < kHalves; h++) {
#pragma unroll
            for (int j = h * TJ / kHalves; j < (h + 1) * TJ / kHalves; j++) {
#pragma unroll
                for (int i = 0; i < TI; i++) {
                    const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                    const int at = 16 * i + 4 * g;
                    put_floats<4>(reinterpret_cast<T *>(spot(16 * j - h * kHigh + col, at / kPiece)) + at % kPiece, v);
                }
            }
            wait_lds();
            T *out = static_cast<T *>(a.out) + (m + h * kHigh + r0) * a.out_stride + n + c;
            if (rows >= (h + 1) * kHigh && left >= 16 * TI) {
                constexpr int kAhead = kReads < 8 ? kReads : 8;
#pragma unroll
                for (int q = 0; q < kReads; q += kAhead) {
                    Vec<T, kPiece> v[kAhead];
#pragma unroll
                    for (int u = 0; u < kAhead; u++) v[u] = piece_of((q + u) * kRows);
#pragma unroll
                    for (int u = 0; u < kAhead; u++) __builtin_memcpy(out + static_cast<int64_t>((q + u) * kRows) * a.out_stride, v[u].v, 16);
                }
            } else {
                const int high = min(rows - h * kHigh, kHigh);
#pragma unroll 1
                for (int r = 0; r < high; r += kRows) {
                    const Vec<T, kPiece> v = piece_of(r);
                    if (r + r0 >= high) continue;
                    T *y = out + static_cast<int64_t>(r) * a.out_stride;
                    if (c + kPiece <= left) {
                        __builtin_memcpy(y, v.v, 16);
                    } else {
#pragma unroll
                        for (int e = 0; e < kPiece; e++)
                            if (c + e < left) y[e] = v.v[e];
                    }
                }
            }
            wait_lds();
        }
        if (!more) return;
    }
}

int check(const Spkv2MatmulF8 *g, bool experts, bool pointers) {
    if (!g) return bad("matmul_f8: no arguments");
    if (!is_dtype(g->dtype)) return bad("matmul_f8: unknown dtype");
    if (g->m < 0 || g->n < 0 || g->k < 0) return bad("matmul_f8: negative size");
    if (g->m == 0 || g->n == 0) return 0;
    if (pointers && (!g->out || (g->k && (!g->a || !g->b || !g->a_scale || !g->b_scale)))) return bad("matmul_f8: a NULL pointer");
    const int64_t blocks = (g->k + 127) / 128;
    if ((g->m > 1 && g->out_stride < g->n) || (!experts && g->m > 1 && (g->a_stride < g->k || g->a_scale_stride < blocks)) ||
        (g->n > 1 && g->b_stride < g->k) || (g->n > 128 && g->b_scale_stride < blocks))
        return bad("matmul_f8: a stride is below its row's length");
    if (g->k > (1 << 24)) return unsupported("matmul_f8: k above 2^24");
    if (g->m > (1 << 20) || g->n > (1 << 26)) return unsupported("matmul_f8: m above 2^20 or n above 2^26");
    return 0;
}

int check(const Spkv2MatmulF8Experts *g, bool pointers) {
    if (!g) return bad("matmul_f8_experts: no arguments");
    if (int rc = check(&g->product, true, pointers)) return rc;
    if (g->experts < 1 || g->per_token < 1 || g->a_rows < 0) return bad("matmul_f8_experts: a size is below 1");
    if (g->experts > 4096) return unsupported("matmul_f8_experts: more than 4096 experts");
    if (pointers && !g->offsets) return bad("matmul_f8_experts: offsets is NULL");
    const Spkv2MatmulF8 &p = g->product;
    if (p.m && p.n && p.k && g->a_rows < 1) return bad("matmul_f8_experts: a has no rows");
    const int64_t blocks = (p.k + 127) / 128;
    if (g->a_rows > 1 && (p.a_stride < p.k || p.a_scale_stride < blocks)) return bad("matmul_f8_experts: a stride is below its row's length");
    if (g->experts > 1 && p.n && p.k && (g->b_expert_stride < (p.n - 1) * p.b_stride + p.k || g->b_scale_expert_stride < (p.n - 1) / 128 * p.b_scale_stride + blocks))
        return bad("matmul_f8_experts: experts' weights overlap");
    return 0;
}

MatmulArgs arguments(const Spkv2MatmulF8 &g) {
    MatmulArgs a{g.a, g.b, g.a_scale, g.b_scale, g.bias, g.out, g.a_stride, g.b_stride, g.out_stride, g.a_scale_stride, g.b_scale_stride,
                 static_cast<int>(g.m), static_cast<int>(g.n), static_cast<int>(g.k), 0, nullptr, nullptr, g.m, 0, 0, 1, 0, 0, 0};
    if (g.m == 1) a.a_stride = 0, a.sa_stride = 0, a.out_stride = 0;
    if (g.n == 1) a.b_stride = 0;
    if (g.n <= 128) a.sb_stride = 0;
    return a;
}

// A kernel's time: a launch's, then steps by every workgroup, of a block of k for
// each of its groups of waves, which take `step` each where a CU's workgroups do
// not fill it, or `work` for each of the CU's workgroups where they do, and the
// workgroup's sums.  Fitted, in us, to 5450 products of log-uniform sizes (m 1 ..
// 8192, n and k 64 .. 16384, up to 2^37 multiplications; half of them by expert):
// the kernel of the least time by these is 1.5% slower than the fastest of them in
// the mean, 25% in one of a hundred.  Tiles of 128 x 256 are the fastest where they
// fill the CUs once and larger ones half of them (2048 x 4096 x 4096 55 -> 41 us).
struct Cost {
    float launch, step, work, sums;
};
struct Form {
    int tokens, channels, groups;  // of a workgroup; groups of waves that deal k out
    bool tiles;
    Cost cost[4];  // 16-bit outputs with rows of whole runs of 16 bytes, and others; fp32 outputs likewise
};
constexpr Form kForms[] = {
    {16, 16, 8, false, {{1.52f, 0.006f, 0.686f, 1.191f}, {1.54f, 0.878f, 0.906f, 1.109f}, {1.50f, 0.446f, 0.751f, 1.241f}, {1.69f, 0.337f, 0.989f, 1.009f}}},
    {16, 32, 8, false, {{1.81f, 1.006f, 1.034f, 0.785f}, {1.89f, 1.298f, 1.340f, 0.630f}, {1.82f, 0.095f, 1.136f, 0.762f}, {2.04f, 1.059f, 1.445f, 0.500f}}},
    {16, 64, 8, false, {{1.71f, 0.106f, 1.567f, 0.733f}, {1.78f, 2.246f, 2.251f, 0.262f}, {1.74f, 0.118f, 1.719f, 0.691f}, {2.01f, 2.253f, 2.328f, 0.183f}}},
    {32, 64, 8, false, {{0.77f, 1.323f, 1.892f, 1.891f}, {0.85f, 0.993f, 2.681f, 1.388f}, {0.93f, 2.156f, 2.164f, 1.689f}, {1.18f, 2.480f, 2.851f, 1.187f}}},
    {64, 64, 1, true, {{3.08f, 0.378f, 0.267f, 0.705f}, {2.77f, 0.809f, 0.443f, 0.731f}, {3.16f, 0.503f, 0.325f, 0.857f}, {2.93f, 0.939f, 0.510f, 0.865f}}},
    {64, 64, 2, true, {{2.61f, 0.534f, 0.527f, 1.348f}, {2.19f, 1.187f, 0.885f, 1.271f}, {2.57f, 0.729f, 0.635f, 1.557f}, {2.45f, 1.351f, 1.033f, 1.308f}}},
    {64, 64, 4, true, {{0.66f, 0.645f, 0.976f, 3.734f}, {0.69f, 0.900f, 1.959f, 2.926f}, {0.85f, 0.401f, 1.305f, 3.733f}, {0.97f, 1.046f, 2.220f, 2.994f}}},
    {32, 128, 1, true, {{3.04f, 0.408f, 0.335f, 0.791f}, {2.67f, 0.929f, 0.556f, 0.804f}, {2.91f, 0.537f, 0.374f, 1.062f}, {2.66f, 1.063f, 0.626f, 0.978f}}},
    {128, 128, 1, true, {{2.66f, 0.668f, 0.570f, 2.334f}, {1.94f, 1.439f, 0.992f, 2.511f}, {2.99f, 1.079f, 0.880f, 2.717f}, {2.39f, 2.080f, 1.425f, 2.711f}}},
    {128, 256, 1, true, {{0.00f, 0.100f, 0.887f, 5.073f}, {0.00f, 0.100f, 1.655f, 4.976f}, {}, {}}},
    {256, 256, 1, true, {{0.00f, 0.100f, 1.118f, 7.074f}, {0.00f, 1.863f, 2.145f, 6.893f}, {}, {}}},
};
constexpr int kFormCount = sizeof(kForms) / sizeof(kForms[0]);

// Workgroups along the rows.  By expert: at most, for the launch; about, for the time.
int64_t most_down(const MatmulArgs &a, bool experts, int height) {
    return experts ? a.m / height + std::min(a.experts, a.m) : (static_cast<int64_t>(a.m) + height - 1) / height;
}
double about_down(const MatmulArgs &a, bool experts, int height) {
    if (!experts) return static_cast<double>(most_down(a, false, height));
    // experts that rows chosen at random leave without one, and half a workgroup's rows missing of each other's last
    const double used = a.experts * (1.0 - pow(1.0 - 1.0 / a.experts, a.m)), each = a.m / used;
    return ceil(each < 0.5 * height ? used : used * (each / height + 0.5));
}

// whether rows are whole runs of 16 bytes at such addresses, as loads into LDS take them
bool whole(const MatmulArgs &a) {
    return a.k % 16 == 0 && aligned(a.a, 16) && aligned(a.b, 16) && a.a_stride % 16 == 0 && a.b_stride % 16 == 0 && a.b_expert % 16 == 0;
}

// the kernel of a call that check() took, as an index of kForms; -1: none
int form(const MatmulArgs &a, bool experts, int dtype) {
    const int kind = (dtype == SPKV2_DTYPE_FP32 ? 2 : 0) + (whole(a) ? 0 : 1);
    // tiles hold offsets of a workgroup's rows (by expert, of all rows of a) in 32 bits
    const int64_t held = experts ? a.a_rows : std::min(a.m, 256);
    const bool near = held * a.a_stride < (int64_t(1) << 31) && held * a.sa_stride < (int64_t(1) << 29) && 256 * a.b_stride < (int64_t(1) << 31);
    const int blocks = (a.k + 127) / 128;
    int best = -1;
    double least = 0.0;
    for (int i = 0; i < kFormCount; i++) {
        const Form &f = kForms[i];
        const int64_t across = (static_cast<int64_t>(a.n) + f.channels - 1) / f.channels, down = most_down(a, experts, f.tokens);
        // a launch has fewer than 2^32 threads along an axis, and as many workgroups along the second as 16 bits hold
        if (f.tiles ? !near || a.k < 16 || down * across >= 1 << 22 : down > 65535) continue;
        // outputs of 32 bits do not fit their LDS, nor two registers' operands beside sums of 256 x 256
        if (f.channels == 256 && dtype == SPKV2_DTYPE_FP32) continue;
        const Cost &c = f.cost[kind];
        const double steps = (blocks + f.groups - 1) / f.groups, each = ceil(about_down(a, experts, f.tokens) * across / 256.0);
        const double time = c.launch + steps * std::max(static_cast<double>(c.step), each * c.work) + each * c.sums;
        if (best < 0 || time < least) least = time, best = i;
    }
    return best;
}

template <bool EXPERTS>
int run(const char *what, int dtype, MatmulArgs a, void *stream) {
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int i = form(a, EXPERTS, dtype);
        if (i < 0) return unsupported("matmul_f8: too many rows or channels for one launch");
        const Form &f = kForms[i];
        const unsigned across = static_cast<unsigned>((static_cast<int64_t>(a.n) + f.channels - 1) / f.channels);
        const unsigned down = static_cast<unsigned>(most_down(a, EXPERTS, f.tokens));
        a.n_tiles = static_cast<int>(across);
        a.most_down = static_cast<int>(down);
        auto rows = [&](auto kernel) { return launch(what, kernel, dim3(across, down), dim3(64 * 8), stream, a); };
        auto tiles = [&](auto direct, auto staged, int waves) {
            const unsigned all = across * down;
            return launch(what, whole(a) ? direct : staged, dim3(goes_on(whole(a), f.channels) ? std::min<unsigned>(all, kCus) : all), dim3(64 * waves), stream, a);
        };
        switch (i) {
            case 0: return rows(matmul_rows<T, EXPERTS, 1, 1>);
            case 1: return rows(matmul_rows<T, EXPERTS, 1, 2>);
            case 2: return rows(matmul_rows<T, EXPERTS, 1, 4>);
            case 3: return rows(matmul_rows<T, EXPERTS, 2, 4>);
            case 4: return tiles(matmul_tiles<T, EXPERTS, true, 2, 2, 1, 2, 2>, matmul_tiles<T, EXPERTS, false, 2, 2, 1, 2, 2>, 4);
            case 5: return tiles(matmul_tiles<T, EXPERTS, true, 2, 2, 2, 2, 2>, matmul_tiles<T, EXPERTS, false, 2, 2, 2, 2, 2>, 8);
            case 6: return tiles(matmul_tiles<T, EXPERTS, true, 2, 2, 4, 2, 2>, matmul_tiles<T, EXPERTS, false, 2, 2, 4, 2, 2>, 16);
            case 7: return tiles(matmul_tiles<T, EXPERTS, true, 1, 4, 1, 2, 2>, matmul_tiles<T, EXPERTS, false, 1, 4, 1, 2, 2>, 4);
            case 8: return tiles(matmul_tiles<T, EXPERTS, true, 2, 2, 1, 4, 4>, matmul_tiles<T, EXPERTS, false, 2, 2, 1, 4, 4>, 4);
            default:
                if constexpr (sizeof(T) == 4) return -1;
                else if (i == 9) return tiles(matmul_tiles<T, EXPERTS, true, 2, 4, 1, 4, 4>, matmul_tiles<T, EXPERTS, false, 2, 4, 1, 4, 4>, 8);
                else return tiles(matmul_tiles<T, EXPERTS, true, 4, 2, 1, 4, 8>, matmul_tiles<T, EXPERTS, false, 4, 2, 1, 4, 8>, 8);
        }
    });
}

int name(const MatmulArgs &a, bool experts, int dtype, char *buf, size_t size) {
    buf[0] = 0;
    if (a.m == 0 || a.n == 0) return 0;
    const int i = form(a, experts, dtype);
    if (i < 0) return unsupported("matmul_f8: too many rows or channels for one launch");
    const Form &f = kForms[i];
    if (f.tiles) snprintf(buf, size, "matmul_tiles<%dx%d,groups=%d,%s>", f.tokens, f.channels, f.groups, whole(a) ? "direct" : "staged");
    else snprintf(buf, size, "matmul_rows<%dx%d>", f.tokens, f.channels);
    return 0;
}

MatmulArgs arguments(const Spkv2MatmulF8Experts &g) {
    MatmulArgs a = arguments(g.product);
    a.offsets = g.offsets;
    a.order = g.order;
    a.a_rows = g.a_rows;
    a.b_expert = g.experts > 1 ? g.b_expert_stride : 0;
    a.sb_expert = g.experts > 1 ? g.b_scale_expert_stride : 0;
    a.experts = g.experts;
    div_magic(static_cast<unsigned>(g.per_token), &a.token_mul, &a.token_shift);
    a.a_stride = g.product.a_stride, a.sa_stride = g.product.a_scale_stride;
    if (g.a_rows == 1) a.a_stride = 0, a.sa_stride = 0;
    return a;
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_matmul_f8(const Spkv2MatmulF8 *g, void *stream) {
    return entry([&]() -> int {
        if (int rc = check(g, false, true)) return rc;
        if (g->m == 0 || g->n == 0) return 0;
        return run<false>("matmul_f8", g->dtype, arguments(*g), stream);
    });
}

extern "C" int spkv2_mi355x_matmul_f8_experts(const Spkv2MatmulF8Experts *g, void *stream) {
    return entry([&]() -> int {
        if (int rc = check(g, true)) return rc;
        if (g->product.m == 0 || g->product.n == 0) return 0;
        return run<true>("matmul_f8_experts", g->product.dtype, arguments(*g), stream);
    });
}

extern "C" int spkv2_mi355x_matmul_f8_kernel_name(const Spkv2MatmulF8 *g, char *buf, size_t buf_size) {
    return entry([&]() -> int {
        if (!buf || !buf_size) return bad("matmul_f8: nowhere to put the name");
        if (int rc = check(g, false, false)) return rc;
        return name(arguments(*g), false, g->dtype, buf, buf_size);
    });
}

extern "C" int spkv2_mi355x_matmul_f8_experts_kernel_name(const Spkv2MatmulF8Experts *g, char *buf, size_t buf_size) {
    return entry([&]() -> int {
        if (!buf || !buf_size) return bad("matmul_f8_experts: nowhere to put the name");
        if (int rc = check(g, false)) return rc;
        return name(arguments(*g), true, g->product.dtype, buf, buf_size);
    });
}
