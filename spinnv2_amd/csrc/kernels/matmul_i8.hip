// Product of int8 rows and int8 weights with a scale for each token and each
// output channel:
//
//   out[m, n] = sa[m] sb[n] sum_k a[m, k] b[n, k] + bias[n]
//
// int32 sums on the int8 matrix cores, exact whatever their order, scaled in
// fp32 and rounded once.  So every kernel here gives the same bits, and which
// one runs is a question of time alone.  Up to k = 2^17 the sums lie between
// -127 128 2^17 > -2^31 and 128 128 2^17 = 2^31: that one, of 2^17 products of
// -128, comes out as -2^31, which no other sum does.
//
// matmul_tiles serves many tokens: bound by the matrix cores, which work in 64%
// of the busy cycles (8192^3 in 474 to 487 us on three chips, 2.3 POP/s).  matmul_rows serves few:
// bound by the weights' bytes (1 x 16384 x 4096 in 13.4 us, 5.0 TB/s) or, where
// they are few, by its launch (64 x 1000 x 2048 in 3.8 us).
#include <cstdio>

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
    int m_tiles, n_tiles;
};

// 16 bytes at p, of which `left` are inside the row: zeros past them
__device__ __forceinline__ intx4 part16(const int8_t *p, int left) {
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

// 16 bytes at p + at, which all lie inside
__device__ __forceinline__ intx4 load16(const int8_t *p, unsigned at) {
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

__device__ __forceinline__ float scaled(int sum, float sa, float sb, float bias) {
    return __builtin_fmaf(static_cast<float>(sum) * sa, sb, bias);
}

// A sum of 2^31 that came out as -2^31, as the int32 that fp32 rounds to it.
// Only k = 2^17 has one: asked of every sum it costs 4 us of 8192 x 8192 x 2048.
__device__ __forceinline__ int unwrapped(int sum) { return sum == INT32_MIN ? INT32_MAX : sum; }
constexpr int kMostTerms = 1 << 17;

// LDS of one wave alone: its writes are done before its reads, and the other way round
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// N floats at p, of which `left` are there: zeros past them
template <int N>
__device__ __forceinline__ void some(const float *p, int left, float (&f)[N]) {
    if (left >= N) {
        __builtin_memcpy(f, p, sizeof(f));
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = e < left ? p[e] : 0.0f;
    }
}

// The order of a phase: its READS of LDS among the first half of its PRODUCTS,
// so that they have arrived when the next phase begins, the WRITES to LDS and
// the LOADS among the second.
template <int READS, int PRODUCTS, int WRITES, int LOADS>
__device__ __forceinline__ void interleave() {
    if constexpr (PRODUCTS >= 4) {
        constexpr int kHalf = PRODUCTS / 2;
#pragma unroll
        for (int i = 0; i < kHalf; i++) {
            __builtin_amdgcn_sched_group_barrier(0x100, (READS + kHalf - 1) / kHalf, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < kHalf; i++) {
            if constexpr (WRITES > 0) __builtin_amdgcn_sched_group_barrier(0x200, (WRITES + kHalf - 1) / kHalf, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if constexpr (LOADS > 0) __builtin_amdgcn_sched_group_barrier(0x020, (LOADS + kHalf - 1) / kHalf, 0);
        }
    }
}

// 64 B tokens x 64 B channels a workgroup of four waves (2 x 2), each B x B
// tiles of 32 x 32; 128 bytes of k a step, in two buffers of LDS.
//
// The widest tile takes a CU: its sums are 256 registers of each lane, and each
// of its four waves reads 512 bytes of LDS a product of 32 cycles, together 64
// bytes a cycle, half of what LDS gives (96 with 128 x 64 a wave).  A step's
// pieces wait in registers from one step to the next, so that memory has a
// step's time to answer, and each piece is written to LDS and loaded anew among
// the products, a few at a time: all at once, the four waves' loads stand in
// line while no product runs (8192^3 495 against 465 us).  The next phase's
// operands are read a phase ahead, across the step's one barrier too.
template <typename T, int B>
__global__ void __launch_bounds__(256, B >= 4 ? 1 : 2) matmul_tiles(MatmulArgs a) {
    constexpr int TM = B, TN = B;
    constexpr int BM = 64 * TM, BN = 64 * TN, BK = 128;
    constexpr int kA = BM / 32, kB = BN / 32;  // 16-byte pieces a thread
    constexpr int kBuffer = (BM + BN) * BK;
    __shared__ __align__(16) int8_t lds[2 * kBuffer];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the eight XCDs in turn; each XCD takes a run of tiles,
    // four tiles of tokens by the channels one after the other, whose operands
    // its L2 then holds for several of them.
    int mt, nt;
    {
        const int tiles = a.m_tiles * a.n_tiles, per = tiles / 8, rest = tiles % 8;
        const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
        const int at = xcd * per + min(xcd, rest) + local;
        constexpr int kGroup = 4;
        const int g = at / (kGroup * a.n_tiles), in = at - g * kGroup * a.n_tiles, height = min(kGroup, a.m_tiles - g * kGroup);
        mt = g * kGroup + in % height;
        nt = in / height;
    }
    const int m0 = mt * BM, n0 = nt * BN;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    const int steps = (a.k + BK - 1) / BK;

    intx16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0;

    // a thread's pieces of a step: kA of a, then kB of b, 32 rows apart
    constexpr int kPieces = kA + kB;
    const int chunk = tid & 7;
    unsigned offset[kPieces];
#pragma unroll
    for (int c = 0; c < kPieces; c++)
        offset[c] = c < kA ? static_cast<unsigned>(min(tid / 8 + 32 * c, a.m - 1 - m0)) * static_cast<unsigned>(a.a_stride) + chunk * 16
                           : static_cast<unsigned>(min(tid / 8 + 32 * (c - kA), a.n - 1 - n0)) * static_cast<unsigned>(a.b_stride) + chunk * 16;
    const int8_t *pa = a.a + m0 * a.a_stride, *pb = a.b + n0 * a.b_stride;
    intx4 staged[kPieces];
    auto fetch = [&](int s, int from, int to) {
#pragma unroll
        for (int c = from; c < to; c++) staged[c] = load16((c < kA ? pa : pb) + s * BK, offset[c]);
    };
    // in the order of the pieces, which the loop waits for one by one
    auto fetch_all = [&](int s) {
#pragma unroll
        for (int c = 0; c < kPieces; c++) {
            fetch(s, c, c + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The last step's pieces that pass the row's end are its last 16 bytes,
    // of which a's are cleared where an earlier piece has them.
    auto fetch_last = [&]() {
        const int k = (steps - 1) * BK + chunk * 16, over = max(0, k + 16 - a.k);  // bytes
        const intx4 keep = behind(over);
#pragma unroll
        for (int c = 0; c < kPieces; c++) {
            staged[c] = load16((c < kA ? pa : pb) + (steps - 1) * BK - over, offset[c]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < kA; c++) staged[c] &= keep;
    };
    // Row r's piece p lies at place p ^ (r / 2 % 8): any 16 rows' pieces of one
    // column are then on different banks.
    const int put_at = (tid / 8) * BK + ((chunk ^ (tid / 16 & 7)) * 16);
    auto store = [&](int8_t *buf, int from, int to) {
#pragma unroll
        for (int c = from; c < to; c++) *reinterpret_cast<intx4 *>(buf + put_at + c * 32 * BK) = staged[c];
    };
    const int row_a = (wm + lane % 32) * BK, row_b = BM * BK + (wn + lane % 32) * BK;
    int swizzle[4];
#pragma unroll
    for (int kk = 0; kk < 4; kk++) swizzle[kk] = ((2 * kk + lane / 32) ^ (lane / 2 & 7)) * 16;
    intx4 fa[2][TM], fb[2][TN];
    auto read = [&](const int8_t *buf, int kk, int to) {
#pragma unroll
        for (int j = 0; j < TM; j++) fa[to][j] = *reinterpret_cast<const intx4 *>(buf + row_a + j * 32 * BK + swizzle[kk]);
#pragma unroll
        for (int i = 0; i < TN; i++) fb[to][i] = *reinterpret_cast<const intx4 *>(buf + row_b + i * 32 * BK + swizzle[kk]);
    };
    auto multiply = [&](int from) {
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[from][i], fa[from][j], acc[i][j], 0, 0, 0);
    };
    if (steps > 0) {
        if (steps > 1) fetch_all(0);
        else fetch_last();
        store(lds, 0, kPieces);
        if (steps > 2) fetch_all(1);
        else if (steps == 2) fetch_last();
        __syncthreads();
        read(lds, 0, 0);
    }
    int s = 0;
    constexpr int kReads = TM + TN, kProducts = TM * TN, kThird = (kPieces + 2) / 3, kQuarter = kPieces / 4;
    for (; s + 3 < steps; s++) {
        int8_t *now = lds + (s & 1) * kBuffer, *then = lds + (~s & 1) * kBuffer;
        read(now, 1, 1);
        store(then, 0, kThird);
        fetch(s + 2, 0, kQuarter);
        multiply(0);
        interleave<kReads, kProducts, kThird, kQuarter>();
        read(now, 2, 0);
        store(then, kThird, 2 * kThird);
        fetch(s + 2, kQuarter, 2 * kQuarter);
        multiply(1);
        interleave<kReads, kProducts, kThird, kQuarter>();
        read(now, 3, 1);
        store(then, 2 * kThird, kPieces);
        fetch(s + 2, 2 * kQuarter, 3 * kQuarter);
        multiply(0);
        interleave<kReads, kProducts, kPieces - 2 * kThird, kQuarter>();
        __syncthreads();
        read(then, 0, 0);
        fetch(s + 2, 3 * kQuarter, kPieces);
        multiply(1);
        interleave<kReads, kProducts, 0, kQuarter>();
    }
    for (; s < steps; s++) {
        int8_t *now = lds + (s & 1) * kBuffer, *then = lds + (~s & 1) * kBuffer;
        read(now, 1, 1);
        if (s + 1 < steps) store(then, 0, kPieces);
        multiply(0);
        read(now, 2, 0);
        if (s + 3 == steps) fetch_last();
        multiply(1);
        read(now, 3, 1);
        multiply(0);
        __syncthreads();
        if (s + 1 < steps) read(then, 0, 0);
        multiply(1);
    }

    if (a.k == kMostTerms) {
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[i][j][r] = unwrapped(acc[i][j][r]);
    }

    // Scaled and rounded, each 32 tokens go through this wave's own part of LDS
    // (every wave is past its last read of the buffers), so that a row's
    // channels leave as 16-byte pieces one after the other.
    constexpr int kCols = 32 * TN, kPiece = 16 / static_cast<int>(sizeof(T)), kOutPitch = kCols * static_cast<int>(sizeof(T)) + 16;
    static_assert(32 * kOutPitch <= kBuffer / 2, "a wave's part of LDS holds 32 rows");
    T *mine = reinterpret_cast<T *>(lds + wave * (kBuffer / 2));
    float sb[TN][16], bias[TN][16];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int n = n0 + wn + i * 32 + 2 * r + 4 * (lane / 32);
            float f[4], c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            some(a.b_scale + n, a.n - n, f);
            if (a.bias) some(a.bias + n, a.n - n, c);
#pragma unroll
            for (int e = 0; e < 4; e++) sb[i][r + e] = f[e], bias[i][r + e] = c[e];
        }
    const int left = a.n - n0 - wn;
#pragma unroll
    for (int j = 0; j < TM; j++) {
        const int m = m0 + wm + j * 32;
        if (m >= a.m) break;
        const float sa = a.a_scale[min(m + lane % 32, a.m - 1)];
        T *row = mine + lane % 32 * (kOutPitch / static_cast<int>(sizeof(T))) + 4 * (lane / 32);
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = scaled(acc[i][j][r + e], sa, sb[i][r + e], bias[i][r + e]);
                put_floats<4>(row + i * 32 + 2 * r, v);
            }
        wait_lds();
        constexpr int kLanes = kCols / kPiece, kRows = 64 / kLanes;
        const int c = lane % kLanes * kPiece;
        T *out = static_cast<T *>(a.out) + (m + lane / kLanes) * a.out_stride + n0 + wn + c;
#pragma unroll
        for (int r = 0; r < 32; r += kRows) {
            const Vec<T, kPiece> v = *reinterpret_cast<const Vec<T, kPiece> *>(mine + (r + lane / kLanes) * (kOutPitch / static_cast<int>(sizeof(T))) + c);
            if (m + r + lane / kLanes < a.m) {
                if (c + kPiece <= left) {
                    __builtin_memcpy(out + r * a.out_stride, v.v, sizeof(v.v));
                } else {
#pragma unroll
                    for (int e = 0; e < kPiece; e++)
                        if (c + e < left) out[r * a.out_stride + e] = v.v[e];
                }
            }
        }
        wait_lds();
    }
}

// 16 TM tokens x 16 TN channels a workgroup, whose waves deal k out among
// them, 128 bytes at a time, and join their sums in LDS.  A wave loads eight
// rows' 128 bytes an instruction and turns them in LDS of its own into the
// matrix cores' order (16 rows' 16 bytes): loaded in that order, neighbouring
// lanes are different rows and each is a request of its own.
template <typename T, int TM, int TN, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) matmul_rows(MatmulArgs a) {
    constexpr int kPieces = 2 * (TM + TN);  // loads of eight rows a chunk: 2 TM of a, then 2 TN of b
    constexpr int kAhead = kPieces <= 4 ? 4 : kPieces <= 8 ? 2 : 1;  // chunks loaded together
    constexpr int kTurn = (kPieces > TM * TN ? kPieces : TM * TN) * 1024;
    __shared__ __align__(16) int8_t lds[WAVES * kTurn];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * TN, m0 = blockIdx.y * 16 * TM;
    const int chunks = (a.k + 127) / 128, per = (chunks + WAVES - 1) / WAVES;
    const int first = wave * per, end = min(first + per, chunks);
    const int8_t *p[kPieces];
#pragma unroll
    for (int c = 0; c < kPieces; c++)
        p[c] = c < 2 * TM ? a.a + min(m0 + 8 * c + lane / 8, a.m - 1) * a.a_stride : a.b + min(n0 + 8 * (c - 2 * TM) + lane / 8, a.n - 1) * a.b_stride;
    int8_t *turn = lds + wave * kTurn;
    const int put_at = lane / 8 * 128;
    intx4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = intx4{0, 0, 0, 0};
    struct Chunk {
        intx4 v[kPieces];
    };
    auto fetch = [&](Chunk &x, int s) {
        const int k = s * 128 + lane % 8 * 16;
        if (s * 128 + 128 <= a.k) {
#pragma unroll
            for (int c = 0; c < kPieces; c++) x.v[c] = load16(p[c], k);
        } else if (a.k >= 16) {
            // pieces past the row's end are its last 16 bytes, a's cleared
            // where another piece has them
            const int at = min(k, a.k - 16);
            const intx4 keep = behind(k - at);
#pragma unroll
            for (int c = 0; c < kPieces; c++) {
                x.v[c] = load16(p[c], at);
                if (c < 2 * TM) x.v[c] &= keep;
            }
        } else {
#pragma unroll
            for (int c = 0; c < kPieces; c++) x.v[c] = part16(p[c], lane % 8 == 0 ? a.k : 0);
        }
    };
    auto multiply = [&](const Chunk &x) {
        // row r's piece lies at place piece ^ (r / 2 % 8), as in matmul_tiles
#pragma unroll
        for (int c = 0; c < kPieces; c++)
            *reinterpret_cast<intx4 *>(turn + c * 1024 + put_at + ((lane % 8) ^ ((c * 4 + lane / 16) & 7)) * 16) = x.v[c];
        wait_lds();
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            const int at = col * 128 + ((4 * kk + g) ^ (col / 2)) * 16;
            intx4 fa[TM], fb[TN];
#pragma unroll
            for (int j = 0; j < TM; j++) fa[j] = *reinterpret_cast<const intx4 *>(turn + j * 2048 + at);
#pragma unroll
            for (int i = 0; i < TN; i++) fb[i] = *reinterpret_cast<const intx4 *>(turn + (TM + i) * 2048 + at);
#pragma unroll
            for (int i = 0; i < TN; i++)
#pragma unroll
                for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[i], fa[j], acc[i][j], 0, 0, 0);
        }
        wait_lds();
    };
    Chunk now[kAhead], next[kAhead];
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
    auto sums = [&](int w, int i, int j) -> intx4 & { return *reinterpret_cast<intx4 *>(lds + w * kTurn + ((i * TM + j) * 64 + lane) * 16); };
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) sums(wave, i, j) = acc[i][j];
    __syncthreads();
    for (int p = wave; p < TM * TN; p += WAVES) {
        const int i = p / TM, j = p % TM;
        intx4 total = sums(0, i, j);
#pragma unroll
        for (int w = 1; w < WAVES; w++) total += sums(w, i, j);
        if (a.k == kMostTerms) {
#pragma unroll
            for (int e = 0; e < 4; e++) total[e] = unwrapped(total[e]);
        }
        const int m = m0 + 16 * j + col, n = n0 + 16 * i + 4 * g, left = a.n - n;
        if (m >= a.m || left <= 0) continue;
        float sb[4], bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        some(a.b_scale + n, left, sb);
        if (a.bias) some(a.bias + n, left, bias);
        const float sa = a.a_scale[m];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = scaled(total[e], sa, sb[e], bias[e]);
        T *out = static_cast<T *>(a.out) + m * a.out_stride + n;
        store_some<4>(out, left, v);
    }
}

// A kernel's time: a launch's, then steps of 128 bytes of k by every wave, which
// take `step` each where a CU's workgroups do not fill it, or `work` for each of
// the CU's workgroups where they do, and the workgroup's sums.  Fitted, in us,
// to 4470 products of log-uniform sizes (m 1 .. 8192, n and k 64 .. 16384, up
// to 2^35 multiplications, bf16 out): the kernel of the least time by these is
// 3.6% slower than the fastest of nineteen (tiles of 16 to 256, four or eight
// waves) in the mean, 29% in one of a hundred.
struct Form {
    int tokens, channels, waves;  // of a workgroup; waves that deal k out
    float launch, step, work, sums;
};
constexpr Form kForms[] = {
    {16, 16, 8, 1.97f, 0.0f, 0.797f, 0.244f}, {16, 32, 8, 2.13f, 0.70f, 1.156f, 0.0f},  {32, 32, 8, 1.52f, 0.02f, 1.482f, 0.546f},
    {32, 64, 8, 1.03f, 1.80f, 2.261f, 0.553f}, {64, 64, 4, 2.92f, 1.22f, 1.376f, 0.994f}, {64, 64, 1, 2.49f, 0.446f, 0.331f, 0.797f},
    {128, 128, 1, 2.17f, 0.683f, 0.699f, 2.911f}, {256, 256, 1, 0.0f, 0.30f, 1.582f, 11.93f},
};

int fastest(int64_t m, int64_t n, int64_t k, bool tiles) {
    int best = 4;
    float least = 0.0f;
    for (int i = 0; i < 8; i++) {
        const Form &f = kForms[i];
        const int64_t down = (m + f.tokens - 1) / f.tokens, across = (n + f.channels - 1) / f.channels;
        if (f.waves == 1 ? !tiles || down * across >= 1 << 24 : down > 65535) continue;  // fewer than 2^32 threads along an axis
        const int64_t steps = ((k + 127) / 128 + f.waves - 1) / f.waves, each = (down * across + 255) / 256;
        const float time = f.launch + steps * std::max(f.step, each * f.work) + each * f.sums;
        if (least == 0.0f || time < least) least = time, best = i;
    }
    return best;
}

// the kernel of a call that check() took, as an index of kForms
int form(const Spkv2MatmulI8 &g) {
    const bool far = (g.m > 1 && g.a_stride >= (1 << 23)) || (g.n > 1 && g.b_stride >= (1 << 23));  // 256 rows pass 2^31 bytes
    return fastest(g.m, g.n, g.k, !far && g.k >= 16);
}

int check(const Spkv2MatmulI8 *g, bool pointers) {
    if (!g) return bad("matmul_i8: no arguments");
    if (!is_dtype(g->dtype)) return bad("matmul_i8: unknown dtype");
    if (g->m < 0 || g->n < 0 || g->k < 0) return bad("matmul_i8: negative size");
    if (g->m == 0 || g->n == 0) return 0;
    if (pointers && (!g->out || !g->a_scale || !g->b_scale || (g->k && (!g->a || !g->b)))) return bad("matmul_i8: a NULL pointer");
    if ((g->m > 1 && (g->a_stride < g->k || g->out_stride < g->n)) || (g->n > 1 && g->b_stride < g->k))
        return bad("matmul_i8: a stride is below its row's length");
    if (g->k > kMostTerms) return unsupported("matmul_i8: k above 2^17, whose sums may pass 32 bits");
    if (g->m > (1 << 21) || g->n > (1 << 26)) return unsupported("matmul_i8: m above 2^21 or n above 2^26");
    return 0;
}

}  // namespace

}  // namespace spk::dec

using namespace spk::dec;

extern "C" int spkv2_mi355x_matmul_i8_kernel_name(const Spkv2MatmulI8 *g, char *buf, size_t buf_size) {
    return entry([&]() -> int {
        if (!buf || !buf_size) return bad("matmul_i8: nowhere to put the name");
        if (int rc = check(g, false)) return rc;
        buf[0] = 0;
        if (g->m == 0 || g->n == 0) return 0;
        const Form &f = kForms[form(*g)];
        if (f.waves == 1) snprintf(buf, buf_size, "matmul_tiles<%dx%d>", f.tokens, f.channels);
        else snprintf(buf, buf_size, "matmul_rows<%dx%d,waves=%d>", f.tokens, f.channels, f.waves);
        return 0;
    });
}

extern "C" int spkv2_mi355x_matmul_i8(const Spkv2MatmulI8 *g, void *stream) {
    return entry([&]() -> int {
        if (int rc = check(g, true)) return rc;
        if (g->m == 0 || g->n == 0) return 0;
        MatmulArgs a{g->a, g->b, g->a_scale, g->b_scale, g->bias, g->out, g->a_stride, g->b_stride, g->out_stride,
                     static_cast<int>(g->m), static_cast<int>(g->n), static_cast<int>(g->k), 0, 0};
        if (g->m == 1) a.a_stride = 0, a.out_stride = 0;
        if (g->n == 1) a.b_stride = 0;
        return with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            const char *what = "matmul_i8";
            auto rows = [&](auto kernel, int tm, int tn, int waves) {
                const dim3 grid(static_cast<unsigned>((g->n + 16 * tn - 1) / (16 * tn)), static_cast<unsigned>((g->m + 16 * tm - 1) / (16 * tm)));
                return launch(what, kernel, grid, dim3(64 * waves), stream, a);
            };
            auto tiles = [&](auto kernel, int blocks) {
                a.m_tiles = (a.m + 64 * blocks - 1) / (64 * blocks);
                a.n_tiles = (a.n + 64 * blocks - 1) / (64 * blocks);
                return launch(what, kernel, dim3(static_cast<unsigned>(a.m_tiles * a.n_tiles)), dim3(256), stream, a);
            };
            switch (form(*g)) {
                case 0: return rows(matmul_rows<T, 1, 1, 8>, 1, 1, 8);
                case 1: return rows(matmul_rows<T, 1, 2, 8>, 1, 2, 8);
                case 2: return rows(matmul_rows<T, 2, 2, 8>, 2, 2, 8);
                case 3: return rows(matmul_rows<T, 2, 4, 8>, 2, 4, 8);
                case 4: return rows(matmul_rows<T, 4, 4, 4>, 4, 4, 4);
                case 5: return tiles(matmul_tiles<T, 1>, 1);
                case 6: return tiles(matmul_tiles<T, 2>, 2);
                default: return tiles(matmul_tiles<T, 4>, 4);
            }
        });
    });
}
