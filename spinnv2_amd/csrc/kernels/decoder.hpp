// What the decoder layer's operators share: types, conversions, the checks of
// their C entry points.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <exception>

#include "../runtime/context.hpp"
#include "spkv2_decoder.h"

namespace spk::dec {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;

// ---- device ----------------------------------------------------------------

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

// N elements at p as floats, 16 bytes an instruction.  Any alignment will do:
// the memory units take wide accesses at every address, and one that crosses
// a line costs a second request, not a byte's each.
template <int N, typename T>
__device__ __forceinline__ void load_floats(const T *p, float (&f)[N]) {
    constexpr int kPer = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += kPer) {
        Vec<T, kPer> x;
        __builtin_memcpy(x.v, p + i, sizeof(x.v));
#pragma unroll
        for (int j = 0; j < kPer; j++) f[i + j] = static_cast<float>(x.v[j]);
    }
}
template <int N, typename T>
__device__ __forceinline__ void store_floats(T *p, const float (&f)[N]) {
    constexpr int kPer = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += kPer) {
        Vec<T, kPer> x;
#pragma unroll
        for (int j = 0; j < kPer; j++) x.v[j] = static_cast<T>(f[i + j]);
        __builtin_memcpy(p + i, x.v, sizeof(x.v));
    }
}
// To LDS, aligned to all N elements.
template <int N, typename T>
__device__ __forceinline__ void put_floats(T *p, const float (&f)[N]) {
    Vec<T, N> x;
#pragma unroll
    for (int j = 0; j < N; j++) x.v[j] = static_cast<T>(f[j]);
    *reinterpret_cast<Vec<T, N> *>(p) = x;
}
// N elements that were loaded from min(i, cols - N) of a row of `cols`, as those
// from i on, zeros past the row's end.  All lanes load so, without a branch:
// under one each of a row's loads is waited for by itself.  TAIL: cols is no
// multiple of N.
template <int N, bool TAIL>
__device__ __forceinline__ void settle(int i, int cols, float (&f)[N]) {
    const int past = i + N - cols;
    if constexpr (TAIL) {
        if (past > 0) {
#pragma unroll
            for (int step = 1; step < N; step *= 2)
#pragma unroll
                for (int j = 0; j < N; j++) f[j] = past & step ? (j + step < N ? f[(j + step) % N] : 0.0f) : f[j];
#pragma unroll
            for (int j = 0; j < N; j++) f[j] = past >= N ? 0.0f : f[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = past > 0 ? 0.0f : f[j];
    }
}
// The first `left` of N elements.
template <int N, typename T>
__device__ __forceinline__ void store_some(T *p, int left, const float (&f)[N]) {
    if (left >= N) {
        store_floats<N>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = static_cast<T>(f[i]);
    }
}

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T *p) {
    Vec<T, N> x;
    __builtin_memcpy(x.v, p, sizeof(x.v));
    return x;
}
template <typename T, int N>
__device__ __forceinline__ void widen(const Vec<T, N> &x, float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; j++) f[j] = static_cast<float>(x.v[j]);
}

constexpr unsigned kInfBits = 0x7f800000u;
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint64_t abs_bits(double x) {
    return static_cast<uint64_t>(__double_as_longlong(x)) & 0x7fffffffffffffffull;
}

// rint(127 x / top) in exact arithmetic, 0 <= x <= top, both of at most 48 bits
// (products of two fp32 values).  127 x has up to 55 bits and a quotient may lie
// closer to a border of two codes than a double tells, so only its integer part
// n is taken from one; whether the border n + 1/2 is passed, (2 n + 1) top <
// 254 x, is one fused product: 256 x - (2 n + 1) top is a multiple of 2^-47 of
// x's power of two, so where it is near 2 x it has at most 50 bits and no rounding.
__device__ __forceinline__ double exact_code(double x, double top) {
    const double n = floor(x * 127.0 / top), rest = __builtin_fma(-(2.0 * n + 1.0), top, 256.0 * x);
    return rest > 2.0 * x || (rest == 2.0 * x && (static_cast<int>(n) & 1)) ? n + 1.0 : n;
}

// Codes rint(127 x / top) of N values with |x| <= top, top > 0 finite.  With
// x, 127 / top and their product each rounded to fp32, t is within 127 * 4 *
// 2^-24 < 2^-15 of the quotient, so it has the quotient's nearest integer
// unless it lies within 2^-14 of the border of two.  One value in eight
// thousand does, and where 127 / top or a wide x leaves fp32's range all do (t
// is then infinite or NaN): those are divided in 64 bits, and so is every value
// where a wide top passes fp32's range, 127 / top is 0 and t says nothing.
template <int N, typename P>
__device__ __forceinline__ void quantise(const P (&x)[N], P top, int8_t (&q)[N]) {
    const float inv = 127.0f / static_cast<float>(top);
    float r[N];
    bool far[N], all = true;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float t = static_cast<float>(x[i]) * inv;
        r[i] = rintf(t);
        far[i] = inv > 0.0f && fabsf(t - r[i]) < 0.5f - 0x1p-14f;
        all &= far[i];
    }
    if (!all) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (!far[i]) r[i] = static_cast<float>(copysign(exact_code(fabs(static_cast<double>(x[i])), static_cast<double>(top)), static_cast<double>(x[i])));
    }
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = static_cast<int8_t>(static_cast<int>(r[i]));
}

// The largest of v over groups of LANES neighbouring lanes (8, 16 or 32), in
// each of them: within 16 by lane moves of the adder's own, past that by LDS's
// crossbar.
template <int LANES>
__device__ __forceinline__ unsigned max_over(unsigned v) {
    v = max(v, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));   // lanes 1 0 3 2
    v = max(v, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));   // lanes 2 3 0 1
    v = max(v, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, true)));  // eight lanes mirrored
    if constexpr (LANES >= 16) v = max(v, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xF, 0xF, true)));  // 16 mirrored
    if constexpr (LANES >= 32) v = max(v, static_cast<unsigned>(__shfl_xor(static_cast<int>(v), 16)));
    return v;
}

// ---- host ------------------------------------------------------------------

inline int bad(const char *text) {
    set_last_error_text(text);
    return -1;
}
inline int unsupported(const char *text) {
    set_last_error_text(text);
    return SPKV2_E_UNSUPPORTED;
}
inline bool is_dtype(int d) { return d == SPKV2_DTYPE_FP32 || d == SPKV2_DTYPE_FP16 || d == SPKV2_DTYPE_BF16; }
inline bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// (mul, shift) with n / d = n mul >> shift for 0 <= n < 2^31, d >= 1: mul =
// ceil(2^shift / d), shift = 31 + ceil(log2 d)
inline void div_magic(unsigned d, unsigned *mul, int *shift) {
    int l = 0;
    while ((uint64_t(1) << l) < d) l++;
    *shift = 31 + l;
    *mul = static_cast<unsigned>(((uint64_t(1) << *shift) + d - 1) / d);
}

// f(T{}) with the element type of a dtype that is_dtype() took
template <typename F>
inline int with_type(int dtype, F &&f) {
    if (dtype == SPKV2_DTYPE_FP32) return f(float{});
    if (dtype == SPKV2_DTYPE_FP16) return f(_Float16{});
    return f(__bf16{});
}

// No exception leaves a C entry point.
template <typename F>
inline int entry(F &&f) noexcept {
    try {
        return f();
    } catch (const std::exception &) {
        return -1;
    }
}

// Launches kernel(args), and returns this launch's own status, where
// hipGetLastError would also give an earlier call's.
template <typename A>
inline int launch(const char *what, void (*kernel)(A), dim3 grid, dim3 block, void *stream, A args) {
    void *ptrs[] = {&args};
    return hip_check(hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, ptrs, 0,
                                     static_cast<hipStream_t>(stream)),
                     what);
}

int check_cache(const Spkv2KvCacheI8 *c);

}  // namespace spk::dec
