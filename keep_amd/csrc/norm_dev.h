#pragma once
// Rows of the norm and of its gradients in registers (norm.hip, norm_grad.hip): TPR threads share a row, NV vectors of eight
// neighbouring values each. Loads and stores are 16 bytes (fp32: 32) wherever a row starts: the memory takes them at any
// address, so that odd widths differ only in the row's last vector.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace keep {

constexpr int NORM_MAX = 16384;  // values of a row: 512 threads of four vectors
constexpr int64_t NORM_BLOCKS = 1 << 22;  // a launch holds 2^32 threads; more rows go round again

// Two values as a 16-bit pair, rounded to nearest even, NaN kept (bf16: one instruction of this GPU, from_float's bits).
template <typename T>
__device__ __forceinline__ uint32_t norm_pair(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(T, bf16s)) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, b2_t));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, h2_t));
}

// How a row ends: whole vectors (n is a multiple of eight), inside one, or before the first one's end. An odd row's last
// vector is read eight values before the row's end, all of it inside the row, and moved down: 4096 rows of 4095 bf16 take 25 us
// (with gradients 57) against 22 (49) of 4096 values. Element by element, each load behind the last one, it was 62 (107).
enum { NORM_EVEN = 0, NORM_ODD = 1, NORM_TINY = 2 };

// Eight values as they lie in memory, read before they are needed.
template <typename T>
struct NormRaw {
  uint32_t w[2 * sizeof(T)];
  template <int END>
  __device__ __forceinline__ void load(const T* row, int i, int n) {
    if (END != NORM_TINY && i < n) {
      __builtin_memcpy(w, row + (END == NORM_ODD ? min(i, n - 8) : i), 8 * sizeof(T));
    } else {
#pragma unroll
      for (int u = 0; u < (int)(2 * sizeof(T)); ++u) w[u] = 0u;
      if constexpr (END == NORM_TINY) {
#pragma unroll
        for (int u = 0; u < 7; ++u)
          if (i + u < n) {
            if constexpr (sizeof(T) == 4) w[u] = __builtin_bit_cast(uint32_t, row[i + u]);
            else w[u / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[i + u]) << (16 * (u & 1));
          }
      }
    }
  }
  // i, n: load's. Zeros past the row's end.
  template <int END>
  __device__ __forceinline__ void get(int i, int n, float (&f)[8]) const {
    constexpr int W = 2 * sizeof(T), PER = 4 / sizeof(T);  // words, and values of a word
    uint32_t m[W];
#pragma unroll
    for (int u = 0; u < W; ++u) m[u] = w[u];
    if (END == NORM_ODD && i + 8 > n) {
      const int down = min(i + 8 - n, 8);
#pragma unroll
      for (int s = 8; s >= PER; s /= 2)
        if (down & s)
#pragma unroll
          for (int u = 0; u < W; ++u) m[u] = u + s / PER < W ? m[u + s / PER < W ? u + s / PER : 0] : 0u;
      if (PER == 2 && (down & 1))
#pragma unroll
        for (int u = 0; u < W; ++u) m[u] = m[u] >> 16 | (u + 1 < W ? m[u + 1 < W ? u + 1 : 0] << 16 : 0u);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if constexpr (sizeof(T) == 4) f[u] = __uint_as_float(m[u]);
      else f[u] = (u & 1) ? pair_hi<PairOf<T>::value>(m[u / 2]) : pair_lo<PairOf<T>::value>(m[u / 2]);
    }
  }
};

// Values i .. i + 8 of a row of n, zeros past its end.
template <int END, typename T>
__device__ __forceinline__ void norm_ld(const T* row, int i, int n, float (&f)[8]) {
  NormRaw<T> r;
  r.template load<END>(row, i, n);
  r.template get<END>(i, n, f);
}

template <int END, typename T>
__device__ __forceinline__ void norm_st(T* row, int i, int n, const float (&f)[8]) {
  if (END == NORM_EVEN ? i < n : i + 8 <= n) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = norm_pair<T>(f[2 * u], f[2 * u + 1]);
      __builtin_memcpy(row + i, w, 16);
    } else {
      __builtin_memcpy(row + i, f, 32);
    }
  } else if constexpr (END != NORM_EVEN) {
#pragma unroll
    for (int u = 0; u < 7; ++u)
      if (i + u < n) row[i + u] = from_float<T>(f[u]);
  }
}

// The weight's values (none: ones).
template <int END>
__device__ __forceinline__ void norm_weight(const void* w, int dt, int i, int n, float (&f)[8]) {
  if (!w) {
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = 1.f;
  } else if (dt == KEEP_F32) {
    norm_ld<END>((const float*)w, i, n, f);
  } else if (dt == KEEP_BF16) {
    norm_ld<END>((const bf16s*)w, i, n, f);
  } else {
    norm_ld<END>((const _Float16*)w, i, n, f);
  }
}

// The sum of v over a row's TPR threads, in every one of them; red: a value per wave of the block.
template <int TPR, int BT>
__device__ __forceinline__ float norm_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6, first = threadIdx.x / TPR * (TPR / 64);
    __syncthreads();  // the last sum is read
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[first + i];
  }
  return v;
}

// f(TPR, NV, END) for rows of n values: as many threads as a row has vectors, up to 512. Few rows wait for one row, which more
// threads shorten, many rows for HBM. bf16 with a residual, 16 rows / 8192 rows, microseconds: 2048 values by 256 threads 3.5 /
// 22.9, by 64 with four vectors 4.8 / 22.6; 4096 by 512 3.6 / 40.7, by 256 4.1 / 40.0; 7168 by 512 4.4 / 84.7, by 256 5.0 / 86.5,
// by 1024 4.0 and the 8-bit form of 4096 rows 40.6 for 38.2. Where a wave holds a row no block waits: 1024 by 64 3.9 / 11.9, by
// 256 3.6 / 14.4.
template <typename F>
void norm_by_width(int64_t n, F f) {
  using std::integral_constant;
  constexpr integral_constant<int, 64> t64;
  constexpr integral_constant<int, 256> t256;
  constexpr integral_constant<int, 512> t512;
  constexpr integral_constant<int, 1> v1;
  constexpr integral_constant<int, 2> v2;
  constexpr integral_constant<int, 4> v4;
  const auto by = [&](auto end) {
    if (n <= 512) f(t64, v1, end);
    else if (n <= 1024) f(t64, v2, end);
    else if (n <= 2048) f(t256, v1, end);
    else if (n <= 4096) f(t512, v1, end);
    else if (n <= 8192) f(t512, v2, end);
    else f(t512, v4, end);
  };
  if (n < 8) f(t64, v1, integral_constant<int, NORM_TINY>{});
  else if (n % 8) by(integral_constant<int, NORM_ODD>{});
  else by(integral_constant<int, NORM_EVEN>{});
}

}  // namespace keep

// What the three entry points ask of their rows.
#define KEEP_REQUIRE_NORM(T, n, eps)                                                                        \
  KEEP_REQUIRE_DIMS(T, n);                                                                                  \
  KEEP_REQUIRE(n >= 1 && n <= NORM_MAX, "rows must hold 1..%d values, got %lld", NORM_MAX, (long long)(n)); \
  KEEP_REQUIRE((eps) >= 0.f, "eps must be non-negative")
