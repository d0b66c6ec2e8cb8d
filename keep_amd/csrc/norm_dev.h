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

// Eight values as they lie in memory, read before they are needed.
template <typename T>
struct NormRaw {
  uint32_t w[2 * sizeof(T)];
  template <bool EVEN>
  __device__ __forceinline__ void load(const T* row, int i, int n) {
    if (EVEN ? i < n : i + 8 <= n) {
      __builtin_memcpy(w, row + i, 8 * sizeof(T));
    } else {
#pragma unroll
      for (int u = 0; u < (int)(2 * sizeof(T)); ++u) w[u] = 0u;
      if constexpr (!EVEN) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (i + u < n) {
            if constexpr (sizeof(T) == 4) w[u] = __builtin_bit_cast(uint32_t, row[i + u]);
            else w[u / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[i + u]) << (16 * (u & 1));
          }
      }
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if constexpr (sizeof(T) == 4) f[u] = __uint_as_float(w[u]);
      else f[u] = (u & 1) ? pair_hi<PairOf<T>::value>(w[u / 2]) : pair_lo<PairOf<T>::value>(w[u / 2]);
    }
  }
};

// Values i .. i + 8 of a row of n, zeros past its end. EVEN: n is a multiple of eight.
template <bool EVEN, typename T>
__device__ __forceinline__ void norm_ld(const T* row, int i, int n, float (&f)[8]) {
  NormRaw<T> r;
  r.template load<EVEN>(row, i, n);
  r.get(f);
}

template <bool EVEN, typename T>
__device__ __forceinline__ void norm_st(T* row, int i, int n, const float (&f)[8]) {
  if (EVEN ? i < n : i + 8 <= n) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = norm_pair<T>(f[2 * u], f[2 * u + 1]);
      __builtin_memcpy(row + i, w, 16);
    } else {
      __builtin_memcpy(row + i, f, 32);
    }
  } else if constexpr (!EVEN) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < n) row[i + u] = from_float<T>(f[u]);
  }
}

// The weight's values (none: ones).
template <bool EVEN>
__device__ __forceinline__ void norm_weight(const void* w, int dt, int i, int n, float (&f)[8]) {
  if (!w) {
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = 1.f;
  } else if (dt == KEEP_F32) {
    norm_ld<EVEN>((const float*)w, i, n, f);
  } else if (dt == KEEP_BF16) {
    norm_ld<EVEN>((const bf16s*)w, i, n, f);
  } else {
    norm_ld<EVEN>((const _Float16*)w, i, n, f);
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

// f(TPR, NV, EVEN) for rows of n values.
template <typename F>
void norm_by_width(int64_t n, F f) {
  using T64 = std::integral_constant<int, 64>;
  using T256 = std::integral_constant<int, 256>;
  using T512 = std::integral_constant<int, 512>;
  using V1 = std::integral_constant<int, 1>;
  using V2 = std::integral_constant<int, 2>;
  using V4 = std::integral_constant<int, 4>;
  if (n % 8) {
    if (n <= 2048) f(T64{}, V4{}, std::false_type{});
    else if (n <= 8192) f(T256{}, V4{}, std::false_type{});
    else f(T512{}, V4{}, std::false_type{});
  } else if (n <= 512) f(T64{}, V1{}, std::true_type{});
  else if (n <= 1024) f(T64{}, V2{}, std::true_type{});
  else if (n <= 2048) f(T64{}, V4{}, std::true_type{});
  else if (n <= 4096) f(T256{}, V2{}, std::true_type{});
  else if (n <= 8192) f(T256{}, V4{}, std::true_type{});
  else f(T512{}, V4{}, std::true_type{});
}

}  // namespace keep

// What the three entry points ask of their rows.
#define KEEP_REQUIRE_NORM(T, n, eps)                                                                        \
  KEEP_REQUIRE_DIMS(T, n);                                                                                  \
  KEEP_REQUIRE(n >= 1 && n <= NORM_MAX, "rows must hold 1..%d values, got %lld", NORM_MAX, (long long)(n)); \
  KEEP_REQUIRE((eps) >= 0.f, "eps must be non-negative")
