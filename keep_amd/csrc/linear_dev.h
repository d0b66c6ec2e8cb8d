#pragma once
// What the dense projection's kernels share: the epilogue and the arguments of the products through LDS.
//   u = x W^T + b,  out = round(residual + act(u))
#include <type_traits>

#include "dense_dev.h"

namespace keep {

struct e4m3s {
  uint8_t bits;
};

enum { LINEAR_NONE = 0, LINEAR_RELU = 1, LINEAR_SILU = 2, LINEAR_GELU = 3, LINEAR_GELU_TANH = 4 };

// exp through v_exp_f32 and reciprocals through v_rcp_f32: |u| 2^-24 + 2^-22 of the value, a few instructions where expf and
// a division take forty (8192 x 8192 outputs of silu: their share of a product's epilogue).
__device__ __forceinline__ float linear_sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __expf(-u)); }

constexpr float GELU_C = 0.7978845608028654f;  // sqrt(2 / pi)

// (ACT by value: a choice per value would be a branch per value.)
template <int ACT>
__device__ __forceinline__ float linear_act(float u) {
  constexpr int act = ACT;
  if (act == LINEAR_RELU) return u > 0.f ? u : u != u ? u : 0.f;
  if (act == LINEAR_SILU) return u * linear_sigmoid(u);
  if (act == LINEAR_GELU) return 0.5f * u * erfcf(u * -0.7071067811865476f);  // (erfc keeps the lower tail's bits)
  // 0.5 (1 + tanh(v)) = sigmoid(2 v)
  if (act == LINEAR_GELU_TANH) return u * linear_sigmoid(2.f * GELU_C * (u + 0.044715f * u * u * u));
  return u;
}

template <int V>
__device__ __forceinline__ void linear_act(float (&f)[V], int act) {
  const auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = linear_act<decltype(a)::value>(f[i]);
  };
  if (act == LINEAR_SILU) all(std::integral_constant<int, LINEAR_SILU>{});
  else if (act == LINEAR_GELU) all(std::integral_constant<int, LINEAR_GELU>{});
  else if (act == LINEAR_GELU_TANH) all(std::integral_constant<int, LINEAR_GELU_TANH>{});
  else if (act == LINEAR_RELU) all(std::integral_constant<int, LINEAR_RELU>{});
}

template <int ACT>
__device__ __forceinline__ float linear_slope(float u) {
  constexpr int act = ACT;
  if (act == LINEAR_RELU) return u > 0.f ? 1.f : u != u ? u : 0.f;
  // (at their ends 1 and 0 without infinity times 0: u that is kept in 16 bits may have become infinite)
  if (act == LINEAR_SILU) {
    if (fabsf(u) > 128.f) return u > 0.f ? 1.f : 0.f;
    const float p = linear_sigmoid(u);
    return p * (1.f + u * (1.f - p));
  }
  if (act == LINEAR_GELU) {
    if (fabsf(u) > 16.f) return u > 0.f ? 1.f : 0.f;
    return 0.5f * erfcf(u * -0.7071067811865476f) + u * __expf(-0.5f * u * u) * 0.3989422804014327f;
  }
  if (act == LINEAR_GELU_TANH) {
    if (fabsf(u) > 16.f) return u > 0.f ? 1.f : 0.f;  // (u^2 of the largest values would overflow)
    const float p = linear_sigmoid(2.f * GELU_C * (u + 0.044715f * u * u * u));
    return p + u * p * (1.f - p) * 2.f * GELU_C * (1.f + 3.f * 0.044715f * u * u);
  }
  return 1.f;
}

// 8-bit values enter the matrix cores as float16, which holds every e4m3 value: the 8-bit products of this GPU (16x16x32 and
// 16x16x128 alike) add what they are given at about 13 bits below the largest term (up to 4900 x 2^-23 of it off, measured on
// 128 terms; as float16 7.6).
typedef _Float16 linear_h8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ linear_h8 linear_e4m3(uint32_t lo, uint32_t hi) {
  union {
    h2_t p[4];
    linear_h8 v;
  } f;
  f.p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  f.p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  f.p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  f.p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return f.v;
}
// The 32 values of a lane's two pieces as the operands of four products.
__device__ __forceinline__ void linear_e4m3(const uint4& a, const uint4& b, linear_h8 (&f)[4]) {
  f[0] = linear_e4m3(a.x, a.y);
  f[1] = linear_e4m3(a.z, a.w);
  f[2] = linear_e4m3(b.x, b.y);
  f[3] = linear_e4m3(b.z, b.w);
}

// d *= act'(u)
template <int V>
__device__ __forceinline__ void linear_slope(float (&d)[V], const float (&u)[V], int act) {
  const auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] *= linear_slope<decltype(a)::value>(u[i]);
  };
  if (act == LINEAR_SILU) all(std::integral_constant<int, LINEAR_SILU>{});
  else if (act == LINEAR_GELU) all(std::integral_constant<int, LINEAR_GELU>{});
  else if (act == LINEAR_GELU_TANH) all(std::integral_constant<int, LINEAR_GELU_TANH>{});
  else if (act == LINEAR_RELU) all(std::integral_constant<int, LINEAR_RELU>{});
}

// n <= V neighbouring values of a row; vec: V of them at an address aligned to them.
template <typename T, int V>
__device__ __forceinline__ void linear_ld(const T* p, int64_t n, float (&f)[V], bool vec) {
  if (vec && n >= V) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float4 q = ((const float4*)p)[i];
        f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const uint2 q = ((const uint2*)p)[i];
        f[4 * i] = pair_lo<PairOf<T>::value>(q.x); f[4 * i + 1] = pair_hi<PairOf<T>::value>(q.x);
        f[4 * i + 2] = pair_lo<PairOf<T>::value>(q.y); f[4 * i + 3] = pair_hi<PairOf<T>::value>(q.y);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < n ? to_float(p[i]) : 0.f;
  }
}

template <int V>
__device__ __forceinline__ void linear_ld_any(const void* p, int dt, int64_t at, int64_t n, float (&f)[V], bool vec) {
  if (dt == KEEP_F32) linear_ld<float, V>((const float*)p + at, n, f, vec);
  else if (dt == KEEP_BF16) linear_ld<bf16s, V>((const bf16s*)p + at, n, f, vec);
  else linear_ld<_Float16, V>((const _Float16*)p + at, n, f, vec);
}

// V neighbouring values of a row, n of them inside. Pairs are rounded by one instruction each (to nearest even, NaN kept).
template <typename T, int V>
__device__ __forceinline__ void linear_st(T* p, int64_t n, const float (&f)[V], bool vec) {
  if constexpr (sizeof(T) == 2) {
    if (vec && n >= V) {
      typedef float f2 __attribute__((ext_vector_type(2)));
      uint32_t w[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (__is_same(T, bf16s))
          w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{f[2 * i], f[2 * i + 1]}, b2_t));
        else w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{f[2 * i], f[2 * i + 1]}, h2_t));
      }
      if constexpr (V % 8 == 0) {
#pragma unroll
        for (int i = 0; i < V / 8; ++i)
          ((uint4*)p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      } else {
        *(uint2*)p = make_uint2(w[0], w[1]);
      }
      return;
    }
  }
  dense_st<T, V>(p, n, f, vec);
}

template <int V>
__device__ __forceinline__ void linear_st_any(void* p, int dt, int64_t at, int64_t n, const float (&f)[V], bool vec) {
  if (dt == KEEP_F32) linear_st<float, V>((float*)p + at, n, f, vec);
  else if (dt == KEEP_BF16) linear_st<bf16s, V>((bf16s*)p + at, n, f, vec);
  else linear_st<_Float16, V>((_Float16*)p + at, n, f, vec);
}

struct LinearEpilogue {
  const void* bias;  // [N] or null
  int bdt, act;
  const void* res;  // [M][N] or null
  int rdt;
  void* u;  // [M][N], the values before the activation, or null
  int udt;
  void* out;  // [M][N]
  int odt;
  int vec;  // N is a multiple of eight and every pointer 16-byte aligned: pieces of up to eight values are read and stored whole

  // The values at (row, col ..): n of them are inside.
  template <int V>
  __device__ __forceinline__ void store(int64_t row, int64_t N, int64_t col, int64_t n, float (&f)[V],
                                        const float (&b)[V]) const {
    const int64_t at = row * N + col;
    const bool v = vec;
    if (bias)
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] += b[i];
    if (u) linear_st_any<V>(u, udt, at, n, f, v);
    if (act) linear_act<V>(f, act);
    if (res) {
      float r[V];
      linear_ld_any<V>(res, rdt, at, n, r, v);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = r[i] + f[i];
    }
    linear_st_any<V>(out, odt, at, n, f, v);
  }
  template <int V>
  __device__ __forceinline__ void load_bias(int64_t col, int64_t n, float (&b)[V]) const {
    if (bias) linear_ld_any<V>(bias, bdt, col, n, b, vec);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = 0.f;
  }
};

// A product of two matrices, out[j][i] = sum over k of J[j][k] I[i][k], whose sides either run along the summed index
// (pitch between rows j or i) or across it (pitch between rows k).
struct LinearGemmArgs {
  const void *pi, *pj;
  int64_t ldi, ldj;  // values between rows, whole 16-byte pieces
  int64_t ni, nj, nk;
  int slices;       // of the summed index; more than one: sums go to part
  float* part;      // [slices][nj][ni]
  int any;          // few rows: rows at any address, and any number of values
  const float *si, *sj;  // 8-bit: scales [ceil(ni / 128)][ceil(nk / 128)] and [nj][ceil(nk / 128)]
  LinearEpilogue e;
};

// Columns x rows of a tile, and the groups of waves that share its sum (2: two).
enum { LINEAR_TILE_FEW = 0, LINEAR_TILE_64, LINEAR_TILE_128_2, LINEAR_TILE_128, LINEAR_TILE_256_128, LINEAR_TILE_256 };
enum { LINEAR_FORWARD = 0, LINEAR_ROWS = 1, LINEAR_WEIGHT = 2 };  // out, dx, dW

}  // namespace keep
