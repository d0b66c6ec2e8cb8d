#pragma once
// Matrix-core fragments of dense rows, straight from global memory.
//
// A 16x16 MFMA sums first[i] . second[j] over a K step: lane (c, q) = (l % 16,
// l / 16) holds row c of both operands at the step's q-th quarter, and the
// result's lane (c, q) holds i = 4 q + v (v = 0..3) of j = c. The first operand
// here is the side whose index is contiguous in the output (a lane then has
// four neighbouring outputs), the second the routes' rows.
//
// fp16 and bf16: 8 values (16 bytes) per lane and step, 32 k. float: 4 values
// (16 bytes) per lane, 16 k, as four 16x16x4 products (product s takes value s
// of every lane: the same permutation of k on both sides).
#include "common.h"

namespace keep {

typedef float f4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Dense {
  static constexpr int V = 16 / sizeof(T);  // values of a lane's fragment
  static constexpr int KS = 4 * V;          // k per step
};

template <typename T>
__device__ __forceinline__ f4 dense_mfma(const uint4& i, const uint4& j, f4 acc) {
  if constexpr (sizeof(T) == 4) {
    const float a[4] = {__uint_as_float(i.x), __uint_as_float(i.y), __uint_as_float(i.z), __uint_as_float(i.w)};
    const float b[4] = {__uint_as_float(j.x), __uint_as_float(j.y), __uint_as_float(j.z), __uint_as_float(j.w)};
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], acc, 0, 0, 0);
    return acc;
  } else if constexpr (__is_same(T, bf16s)) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, i), __builtin_bit_cast(b8, j), acc, 0, 0, 0);
  } else {
    typedef _Float16 h8v __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, i), __builtin_bit_cast(h8v, j), acc, 0, 0, 0);
  }
}

// Values k .. k + V of a row, all there, at an aligned address.
template <typename T>
__device__ __forceinline__ uint4 dense_ld16(const T* row, int64_t k) {
  typedef unsigned int v4u __attribute__((ext_vector_type(4)));
  const v4u v = *(const __attribute__((address_space(1))) v4u*)(row + k);
  return uint4{v.x, v.y, v.z, v.w};
}

// Values k .. k + V of a row of n values, zeros past its end. VEC: rows hold whole 16-byte fragments at aligned addresses.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 dense_ld(const T* row, int64_t k, int64_t n) {
  if constexpr (VEC) {
    return k < n ? dense_ld16(row, k) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < Dense<T>::V; ++i) {
      if (k + i < n) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(row[k + i]);
        else w[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, row[k + i]) << (16 * (i & 1));
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Value u of a fragment as a float.
template <typename T>
__device__ __forceinline__ float dense_at(const uint4& f, int u) {
  const uint32_t w[4] = {f.x, f.y, f.z, f.w};
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[u]);
  else return (u & 1) ? pair_hi<PairOf<T>::value>(w[u >> 1]) : pair_lo<PairOf<T>::value>(w[u >> 1]);
}

// n <= V consecutive outputs.
template <typename T, int V>
__device__ __forceinline__ void dense_st(T* p, int64_t n, const float (&f)[V], bool vec) {
  if (vec && n >= V) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        ((float4*)p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
    } else {
      uint32_t w[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(f[2 * i])) |
               ((uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(f[2 * i + 1])) << 16);
      if constexpr (V % 8 == 0) {
#pragma unroll
        for (int i = 0; i < V / 8; ++i) ((uint4*)p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) ((uint2*)p)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = from_float<T>(f[i]);
  }
}

// The routes of a tile of up to 16, grouped without a plan: position r of a window of 128 positions heads a tile if a
// multiple of 16 earlier positions of the window share its group; the tile is those of the next 16 that do. A wave keeps
// the window's groups in two registers and finds a tile with two ballots.
constexpr int DENSE_WINDOW = 128;
struct DenseTile {
  int group;
  int count;     // routes of the tile (0: the position heads none)
  int64_t mine;  // position of the tile's row c = lane % 16 (-1: none)
};

struct DenseWindow {
  int64_t base;
  int g0, g1;     // groups of positions base + lane and base + 64 + lane
  uint64_t v0, v1;

  template <typename Group>
  __device__ __forceinline__ DenseWindow(Group group, int64_t r, int64_t routes, int lane) {
    base = r / DENSE_WINDOW * DENSE_WINDOW;
    const bool h0 = base + lane < routes, h1 = base + 64 + lane < routes;
    g0 = h0 ? group(base + lane) : 0;
    g1 = h1 ? group(base + 64 + lane) : 0;
    v0 = __ballot(h0);
    v1 = __ballot(h1);
  }

  // r: a position of this window, the same in every lane
  __device__ __forceinline__ DenseTile tile(int64_t r, int lane) const {
    const int at = __builtin_amdgcn_readfirstlane((int)(r - base));
    DenseTile t;
    t.group = at < 64 ? __builtin_amdgcn_readlane(g0, at) : __builtin_amdgcn_readlane(g1, at - 64);
    t.count = 0;
    t.mine = -1;
    const uint64_t m0 = __ballot(g0 == t.group) & v0, m1 = __ballot(g1 == t.group) & v1;
    const int n0 = __popcll(m0);
    const int below = at < 64 ? __popcll(m0 & ((1ull << at) - 1ull)) : n0 + __popcll(m1 & ((1ull << (at - 64)) - 1ull));
    if (below & 15) return t;
    t.count = min(16, n0 + __popcll(m1) - below);
    const int c = lane & 15;
    if (c < t.count) {  // the (below + c)-th set bit, by halving
      int k = below + c, pos = 0;
      uint64_t m = m0;
      if (k >= n0) {
        k -= n0;
        m = m1;
        pos = 64;
      }
      int at2 = 0;
#pragma unroll
      for (int w = 32; w >= 1; w >>= 1) {
        const int n = __popcll((m >> at2) & ((1ull << w) - 1ull));
        if (k >= n) {
          k -= n;
          at2 += w;
        }
      }
      t.mine = base + pos + at2;
    }
    return t;
  }
};

}  // namespace keep
