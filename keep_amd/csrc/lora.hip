// Low-rank adapters of many requests at once, added to a projection's rows:
//
//   out[r] = base[r] + s[a] (x[row_r] A[a]^T) B[a]^T,   a = idx[r]   (A [n][R][K], B [n][N][R])
//
// a < 0: no adapter (out = base, or zeros); a >= n: a NaN row. Two launches over
// the same tiles of up to 32 neighbouring routes of one adapter:
//
// k_lora_shrink: t = x A^T. Blocks along K take a slice each; a block's waves
// share the slice and are added in order through LDS, and the slice's partial t
// goes to the workspace in fp32.
// k_lora_expand: adds the slices in order, times s, and streams B's rows of the
// block's columns: out = base + t B^T.
//
// Tiles need no plan: a wave finds the runs of one adapter in a window of 128
// positions with two ballots (LoraWindow), since rows of a request lie together
// in a batch. Routes of several experts do not: those come with a plan's order.
// One launch that repeats t in every block of columns took 1.1 to 1.6 times as
// long at every size (one CU reads A, where the slices read it on many).
//
// Bound: the dependent loads at a block's start (window, partial sums, rows):
// waves wait 48 % (shrink) and 57 % (expand) of their cycles at 4093 rows.
// In a graph, both launches: one row, r = 16, 4096 -> 4096, 8.5 us, of which two
// empty launches take about 5; 64 requests of r = 64, 4096 -> 2048, 17 us, the
// bytes alone 7; 4093 rows in runs of about 100, r = 32, 4096 -> 4096, 49 us (17
// + 32), the bytes alone 21.
//
// t enters the second product whole: in 16 bits as a sum of terms of that type,
// each row times a power of two that brings its largest finite value to [1, 4).
// Three bf16 terms hold float's 24 bits; two of fp16 hold 22, and are off by at
// most 2^-25 of the row's largest value. (One term is a rounding to 8 or 11 bits
// of every t; the others take 1 us of the 52 for 4093 rows, nothing for 64.) float rows
// stay float throughout.
#include <algorithm>
#include <type_traits>

#include "dense_dev.h"
#include "dense_outer.h"

namespace keep {

constexpr int LS_WAVES = 8, LE_WAVES = 8;
constexpr int LORA_ROWS = 32;  // of a tile
constexpr int64_t LORA_BLOCKS = 0xffffffffLL / (64 * LS_WAVES);  // a launch holds 2^32 threads

struct LoraArgs {
  const void* x;
  int64_t x_rows;
  const void *a, *b;
  const float* scales;  // null: ones
  const int32_t *idx, *order;
  int64_t routes, x_div;
  int64_t n, R, K, N;
  int heads;      // blocks per window: each takes every heads-th tile
  int64_t split;  // slices of K; blocks along N
  int64_t slices;
  float* ws;  // [slices][routes][16 RT]
  float* t_out;
  const void* base;  // null: zeros
  void* out;  // null: t_out alone
};

struct LoraTile {
  int g, count;   // adapter (-1: none, n: out of range), routes (0: no tile)
  int64_t first;  // their first position
  bool has;
};

// The tiles of 128 positions: runs of one adapter, cut after LORA_ROWS rows.
struct LoraWindow {
  int64_t base;
  int g0, g1, valid;
  uint64_t h0, h1;  // positions that start a tile

  __device__ __forceinline__ LoraWindow(const LoraArgs& a, int64_t window, int lane) {
    base = window * 128;
    valid = (int)min((int64_t)128, a.routes - base);
    auto group = [&](int64_t p) {
      const int g = a.idx[a.order ? (int64_t)a.order[p] : p];
      return g < 0 ? -1 : g >= a.n ? (int)a.n : g;
    };
    g0 = lane < valid ? group(base + lane) : -2;
    g1 = lane + 64 < valid ? group(base + 64 + lane) : -2;
    const int p0 = __shfl_up(g0, 1, 64), p1 = __shfl_up(g1, 1, 64), last = __builtin_amdgcn_readlane(g0, 63);
    const uint64_t f0 = __ballot(lane < valid && (lane == 0 || g0 != p0));
    const uint64_t f1 = __ballot(lane + 64 < valid && g1 != (lane == 0 ? last : p1));
    // from its run's start on, every LORA_ROWS-th position starts a tile
    const uint64_t upto = (2ull << lane) - 1ull;
    const int s0 = 63 - __clzll(f0 & upto), s1 = f1 & upto ? 127 - __clzll(f1 & upto) : 63 - __clzll(f0);
    h0 = __ballot(lane < valid && ((lane - s0) & (LORA_ROWS - 1)) == 0);
    h1 = __ballot(lane + 64 < valid && ((lane + 64 - s1) & (LORA_ROWS - 1)) == 0);
  }

  __device__ __forceinline__ int tiles() const { return __popcll(h0) + __popcll(h1); }

  __device__ __forceinline__ LoraTile tile(const LoraArgs& a, int k) const {
    const int n0 = __popcll(h0);
    uint64_t m = k < n0 ? h0 : h1;
    int i = k < n0 ? k : k - n0, at = 0;
#pragma unroll
    for (int w = 32; w >= 1; w >>= 1) {  // the i-th set bit of m, by halving
      const int n = __popcll((m >> at) & ((1ull << w) - 1ull));
      if (i >= n) {
        i -= n;
        at += w;
      }
    }
    m = at == 63 ? 0 : m >> (at + 1) << (at + 1);
    const int pos = __builtin_amdgcn_readfirstlane(at + (k < n0 ? 0 : 64));
    int end = m ? __ffsll((unsigned long long)m) - 1 + (pos & 64) : pos < 64 && h1 ? 63 + __ffsll((unsigned long long)h1) : valid;
    LoraTile t;
    t.g = pos < 64 ? __builtin_amdgcn_readlane(g0, pos) : __builtin_amdgcn_readlane(g1, pos - 64);
    t.count = __builtin_amdgcn_readfirstlane(end - pos);
    t.first = base + pos;
    t.has = t.g >= 0 && t.g < a.n;
    return t;
  }
};

__device__ __forceinline__ bool lora_finite(float v) { return fabsf(v) < __builtin_inff(); }  // (NaN: false)

// Route of row `row` of a tile (-1: past its last).
__device__ __forceinline__ int64_t lora_route(const LoraArgs& a, const LoraTile& t, int row) {
  if (row >= t.count) return -1;
  return a.order ? (int64_t)a.order[t.first + row] : t.first + row;
}

// NJ fragments of 16 rows over the steps s0 .. s1: rank 16 u + 4 q + v of row 16 j + c.
template <typename T, bool VEC, int RT, int NJ>
__device__ __forceinline__ void lora_dot(const LoraArgs& a, const LoraTile& t, int64_t s0, int64_t s1, int lane,
                                         f4 (&acc)[NJ][RT]) {
  constexpr int V = Dense<T>::V, KS = Dense<T>::KS, UN = RT + NJ <= 4 ? 4 : 2;
  const int c = lane & 15, q = lane >> 4;
  const T *xrow[NJ], *arow[RT];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {  // rows past the tile's last: row 0's values, not stored
    const int64_t route = lora_route(a, t, 16 * j + c);
    const int64_t xr = route < 0 ? 0 : min((int64_t)((uint32_t)route / (uint32_t)a.x_div), a.x_rows - 1);
    xrow[j] = (const T*)a.x + xr * a.K;
#pragma unroll
    for (int u = 0; u < RT; ++u) acc[j][u] = f4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int u = 0; u < RT; ++u) arow[u] = (const T*)a.a + ((int64_t)t.g * a.R + min((int64_t)(16 * u + c), a.R - 1)) * a.K;
  // UN steps' loads in flight together; past the share's last step, or K's end, zeros on both sides
  for (int64_t s = s0; s < s1; s += UN) {
    uint4 fi[UN][RT], fj[UN][NJ];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int64_t k = min(s + i, s1 - 1) * KS + q * V;
      if constexpr (VEC) {
        const int64_t kk = min(k, a.K - V);
        const bool in = s + i < s1 && k < a.K;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          fj[i][j] = dense_ld16(xrow[j], kk);
          if (!in) fj[i][j] = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          fi[i][u] = dense_ld16(arow[u], kk);
          if (!in) fi[i][u] = make_uint4(0u, 0u, 0u, 0u);
        }
      } else {
        const int64_t n = s + i < s1 ? a.K : 0;
#pragma unroll
        for (int j = 0; j < NJ; ++j) fj[i][j] = dense_ld<T, VEC>(xrow[j], k, n);
#pragma unroll
        for (int u = 0; u < RT; ++u) fi[i][u] = dense_ld<T, VEC>(arow[u], k, n);
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int u = 0; u < RT; ++u) acc[j][u] = dense_mfma<T>(fi[i][u], fj[i][j], acc[j][u]);
  }
}

template <typename T, bool VEC, int RT>
__global__ __launch_bounds__(64 * LS_WAVES) void k_lora_shrink(LoraArgs a) {
  constexpr int KS = Dense<T>::KS;
  __shared__ float4 red[LS_WAVES][RT][64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t cb = blockIdx.x / a.split, slice = blockIdx.x - cb * a.split;
  const int64_t window = cb / a.heads;
  const LoraWindow w(a, window, lane);
  const int64_t steps = (a.K + KS - 1) / KS, shares = a.split * LS_WAVES, per = (steps + shares - 1) / shares;
  const int64_t s0 = min(steps, (slice * LS_WAVES + wv) * per), s1 = min(steps, s0 + per);
  const int tiles = w.tiles();
  for (int k = (int)(cb - window * a.heads); k < tiles; k += a.heads) {
    const LoraTile t = w.tile(a, k);
    if (!t.has) continue;
    auto rows = [&](auto nj_c) {
      constexpr int NJ = decltype(nj_c)::value;
      f4 acc[NJ][RT];
      lora_dot<T, VEC, RT, NJ>(a, t, s0, s1, lane, acc);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int u = 0; u < RT; ++u) red[wv][u][lane] = make_float4(acc[j][u][0], acc[j][u][1], acc[j][u][2], acc[j][u][3]);
        __syncthreads();
        const int64_t route = lora_route(a, t, 16 * j + c);
        for (int u = wv; u < RT; u += LS_WAVES) {
          float4 p[LS_WAVES];
#pragma unroll
          for (int i = 0; i < LS_WAVES; ++i) p[i] = red[i][u][lane];
          float4 f = p[0];
#pragma unroll
          for (int i = 1; i < LS_WAVES; ++i) {
            f.x += p[i].x; f.y += p[i].y; f.z += p[i].z; f.w += p[i].w;
          }
          if (route >= 0) *(float4*)(a.ws + (slice * a.routes + route) * (16 * RT) + 16 * u + 4 * q) = f;
        }
        __syncthreads();  // red is written again
      }
    };
    if (t.count <= 16) rows(std::integral_constant<int, 1>{});
    else rows(std::integral_constant<int, 2>{});
  }
}

// A wave takes 64 columns of a tile. Lane (c, q) of product u holds B row 32 (u / 2) + 8 (c / 4) + 4 (u % 2) + c % 4 of
// them, so that the lane's results over two products are 8 neighbouring columns of route c, and a row's four lanes make
// 64 bytes of each load and store. (No loop over columns: loads of a second turn would wait for the first one's stores.)
// OT: base's and out's type. VEC, WIDE: rows of B, and of base and out, hold whole 16-byte pieces at aligned addresses.
// Up to rank 32 and 16-bit outputs, 128 registers keep two blocks on a CU (4093 rows of r = 32: 52 us, 65 with one).
template <typename T, typename OT, bool VEC, bool WIDE, int RT>
__global__ __launch_bounds__(64 * LE_WAVES, sizeof(OT) == 2 && RT <= 2 ? 4 : 1) void k_lora_expand(LoraArgs a) {
  constexpr int V = Dense<T>::V, KS = Dense<T>::KS, RP = 16 * RT, NK = (RP + KS - 1) / KS;
  constexpr int TERMS = sizeof(T) == 4 ? 1 : __is_same(T, bf16s) ? 3 : 2;
  __shared__ __attribute__((aligned(16))) T ts[TERMS][LORA_ROWS][NK * KS + V];  // t's terms (the pad spreads rows over the banks)
  __shared__ float tback[LORA_ROWS];                                            // and the rows' powers of two
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t cb = blockIdx.x / a.split, nb = blockIdx.x - cb * a.split;
  const int64_t window = cb / a.heads;
  const LoraWindow w(a, window, lane);
  const int64_t n0 = (nb * LE_WAVES + wv) * 64, ncol = a.out ? a.N : 0;
  const int tiles = w.tiles();
  for (int k = (int)(cb - window * a.heads); k < tiles; k += a.heads) {
    const LoraTile t = w.tile(a, k);
    if (!t.has) {  // base as it is, zeros, or NaN
      for (int64_t i = threadIdx.x; a.t_out && nb == 0 && i < t.count * RP; i += 64 * LE_WAVES)
        a.t_out[lora_route(a, t, (int)(i / RP)) * RP + i % RP] = 0.f;
      const int64_t n = n0 + lane;
      for (int row = 0; row < t.count && n < ncol; ++row) {
        const int64_t at = lora_route(a, t, row) * a.N + n;
        ((OT*)a.out)[at] = t.g >= 0 ? from_float<OT>(__builtin_nanf("")) : a.base ? ((const OT*)a.base)[at] : from_float<OT>(0.f);
      }
      continue;
    }
    auto rows = [&](auto nj_c) {
      constexpr int NJ = decltype(nj_c)::value, OV = 16 / sizeof(OT);
      int at[NJ];  // the routes of this lane's rows (-1: none)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int64_t r = lora_route(a, t, 16 * j + c);
        at[j] = (int)r;
      }
      // B's rows and base are read before t is there
      uint4 fi[NK][4], base[NJ][2][8 / OV];
      const T* bb = (const T*)a.b + (int64_t)t.g * a.N * a.R;
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t n = min(n0 + (u >> 1) * 32 + (c >> 2) * 8 + (u & 1) * 4 + (c & 3), a.N - 1);
          const int r = i * KS + q * V;
          if constexpr (VEC) {  // past the rank: zeros, loaded from the row's first values
            fi[i][u] = dense_ld16(bb + n * a.R, r < a.R ? r : 0);
            if (r >= a.R) fi[i][u] = make_uint4(0u, 0u, 0u, 0u);
          } else {
            fi[i][u] = dense_ld<T, VEC>(bb + n * a.R, r, a.R);
          }
        }
      if (WIDE && a.base) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int h = 0; h < 8 / OV; ++h)
              base[j][p][h] = dense_ld16((const OT*)a.base + (int64_t)max(at[j], 0) * a.N, min(n0 + p * 32 + q * 8, a.N - 8) + h * OV);
      }
      const float sc = a.scales ? a.scales[t.g] : 1.f;
      for (int i = threadIdx.x; i < NJ * 16 * RP / 4; i += 64 * LE_WAVES) {
        const int row = i / (RP / 4), k4 = (i - row * (RP / 4)) * 4;
        const int64_t tr = lora_route(a, t, row);
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tr >= 0) {
          for (int64_t sl = 0; sl < a.slices; sl += 4) {  // four loads in flight, added in order
            float4 p[4];
#pragma unroll
            for (int d = 0; d < 4; ++d)
              p[d] = *(const float4*)(a.ws + (min(sl + d, a.slices - 1) * a.routes + tr) * RP + k4);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              if (sl + d >= a.slices) break;
              f.x += p[d].x; f.y += p[d].y; f.z += p[d].z; f.w += p[d].w;
            }
          }
          f.x = k4 < a.R ? f.x * sc : 0.f;
          f.y = k4 + 1 < a.R ? f.y * sc : 0.f;
          f.z = k4 + 2 < a.R ? f.z * sc : 0.f;
          f.w = k4 + 3 < a.R ? f.w * sc : 0.f;
          if (a.t_out && nb == 0) *(float4*)(a.t_out + tr * RP + k4) = f;
        }
        if constexpr (TERMS == 1) {
          *(float4*)&ts[0][row][k4] = f;
        } else {
          // a row is RP / 4 neighbouring lanes (whole waves are here): 2^e <= its largest value < 2^(e + 1), within the
          // powers whose inverse is a normal number too
          float v[4] = {f.x, f.y, f.z, f.w}, mx = 0.f;
#pragma unroll
          for (int u = 0; u < 4; ++u) mx = fmaxf(mx, lora_finite(v[u]) ? fabsf(v[u]) : 0.f);
#pragma unroll
          for (int d = 1; d < RP / 4; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
          const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -126), 126);
          const float fac = __uint_as_float((uint32_t)(127 - e) << 23);
          if (k4 == 0) tback[row] = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] *= fac;
#pragma unroll
          for (int m = 0; m < TERMS; ++m) {
            uint32_t w[2] = {0u, 0u};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const T h = from_float<T>(v[u]);
              const float left = v[u] - to_float(h);  // exact
              v[u] = lora_finite(left) ? left : 0.f;  // nothing is left of an infinity or NaN
              w[u >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, h) << (16 * (u & 1));
            }
            *(uint2*)&ts[m][row][k4] = make_uint2(w[0], w[1]);
            if (NK * KS > RP) *(uint2*)&ts[m][row][RP + k4] = make_uint2(0u, 0u);
          }
        }
      }
      __syncthreads();
      f4 acc[NJ][4];
      float back[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        back[j] = TERMS == 1 ? 1.f : tback[16 * j + c];
        uint4 fj[TERMS][NK];
#pragma unroll
        for (int m = 0; m < TERMS; ++m)
#pragma unroll
          for (int i = 0; i < NK; ++i) fj[m][i] = *(const uint4*)&ts[m][16 * j + c][i * KS + q * V];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          acc[j][u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = TERMS - 1; m >= 0; --m)
#pragma unroll
            for (int i = 0; i < NK; ++i) acc[j][u] = dense_mfma<T>(fi[i][u], fj[m][i], acc[j][u]);
        }
        if constexpr (TERMS > 1) {
          // an infinity in B is one in the output, whatever the signs of t's other terms: there the first term's sums count
          float z = 0.f;
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int v = 0; v < 4; ++v) z = fmaf(acc[j][u][v], 0.f, z);
          if (__any(!(z == 0.f))) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              f4 first{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int i = 0; i < NK; ++i) first = dense_mfma<T>(fi[i][u], fj[0][i], first);
#pragma unroll
              for (int v = 0; v < 4; ++v)
                if (!lora_finite(first[v])) acc[j][u][v] = first[v];
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int64_t n = n0 + p * 32 + q * 8;
          if (at[j] < 0 || n >= ncol) continue;
          float f[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            f[u] = acc[j][2 * p + (u >> 2)][u & 3] * back[j];
            if (a.base) {
              if constexpr (WIDE) f[u] += dense_at<OT>(base[j][p][u / OV], u % OV);
              else f[u] += n + u < a.N ? to_float(((const OT*)a.base)[at[j] * a.N + n + u]) : 0.f;
            }
          }
          dense_st<OT, 8>((OT*)a.out + at[j] * a.N + n, a.N - n, f, WIDE);
        }
      __syncthreads();  // ts is written again
    };
    if (t.count <= 16) rows(std::integral_constant<int, 1>{});
    else rows(std::integral_constant<int, 2>{});
  }
}

// Both factors transposed for the backward pass: [n][P][Q] -> [n][Q][P], 64 x 64 tiles through LDS.
struct TransposeArgs {
  const void* from[2];
  void* to[2];
  int64_t P[2], Q[2], blocks[2];
};

template <typename T>
__global__ __launch_bounds__(256) void k_lora_transpose(TransposeArgs a) {
  __shared__ T tile[64][66];
  const int m = blockIdx.x >= a.blocks[0] ? 1 : 0;
  int64_t b = blockIdx.x - (m ? a.blocks[0] : 0);
  const int64_t P = a.P[m], Q = a.Q[m], pb = (P + 63) / 64, qb = (Q + 63) / 64;
  const int64_t n = b / (pb * qb);
  b -= n * pb * qb;
  const int64_t p0 = b / qb * 64, q0 = (b - b / qb * qb) * 64;
  const T* from = (const T*)a.from[m] + n * P * Q;
  T* to = (T*)a.to[m] + n * P * Q;
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 64; i += 4)
    if (p0 + i + r < P && q0 + c < Q) tile[i + r][c] = from[(p0 + i + r) * Q + q0 + c];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 64; i += 4)
    if (q0 + i + r < Q && p0 + c < P) to[(q0 + i + r) * P + p0 + c] = tile[c][i + r];
}

// ------------------------------------------------------------------ host side

static int lora_rt(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8; }

// Blocks per window: one per position while every row may be a request of its own and the windows are few, down to about
// as many as a window of long runs has tiles (4093 rows in runs of about 100: 6 blocks 49 us, 8 54).
static int64_t lora_heads(int64_t routes) {
  const int64_t windows = (routes + 127) / 128;
  return std::min<int64_t>(std::min<int64_t>(routes, 128), windows <= 2 ? 128 : std::max<int64_t>(6, 192 / windows));
}
static int64_t lora_blocks(int64_t routes) { return (routes + 127) / 128 * lora_heads(routes); }

// Slices of K, a power of two (a wave's steps then come in whole batches): about 40 KiB of A each (one row, r = 16 of 4096:
// 4 slices 8.5 us, 1 11.1; r = 128 of 8192: 16 slices 19, 4 26), while the tiles leave CUs free (64 requests of r = 64: 4
// slices 17.3 us, 8 18.8; 4093 rows of r = 32: 4 slices 49, 16 97). Each wave takes at least a step of 64 bytes of a row.
// Up to 256 rows count as requests of their own, which they need not be: of r = 64, 256 rows of one adapter take 35 us in
// their one slice and 21 in four (257 rows: 20), 256 rows of 96 adapters in turn 44 and 51; 512 such rows 107, in one 94.
static int64_t lora_slices(int64_t routes, int64_t R, int64_t K, int size) {
  const int64_t steps = (K * size + 63) / 64, want = R * K * size / (40 << 10) + 1;
  const int64_t room = routes <= 256 ? 256 / routes : 20000 / routes;
  const int64_t most = std::min<int64_t>({want, room, 16, steps / LS_WAVES});
  int64_t n = 1;
  while (2 * n <= most) n *= 2;
  return n;
}

template <typename T, typename OT, bool VECR, bool WIDE>
static void lora_launch(LoraArgs a, bool veck, hipStream_t s) {
  const int64_t blocks = lora_blocks(a.routes), groups = (a.N + 64 * LE_WAVES - 1) / (64 * LE_WAVES);
  auto go = [&](auto c) {
    constexpr int RT = decltype(c)::value;
    a.split = a.slices;
    const dim3 shrink((unsigned)(blocks * a.split));
    if (veck) hipLaunchKernelGGL((k_lora_shrink<T, true, RT>), shrink, dim3(64 * LS_WAVES), 0, s, a);
    else hipLaunchKernelGGL((k_lora_shrink<T, false, RT>), shrink, dim3(64 * LS_WAVES), 0, s, a);
    a.split = a.out ? groups : 1;
    hipLaunchKernelGGL((k_lora_expand<T, OT, VECR, WIDE, RT>), dim3((unsigned)(blocks * a.split)), dim3(64 * LE_WAVES), 0, s, a);
  };
  const int rt = lora_rt(a.R);
  if (rt == 1) go(std::integral_constant<int, 1>{});
  else if (rt == 2) go(std::integral_constant<int, 2>{});
  else if (rt == 4) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 8>{});
}

template <typename T>
static void lora_pick(const LoraArgs& a, bool out_float, bool vk, bool vr, bool wide, hipStream_t s) {
  auto go = [&](auto ot) {
    typedef decltype(ot) OT;
    if (vr && wide) lora_launch<T, OT, true, true>(a, vk, s);
    else if (vr) lora_launch<T, OT, true, false>(a, vk, s);
    else if (wide) lora_launch<T, OT, false, true>(a, vk, s);
    else lora_launch<T, OT, false, false>(a, vk, s);
  };
  if (out_float) go(float{});
  else go(T{});
}

}  // namespace keep

namespace keep {

// A plan's arrays in a workspace.
struct LoraPlan {
  int32_t *order, *inverse, *counts, *offsets, *tiles;
  int64_t room;
  static int64_t bytes(int64_t routes, int64_t n) {
    return (4 * (2 * routes + 2 * n + 3 * ((routes + 15) / 16 + n) + 1) + 255) / 256 * 256;
  }
  int make(void* ws, const int32_t* idx, int64_t routes, int64_t n, void* stream) {
    order = (int32_t*)ws;
    inverse = order + routes;
    counts = inverse + routes;
    offsets = counts + n;
    tiles = offsets + n;
    room = (routes + 15) / 16 + n;
    return keep_route_plan(idx, routes, n, 16, order, inverse, counts, offsets, tiles, tiles + room, tiles + 2 * room,
                           room, tiles + 3 * room, stream);
  }
};

static int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }

// Whether every size in bytes that these sizes make fits 63 bits with room (dims_ok and the rank's range are checked first).
static bool lora_sizes_ok(int64_t routes, int64_t n, int64_t rank, int64_t K, int64_t N) {
  const int64_t most = int64_t(1) << 46, width = std::max<int64_t>({K, N, 1});
  return n <= most / (rank * width) && routes <= most / width;
}

static int64_t lora_partials(int dtype, int64_t routes, int64_t rank, int64_t K) {
  return round256(lora_slices(routes, rank, K, dtype_size(dtype)) * routes * 16 * lora_rt(rank) * 4);
}

static void lora_run(LoraArgs p, int dtype, int out_dtype, hipStream_t s) {
  const int64_t size = dtype_size(dtype), v = 16 / size;
  p.heads = (int)lora_heads(p.routes);
  p.slices = lora_slices(p.routes, p.R, p.K, (int)size);
  const bool vk = p.K % v == 0 && aligned(p.x, 16) && aligned(p.a, 16);
  const bool vr = p.R % v == 0 && aligned(p.b, 16);
  const bool w = p.N % 8 == 0 && aligned(p.base, 16) && aligned(p.out, 16);
  const bool f = out_dtype == KEEP_F32;
  if (dtype == KEEP_F32) lora_pick<float>(p, f, vk, vr, w, s);
  else if (dtype == KEEP_F16) lora_pick<_Float16>(p, f, vk, vr, w, s);
  else lora_pick<bf16s>(p, f, vk, vr, w, s);
}

static int lora_check(int dtype, int64_t x_rows, int64_t routes, int64_t x_div, int64_t adapters, int64_t rank,
                      int64_t K, int64_t N, int grouped) {
  KEEP_REQUIRE_DIMS(x_rows, routes, x_div, adapters, rank, K, N);
  KEEP_REQUIRE(dtype_ok(dtype), "bad dtype enum");
  KEEP_REQUIRE(rank >= 1 && rank <= 128, "rank must be in 1..128");
  KEEP_REQUIRE(adapters > 0 && K > 0 && N > 0 && x_div > 0, "adapters, K, N and x_div must be positive");
  KEEP_REQUIRE(lora_sizes_ok(routes, adapters, rank, K, N), "too many values");
  KEEP_REQUIRE(!grouped || adapters <= 1024, "a plan holds at most 1024 adapters");
  KEEP_REQUIRE(routes == 0 || (routes - 1) / x_div < x_rows, "x holds %lld rows, %lld routes need more",
               (long long)x_rows, (long long)routes);
  KEEP_REQUIRE(routes == 0 || lora_blocks(routes) <= LORA_BLOCKS / std::max<int64_t>(16, (std::max(N, K) + 511) / 512),
               "too many outputs");
  return KEEP_OK;
}

}  // namespace keep

using namespace keep;

extern "C" int64_t keep_lora_rank_stride(int64_t rank) { return rank >= 1 && rank <= 128 ? 16 * lora_rt(rank) : 0; }

extern "C" int64_t keep_lora_workspace_bytes(int dtype, int64_t routes, int64_t adapters, int64_t rank, int64_t K,
                                             int grouped) {
  if (!dtype_ok(dtype) || !dims_ok({routes, adapters, rank, K}) || rank < 1 || rank > 128 || routes == 0 ||
      !lora_sizes_ok(routes, adapters, rank, K, 1))
    return 0;
  return lora_partials(dtype, routes, rank, K) + (grouped ? LoraPlan::bytes(routes, adapters) : 0);
}

extern "C" int keep_lora(const void* x, int dtype, int64_t x_rows, const void* a, const void* b, const float* scales,
                         const int32_t* idx, int64_t routes, int64_t x_div, int64_t adapters, int64_t rank, int64_t K,
                         int64_t N, const void* base, int base_dtype, float* t_out, int grouped, void* workspace,
                         int64_t workspace_bytes, void* out, int out_dtype, void* stream) {
  if (int rc = lora_check(dtype, x_rows, routes, x_div, adapters, rank, K, N, grouped)) return rc;
  KEEP_REQUIRE((out_dtype == dtype || out_dtype == KEEP_F32) && (!base || base_dtype == out_dtype),
               "out must have x's dtype or float32, and base out's");
  if (routes == 0) return KEEP_OK;
  KEEP_REQUIRE(x && a && b && idx && out && workspace && x_rows > 0, "null pointer argument");
  const int64_t size = dtype_size(dtype);
  KEEP_REQUIRE(aligned(x, size) && aligned(a, size) && aligned(b, size) && aligned(out, dtype_size(out_dtype)) &&
                   aligned(base, dtype_size(out_dtype)) && aligned(workspace, 16) && aligned(t_out, 16),
               "misaligned pointer");
  const int64_t need = keep_lora_workspace_bytes(dtype, routes, adapters, rank, K, grouped);
  KEEP_REQUIRE(workspace_bytes >= need, "workspace needs %lld bytes, has %lld", (long long)need,
               (long long)workspace_bytes);
  LoraArgs p{};
  p.x = x; p.x_rows = x_rows; p.a = a; p.b = b; p.scales = scales; p.idx = idx;
  p.routes = routes; p.x_div = x_div; p.n = adapters; p.R = rank; p.K = K; p.N = N;
  p.ws = (float*)workspace; p.t_out = t_out; p.base = base; p.out = out;
  if (grouped) {
    LoraPlan plan;
    if (int rc = plan.make((char*)workspace + lora_partials(dtype, routes, rank, K), idx, routes, adapters, stream)) return rc;
    p.order = plan.order;
  }
  lora_run(p, dtype, out_dtype, (hipStream_t)stream);
  return launch_status("keep_lora");
}

// The backward workspace: both factors transposed, partial sums, dt, the routes' dx in float32 (several routes a row), the
// plan.
namespace keep {
struct LoraBackward {
  int64_t bt, at, partials, dt, rows, plan, total;
  LoraBackward(int dtype, int64_t routes, int64_t x_div, int64_t n, int64_t rank, int64_t K, int64_t N, bool dx, bool planned) {
    const int64_t size = dtype_size(dtype);
    bt = 0;
    at = bt + round256(n * rank * N * size);
    partials = at + round256(n * rank * K * size);
    dt = partials + lora_partials(dtype, routes, rank, N);
    rows = dt + round256(routes * 16 * lora_rt(rank) * 4);
    plan = rows + (dx && x_div > 1 ? round256(routes * K * 4) : 0);
    total = plan + (planned ? LoraPlan::bytes(routes, n) : 0);
  }
};
}  // namespace keep

extern "C" int64_t keep_lora_backward_workspace_bytes(int dtype, int64_t routes, int64_t x_div, int64_t adapters,
                                                      int64_t rank, int64_t K, int64_t N, int dx, int planned) {
  if (!dtype_ok(dtype) || !dims_ok({routes, x_div, adapters, rank, K, N}) || rank < 1 || rank > 128 ||
      routes == 0 || !lora_sizes_ok(routes, adapters, rank, K, N))
    return 0;
  return LoraBackward(dtype, routes, x_div, adapters, rank, K, N, dx, planned).total;
}

extern "C" int keep_lora_backward(const void* x, int dtype, int64_t x_rows, const void* a, const void* b,
                                  const float* scales, const int32_t* idx, int64_t routes, int64_t x_div,
                                  int64_t adapters, int64_t rank, int64_t K, int64_t N, const float* t, const void* dy,
                                  void* dx, void* da, void* db, int planned, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (int rc = lora_check(dtype, x_rows, routes, x_div, adapters, rank, K, N, planned)) return rc;
  KEEP_REQUIRE(planned || (!da && !db), "gradients of the factors need a plan");
  KEEP_REQUIRE(x_rows * x_div == routes, "x holds %lld rows of %lld routes, not %lld", (long long)x_rows,
               (long long)x_div, (long long)routes);
  if (routes == 0) return KEEP_OK;
  KEEP_REQUIRE(x && a && b && idx && dy && workspace && (t || !db), "null pointer argument");
  const int64_t size = dtype_size(dtype);
  KEEP_REQUIRE(aligned(x, size) && aligned(a, size) && aligned(b, size) && aligned(dy, size) && aligned(dx, size) &&
                   aligned(da, size) && aligned(db, size) && aligned(t, 16) && aligned(workspace, 256),
               "misaligned pointer");
  const LoraBackward w(dtype, routes, x_div, adapters, rank, K, N, dx != nullptr, planned);
  KEEP_REQUIRE(workspace_bytes >= w.total, "workspace needs %lld bytes, has %lld", (long long)w.total,
               (long long)workspace_bytes);
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  LoraPlan plan{};
  if (planned)
    if (int rc = plan.make(ws + w.plan, idx, routes, adapters, stream)) return rc;
  float* dt = (float*)(ws + w.dt);
  const int64_t stride = 16 * lora_rt(rank);
  if (dx || da) {  // dt = s dy B, dx = dt A: the forward's two products on the transposed factors
    TransposeArgs tr{{b, a}, {ws + w.bt, ws + w.at}, {N, rank}, {rank, K}, {0, 0}};
    for (int m = 0; m < 2; ++m) tr.blocks[m] = adapters * ((tr.P[m] + 63) / 64) * ((tr.Q[m] + 63) / 64);
    if (!dx) tr.blocks[1] = 0;
    KEEP_REQUIRE(tr.blocks[0] + tr.blocks[1] <= 2 * LORA_BLOCKS, "too many factors");
    const dim3 grid((unsigned)(tr.blocks[0] + tr.blocks[1]));
    if (size == 4) hipLaunchKernelGGL(k_lora_transpose<uint32_t>, grid, dim3(256), 0, s, tr);
    else hipLaunchKernelGGL(k_lora_transpose<uint16_t>, grid, dim3(256), 0, s, tr);
    LoraArgs p{};
    p.x = dy; p.x_rows = routes; p.a = ws + w.bt; p.b = ws + w.at; p.scales = scales; p.idx = idx;
    p.order = planned && x_div > 1 ? plan.order : nullptr;
    p.routes = routes; p.x_div = 1; p.n = adapters; p.R = rank; p.K = N; p.N = K;
    p.ws = (float*)(ws + w.partials); p.t_out = dt;
    const bool apart = dx && x_div > 1;  // a row's routes are added in float32 and rounded once
    p.out = apart ? ws + w.rows : dx;
    lora_run(p, dtype, apart ? KEEP_F32 : dtype, s);
    if (apart)
      if (int rc = keep_route_combine_rows(ws + w.rows, KEEP_F32, nullptr, x_rows, x_div, K, dx, dtype, stream)) return rc;
  }
  OuterArgs o{};
  o.order = plan.order; o.offsets = plan.offsets; o.counts = plan.counts; o.routes = routes;
  if (da) {
    o.i = x; o.i_rows = x_rows; o.i_div = x_div; o.i_dim = K;
    o.j = dt; o.j_ld = stride; o.j_dim = rank;
    o.out = da; o.j_inner = 0;
    if (int rc = rows_outer(o, dtype, true, adapters, s, "keep_lora_backward")) return rc;
  }
  if (db) {
    o.i = dy; o.i_rows = routes; o.i_div = 1; o.i_dim = N;
    o.j = t; o.j_ld = stride; o.j_dim = rank;
    o.out = db; o.j_inner = 1;
    if (int rc = rows_outer(o, dtype, true, adapters, s, "keep_lora_backward")) return rc;
  }
  return launch_status("keep_lora_backward");
}
