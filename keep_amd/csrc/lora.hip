// Low-rank adapters of many requests at once, added to a projection's rows:
//
//   out[r] = base[r] + s[a] (x[row_r] A[a]^T) B[a]^T,   a = idx[r]   (A [n][R][K], B [n][N][R])
//
// a < 0: no adapter (out = base, or zeros); a >= n: a NaN row. Two launches:
//
// k_lora_shrink: t = x A^T. A block takes a tile of up to 16 routes of one
// adapter and a slice of K; its four waves split the slice, are added in order
// through LDS, and the slice's partial t goes to the workspace in fp32.
// k_lora_expand: adds the slices in order, times s, and streams B's rows of the
// block's columns: out = base + t B^T.
//
// Tiles need no plan: rows of one adapter are found with two ballots over a
// window of 128 positions (dense_window_tile), since rows of a request lie
// together in a batch, or, of many requests, are few.
//
// t enters the second product in the rows' 16-bit type (one rounding, half a
// step of that type relative to the row's largest t), each row times a power of
// two that brings its largest value to [1, 2): fp16 then holds every row
// whatever its range. float rows stay float throughout.
#include <algorithm>

#include "dense_dev.h"
#include "dense_outer.h"

namespace keep {

constexpr int LR_WAVES = 4;

struct LoraArgs {
  const void* x;
  int64_t x_rows;
  const void *a, *b;
  const float* scales;  // null: ones
  const int32_t *idx, *order;
  int64_t routes, x_div;
  int64_t n, R, K, N;
  int cand;       // candidate positions per block
  int64_t split;  // shrink: slices of K; expand: blocks along N
  int64_t slices;
  float* ws;  // [slices][routes][16 RT]
  float* t_out;
  const void* base;
  int bdt;
  void* out;
  int odt;
  int wide;  // rows of base and out hold whole 16-byte pieces at aligned addresses
};

__device__ __forceinline__ int lora_group(const LoraArgs& a, int64_t p) {
  const int g = a.idx[a.order ? (int64_t)a.order[p] : p];
  return g < 0 ? -1 : g >= a.n ? (int)a.n : g;
}

template <typename T, bool VEC, int RT>
__global__ __launch_bounds__(64 * LR_WAVES) void k_lora_shrink(LoraArgs a) {
  constexpr int V = Dense<T>::V, KS = Dense<T>::KS, UN = RT <= 2 ? 4 : RT == 4 ? 2 : 1;
  __shared__ float4 red[LR_WAVES][RT][64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t cb = blockIdx.x / a.split, slice = blockIdx.x - cb * a.split;
  const int64_t steps = (a.K + KS - 1) / KS, shares = a.split * LR_WAVES, per = (steps + shares - 1) / shares;
  const int64_t s0 = min(steps, (slice * LR_WAVES + wv) * per), s1 = min(steps, s0 + per);
  const int64_t whole = VEC ? min(s1, a.K / KS) : s0;
  for (int cc = 0; cc < a.cand; ++cc) {
    const int64_t pos = cb * a.cand + cc;
    if (pos >= a.routes) break;
    const int g = lora_group(a, pos);
    if (g < 0 || g >= a.n) continue;
    const DenseTile d = dense_window_tile([&](int64_t p) { return lora_group(a, p); }, pos, a.routes, lane);
    if (d.count == 0) continue;
    const int64_t route = d.mine < 0 ? -1 : a.order ? (int64_t)a.order[d.mine] : d.mine;
    const int64_t xr = route < 0 ? 0 : min(route / a.x_div, a.x_rows - 1);
    const T* xrow = (const T*)a.x + xr * a.K;  // lanes without a route: row 0's, not stored
    const T* arow[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) arow[u] = (const T*)a.a + ((int64_t)g * a.R + min((int64_t)(16 * u + c), a.R - 1)) * a.K;
    f4 acc[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) acc[u] = f4{0.f, 0.f, 0.f, 0.f};
    int64_t s = s0;
    for (; s + UN <= whole; s += UN) {
      uint4 fi[UN][RT], fj[UN];
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int64_t k = (s + i) * KS + q * V;
        fj[i] = dense_ld<T, VEC>(xrow, k, INT64_MAX);
#pragma unroll
        for (int u = 0; u < RT; ++u) fi[i][u] = dense_ld<T, VEC>(arow[u], k, INT64_MAX);
      }
#pragma unroll
      for (int i = 0; i < UN; ++i)
#pragma unroll
        for (int u = 0; u < RT; ++u) acc[u] = dense_mfma<T>(fi[i][u], fj[i], acc[u]);
    }
    for (; s < s1; ++s) {
      const int64_t k = s * KS + q * V;
      const uint4 fj = dense_ld<T, VEC>(xrow, k, a.K);
#pragma unroll
      for (int u = 0; u < RT; ++u) acc[u] = dense_mfma<T>(dense_ld<T, VEC>(arow[u], k, a.K), fj, acc[u]);
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) red[wv][u][lane] = make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
    __syncthreads();
    for (int u = wv; u < RT; u += LR_WAVES) {
      float4 f = red[0][u][lane];
#pragma unroll
      for (int w = 1; w < LR_WAVES; ++w) {
        const float4 p = red[w][u][lane];
        f.x += p.x; f.y += p.y; f.z += p.z; f.w += p.w;
      }
      if (route >= 0) *(float4*)(a.ws + (slice * a.routes + route) * (16 * RT) + 16 * u + 4 * q) = f;
    }
    __syncthreads();  // red is written again
  }
}

__device__ __forceinline__ float lora_ld(const void* p, int dt, int64_t i) {
  if (dt == KEEP_F32) return ((const float*)p)[i];
  if (dt == KEEP_BF16) return to_float(((const bf16s*)p)[i]);
  return to_float(((const _Float16*)p)[i]);
}

// A block's four waves take groups of 64 columns in turn. Lane (c, q) of product u holds B row 16 (c / 4) + 4 u + c % 4
// of the group, so that the lane's results over the four products are 16 neighbouring columns of route c.
template <typename T, bool VEC, int RT>
__global__ __launch_bounds__(64 * LR_WAVES) void k_lora_expand(LoraArgs a) {
  constexpr int V = Dense<T>::V, KS = Dense<T>::KS, RP = 16 * RT, NK = (RP + KS - 1) / KS;
  __shared__ float ts[16][NK * KS + 4];
  __shared__ float inv[16];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t cb = blockIdx.x / a.split, nb = blockIdx.x - cb * a.split;
  for (int cc = 0; cc < a.cand; ++cc) {
    const int64_t pos = cb * a.cand + cc;
    if (pos >= a.routes) break;
    const DenseTile d = dense_window_tile([&](int64_t p) { return lora_group(a, p); }, pos, a.routes, lane);
    if (d.count == 0) continue;
    const int g = lora_group(a, pos);
    const bool has = g >= 0 && g < a.n;
    const int64_t route = d.mine < 0 ? -1 : a.order ? (int64_t)a.order[d.mine] : d.mine;
    uint4 fj[NK];
    if (has) {
      const float sc = a.scales ? a.scales[g] : 1.f;
      // 16 threads per row: thread k of row tid / 16 adds the slices of ranks k, k + 16, ...
      const int row = threadIdx.x >> 4, k0 = threadIdx.x & 15;
      const int64_t tr = __shfl(route, row, 64);  // lane row holds route row
      float mx = 0.f;
#pragma unroll
      for (int u = 0; u < NK * KS / 16; ++u) {
        const int k = 16 * u + k0;
        float v = 0.f;
        if (tr >= 0 && k < a.R) {
          for (int64_t s = 0; s < a.slices; ++s) v += a.ws[(s * a.routes + tr) * RP + k];
          v *= sc;
        }
        if (a.t_out && nb == 0 && tr >= 0 && k < RP) a.t_out[tr * RP + k] = v;
        ts[row][k] = v;
        mx = fmaxf(mx, fabsf(v));
      }
#pragma unroll
      for (int m = 8; m >= 1; m >>= 1) mx = fmaxf(mx, __shfl_xor(mx, m, 64));
      // 2^e <= mx: the factor 2^-e (1 for rows of zeros, subnormals, infinities; NaN does not reach mx)
      const int e = (int)(__float_as_uint(mx) >> 23) - 127;
      const bool use = sizeof(T) == 2 && e > -127 && e < 127;
      if (k0 == 0) inv[row] = use ? __uint_as_float((uint32_t)(127 + e) << 23) : 1.f;
      const float fac = use ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.f;
#pragma unroll
      for (int u = 0; u < NK * KS / 16; ++u) ts[row][16 * u + k0] *= fac;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const float* p = &ts[c][i * KS + q * V];
        if constexpr (sizeof(T) == 4) {
          fj[i] = make_uint4(__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3]));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int h = 0; h < 4; ++h)
            w[h] = (uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(p[2 * h])) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(p[2 * h + 1])) << 16);
          fj[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    } else if (a.t_out && nb == 0 && d.mine >= 0) {
      for (int k = wv * 4 + q; k < RP; k += 16) a.t_out[route * RP + k] = 0.f;
    }
    const float back = has ? inv[c] : 0.f;
    const int64_t groups = (a.N + 63) / 64;
    for (int64_t gi = nb * LR_WAVES + wv; gi < groups; gi += a.split * LR_WAVES) {
      const int64_t n0 = gi * 64;
      f4 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = f4{0.f, 0.f, 0.f, 0.f};
      if (has) {
        const T* bb = (const T*)a.b + (int64_t)g * a.N * a.R;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          uint4 fi[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int64_t n = min(n0 + (c >> 2) * 16 + u * 4 + (c & 3), a.N - 1);
            fi[u] = dense_ld<T, VEC>(bb + n * a.R, i * KS + q * V, a.R);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[u] = dense_mfma<T>(fi[u], fj[i], acc[u]);
        }
      }
      const int64_t n = n0 + q * 16;
      if (route < 0 || n >= a.N) continue;
      const int64_t at = route * a.N + n, left = a.N - n;
      float f[16];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) f[4 * u + v] = has ? acc[u][v] * back : g >= 0 ? __builtin_nanf("") : 0.f;
      const bool whole = left >= 16 && a.wide;
      if (a.base) {
        if (whole && a.bdt != KEEP_F32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 w = *(const uint4*)((const uint16_t*)a.base + at + 8 * h);
#pragma unroll
            for (int u = 0; u < 8; ++u)
              f[8 * h + u] += a.bdt == KEEP_BF16 ? dense_at<bf16s>(w, u) : dense_at<_Float16>(w, u);
          }
        } else {
#pragma unroll
          for (int u = 0; u < 16; ++u)
            if (u < left) f[u] += lora_ld(a.base, a.bdt, at + u);
        }
      }
      if (a.odt == KEEP_F32) dense_st<float, 16>((float*)a.out + at, left, f, whole);
      else if (a.odt == KEEP_BF16) dense_st<bf16s, 16>((bf16s*)a.out + at, left, f, whole);
      else dense_st<_Float16, 16>((_Float16*)a.out + at, left, f, whole);
    }
    __syncthreads();  // ts and inv are written again
  }
}

// ------------------------------------------------------------------ host side

static int lora_rt(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8; }

// Positions per block: one while every position may be an adapter of its own, else 16 (about one tile's).
static int lora_cand(int64_t routes) { return routes <= 256 ? 1 : 16; }

static int64_t lora_slices(int64_t routes, int64_t R, int64_t K, int size) {
  const int64_t steps = (K * size + 63) / 64;                 // of 64 bytes of a row
  const int64_t tiles = (routes + 15) / 16;
  const int64_t want = std::max<int64_t>(1, 1024 / tiles);    // about four blocks per CU
  return std::max<int64_t>(1, std::min<int64_t>({want, 16, (steps + 15) / 16}));
}

template <typename T, bool VECK, bool VECR>
static void lora_launch(LoraArgs a, int64_t nsplit, hipStream_t s) {
  const int64_t cbs = (a.routes + a.cand - 1) / a.cand;
  const int rt = lora_rt(a.R);
  auto go = [&](auto c) {
    constexpr int RT = decltype(c)::value;
    a.split = a.slices;
    hipLaunchKernelGGL((k_lora_shrink<T, VECK, RT>), dim3((unsigned)(cbs * a.slices)), dim3(64 * LR_WAVES), 0, s, a);
    a.split = nsplit;
    hipLaunchKernelGGL((k_lora_expand<T, VECR, RT>), dim3((unsigned)(cbs * nsplit)), dim3(64 * LR_WAVES), 0, s, a);
  };
  if (rt == 1) go(std::integral_constant<int, 1>{});
  else if (rt == 2) go(std::integral_constant<int, 2>{});
  else if (rt == 4) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 8>{});
}

template <typename T>
static void lora_pick(const LoraArgs& a, int64_t nsplit, bool vk, bool vr, hipStream_t s) {
  if (vk && vr) lora_launch<T, true, true>(a, nsplit, s);
  else if (vk) lora_launch<T, true, false>(a, nsplit, s);
  else if (vr) lora_launch<T, false, true>(a, nsplit, s);
  else lora_launch<T, false, false>(a, nsplit, s);
}

}  // namespace keep

using namespace keep;

extern "C" int64_t keep_lora_rank_stride(int64_t rank) { return rank >= 1 && rank <= 128 ? 16 * lora_rt(rank) : 0; }

extern "C" int64_t keep_lora_workspace_bytes(int dtype, int64_t routes, int64_t rank, int64_t K) {
  if (!dtype_ok(dtype) || !dims_ok({routes, rank, K}) || rank < 1 || rank > 128) return 0;
  return lora_slices(routes, rank, K, dtype_size(dtype)) * routes * 16 * lora_rt(rank) * 4;
}

extern "C" int keep_lora(const void* x, int dtype, int64_t x_rows, const void* a, const void* b, const float* scales,
                         const int32_t* idx, const int32_t* order, int64_t routes, int64_t x_div, int64_t adapters,
                         int64_t rank, int64_t K, int64_t N, const void* base, int base_dtype, float* t_out,
                         void* workspace, int64_t workspace_bytes, void* out, int out_dtype, void* stream) {
  KEEP_REQUIRE_DIMS(x_rows, routes, x_div, adapters, rank, K, N);
  KEEP_REQUIRE(dtype_ok(dtype) && dtype_ok(out_dtype) && (!base || dtype_ok(base_dtype)), "bad dtype enum");
  KEEP_REQUIRE(rank >= 1 && rank <= 128, "rank must be in 1..128");
  KEEP_REQUIRE(adapters > 0 && K > 0 && N > 0 && x_div > 0, "adapters, K, N and x_div must be positive");
  if (routes == 0) return KEEP_OK;
  KEEP_REQUIRE(x && a && b && idx && out && workspace && x_rows > 0, "null pointer argument");
  KEEP_REQUIRE((routes - 1) / x_div < x_rows, "x holds %lld rows, %lld routes need more", (long long)x_rows,
               (long long)routes);
  const int64_t size = dtype_size(dtype);
  KEEP_REQUIRE(aligned(x, size) && aligned(a, size) && aligned(b, size) && aligned(out, dtype_size(out_dtype)) &&
                   aligned(workspace, 16) && aligned(t_out, 4),
               "misaligned pointer");
  const int64_t need = keep_lora_workspace_bytes(dtype, routes, rank, K);
  KEEP_REQUIRE(workspace_bytes >= need, "workspace needs %lld bytes, has %lld", (long long)need,
               (long long)workspace_bytes);
  LoraArgs p{};
  p.x = x; p.x_rows = x_rows; p.a = a; p.b = b; p.scales = scales; p.idx = idx; p.order = order;
  p.routes = routes; p.x_div = x_div; p.n = adapters; p.R = rank; p.K = K; p.N = N;
  p.cand = lora_cand(routes);
  p.slices = lora_slices(routes, rank, K, (int)size);
  p.ws = (float*)workspace; p.t_out = t_out;
  p.base = base; p.bdt = base ? base_dtype : KEEP_F32;
  p.out = out; p.odt = out_dtype;
  const int64_t cbs = (routes + p.cand - 1) / p.cand, groups = (N + 255) / 256;  // 256 columns a block and turn
  const int64_t nsplit = std::max<int64_t>(1, std::min<int64_t>(groups, 2048 / std::max<int64_t>(1, (routes + 15) / 16)));
  KEEP_REQUIRE(cbs <= 0x7fffffffLL / std::max(nsplit, p.slices), "too many routes");
  const int64_t v = 16 / size;
  const bool vk = K % v == 0 && aligned(x, 16) && aligned(a, 16);
  const bool vr = rank % v == 0 && aligned(b, 16);
  p.wide = N % 8 == 0 && aligned(base, 16) && aligned(out, 16);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KEEP_F32) lora_pick<float>(p, nsplit, vk, vr, s);
  else if (dtype == KEEP_F16) lora_pick<_Float16>(p, nsplit, vk, vr, s);
  else lora_pick<bf16s>(p, nsplit, vk, vr, s);
  return launch_status("keep_lora");
}

extern "C" int keep_lora_grad(const void* rows, int dtype, int64_t n_rows, int64_t x_div, int64_t dim, const float* t,
                              int64_t t_stride, int64_t rank, int rank_inner, int64_t routes, int64_t adapters,
                              const int32_t* order, const int32_t* offsets, const int32_t* counts, void* out,
                              void* stream) {
  KEEP_REQUIRE_DIMS(n_rows, x_div, dim, t_stride, rank, routes, adapters);
  KEEP_REQUIRE(dtype_ok(dtype), "bad dtype enum");
  KEEP_REQUIRE(rank >= 1 && rank <= 128 && t_stride >= rank, "rank must be in 1..128 and t_stride at least it");
  KEEP_REQUIRE(adapters > 0 && adapters <= 65535 && dim > 0 && x_div > 0, "adapters, dim and x_div must be positive");
  KEEP_REQUIRE(offsets && counts && out && (routes == 0 || (rows && t && order && n_rows > 0)), "null pointer argument");
  KEEP_REQUIRE(aligned(rows, dtype_size(dtype)) && aligned(out, dtype_size(dtype)) && aligned(t, 4),
               "misaligned pointer");
  OuterArgs a{};
  a.i = rows; a.i_rows = n_rows; a.i_div = x_div; a.i_dim = dim;
  a.j = t; a.j_ld = t_stride; a.j_dim = rank;
  a.order = order; a.offsets = offsets; a.counts = counts; a.routes = routes;
  a.out = out; a.j_inner = rank_inner;
  return rows_outer(a, dtype, true, adapters, (hipStream_t)stream, "keep_lora_grad");
}
