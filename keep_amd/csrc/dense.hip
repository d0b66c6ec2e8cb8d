// Routed products with dense expert weights, straight from global memory: the
// form for few routes (decode, verify windows), for any alignment and for float
// rows. Large 16-bit products run in dense_gemm.hip.
//
//   forward     out[r] = W[e_r] x[row_r]           W [E][N][K]   (k_gather_few)
//   transposed  out[r] = W[e_r]^T x[row_r]         W [E][K][N]   (k_gather_trans)
//   gradient    dW[e][n][k] = sum_{r: e_r = e} dy[r][n] x[row_r][k]   (k_rows_outer)
//
// Sums are held in fp32 on the matrix cores. k_gather_few multiplies 16-bit
// rows as they are; the other two take one value of a row per lane and product
// (16x16x4, in float), since their contraction runs across rows: a lane's
// 16-byte load then serves as many products as it has values, with no
// transposition. A row's result depends on its own operands only, in a fixed
// order, whatever routes share its tile.
#include <algorithm>

#include "dense_dev.h"
#include "dense_gemm.h"
#include "dense_outer.h"

namespace keep {

struct GatherArgs {
  const void* x;
  int64_t x_rows;
  const void* w;
  const int32_t *rhs, *lhs;
  int64_t routes, x_div;
  int64_t E, N, K;
  const int32_t *order, *te, *to, *tc;  // tiles of a route plan (null: grouped here, in windows)
  int64_t tiles;
  void* out;
  int odt;
};

// A block's tile: strips of outputs along x, tiles along y and z (a launch holds 2^32 threads along x, 65535 blocks along
// y and z).
constexpr int64_t GATHER_Y = 32768;
__device__ __forceinline__ int64_t gather_block() { return (int64_t)blockIdx.z * GATHER_Y + blockIdx.y; }

// The routes of a block's tile: lane c's route (-1: none), its x row (0 where there is none), whether its row is valid.
struct GatherTile {
  int count;
  int64_t e, route, xr;
  bool ok;
};

__device__ __forceinline__ GatherTile gather_tile(const GatherArgs& a, int64_t tile, int lane) {
  GatherTile t{0, -1, -1, 0, false};
  if (tile >= a.tiles) return t;
  const int c = lane & 15;
  if (a.te) {
    t.count = min(16, a.tc[tile]);
    if (t.count == 0) return t;
    t.e = a.te[tile];
    const int64_t p = (int64_t)a.to[tile] + c;
    if (c < t.count && p >= 0 && p < a.routes) t.route = a.order[p];
  } else {
    const DenseWindow w([&](int64_t p) { return a.rhs[p]; }, tile, a.routes, lane);
    const DenseTile d = w.tile(tile, lane);
    t.count = d.count;
    if (t.count == 0) return t;
    t.e = d.group;
    t.route = d.mine;
  }
  if (t.route >= a.routes) t.route = -1;
  if (t.e < 0 || t.e >= a.E) t.e = -1;
  if (t.route >= 0) {
    const int64_t xr = a.lhs ? (int64_t)a.lhs[t.route] : t.route / a.x_div;
    t.ok = t.e >= 0 && xr >= 0 && xr < a.x_rows;
    t.xr = t.ok ? xr : 0;
  }
  return t;
}

__device__ __forceinline__ void gather_store(const GatherArgs& a, int64_t at, int64_t left, const float (&f)[4],
                                             bool vec) {
  if (a.odt == KEEP_F32) dense_st<float, 4>((float*)a.out + at, left, f, vec);
  else if (a.odt == KEEP_BF16) dense_st<bf16s, 4>((bf16s*)a.out + at, left, f, vec);
  else dense_st<_Float16, 4>((_Float16*)a.out + at, left, f, vec);
}

// Eight waves share a tile's rows against 16 rows of W: wave s takes the s-th share of K and the shares are added in order
// through LDS. Lane (c, q) holds W row n0 + c, so that its results are outputs n0 + 4 q + v of route c.
//
// Bound by the bytes of W of the experts that are hit (a byte of W serves at most 16 routes, far below the matrix cores'
// rate): one token of 6 experts, fp16 4096 -> 2048, 101 MB in 18.7 us, 5.4 TB/s; eight tokens, bf16, 743 MB of
// weights in 124 us, 6.0 TB/s. Eight loads per wave are in flight; the fine strips (16 outputs) are what
// fills 256 CUs with a token's few tiles.
constexpr int GF_WAVES = 8;

template <typename T, bool VEC>
__global__ __launch_bounds__(64 * GF_WAVES) void k_gather_few(GatherArgs a) {
  constexpr int V = Dense<T>::V, KS = Dense<T>::KS, UN = 8;
  __shared__ float4 red[GF_WAVES][64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const GatherTile t = gather_tile(a, gather_block(), lane);
  if (t.count == 0) return;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  f4 acc{0.f, 0.f, 0.f, 0.f};
  if (t.e >= 0) {
    const T* xrow = (const T*)a.x + t.xr * a.K;  // lanes without a route read row 0's: their results are not stored
    const T* wrow = (const T*)a.w + (t.e * a.N + min(n0 + c, a.N - 1)) * a.K;
    const int64_t steps = (a.K + KS - 1) / KS, per = (steps + GF_WAVES - 1) / GF_WAVES;
    const int64_t s0 = min(steps, wv * per), s1 = min(steps, s0 + per);
    int64_t s = s0;
    const int64_t whole = VEC ? min(s1, a.K / KS) : s0;  // steps with no end inside
    for (; s + UN <= whole; s += UN) {
      uint4 fi[UN], fj[UN];
#pragma unroll
      for (int d = 0; d < UN; ++d) {
        const int64_t k = (s + d) * KS + q * V;
        fi[d] = dense_ld16(wrow, k);
        fj[d] = dense_ld16(xrow, k);
      }
#pragma unroll
      for (int d = 0; d < UN; ++d) acc = dense_mfma<T>(fi[d], fj[d], acc);
    }
    for (; s < s1; ++s) {
      const int64_t k = s * KS + q * V;
      const uint4 fj = dense_ld<T, VEC>(xrow, k, a.K);
      acc = dense_mfma<T>(dense_ld<T, VEC>(wrow, k, a.K), fj, acc);
    }
  }
  red[wv][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (wv > 0) return;
  float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < GF_WAVES; ++w) {
    const float4 p = red[w][lane];
    f[0] += p.x; f[1] += p.y; f[2] += p.z; f[3] += p.w;
  }
  const int64_t n = n0 + q * 4;
  if (t.route < 0 || n >= a.N) return;
  if (!t.ok)
#pragma unroll
    for (int v = 0; v < 4; ++v) f[v] = __builtin_nanf("");
  gather_store(a, t.route * a.N + n, a.N - n, f, VEC && a.N % 4 == 0);
}

// W [E][K][N]: a lane loads V neighbouring columns of V rows of W (rows V q + s of the step) and V values of its route's
// x; product (s, u) takes value u of row s and value s of x. Bound by the wait for each step's loads: a wave walks all of K
// for its 128 columns, so a token fills few CUs. One token of 6 experts, fp16 4096 -> 2048, 258 us (k_gather_few on the other
// layout 17.6); eight tokens of 6, bf16, 298 (127).
constexpr int GT_WAVES = 4;

template <typename T, bool VEC>
__global__ __launch_bounds__(64 * GT_WAVES) void k_gather_trans(GatherArgs a) {
  constexpr int V = Dense<T>::V, KS = Dense<T>::KS;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const GatherTile t = gather_tile(a, gather_block(), lane);
  const int64_t n0 = ((int64_t)blockIdx.x * GT_WAVES + wv) * (16 * V);
  if (t.count == 0 || n0 >= a.N) return;
  f4 acc[V];
#pragma unroll
  for (int u = 0; u < V; ++u) acc[u] = f4{0.f, 0.f, 0.f, 0.f};
  if (t.e >= 0) {
    const T* xrow = (const T*)a.x + t.xr * a.K;
    const T* wb = (const T*)a.w + t.e * a.K * a.N;
    const int64_t n = n0 + c * V;
    for (int64_t k0 = 0; k0 < a.K; k0 += KS) {
      const int64_t k = k0 + q * V;
      const uint4 fj = dense_ld<T, VEC>(xrow, k, a.K);
      uint4 fi[V];
#pragma unroll
      for (int s = 0; s < V; ++s)
        fi[s] = k + s < a.K ? dense_ld<T, VEC>(wb + (k + s) * a.N, n, a.N) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int s = 0; s < V; ++s)
#pragma unroll
        for (int u = 0; u < V; ++u)
          acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(dense_at<T>(fi[s], u), dense_at<T>(fj, s), acc[u], 0, 0, 0);
    }
  }
  if (t.route < 0) return;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int64_t n = n0 + (4 * q + v) * V;
    if (n >= a.N) continue;
#pragma unroll
    for (int h = 0; h < V; h += 4) {
      float f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) f[u] = t.ok ? acc[h + u][v] : __builtin_nanf("");
      if (n + h < a.N) gather_store(a, t.route * a.N + n + h, a.N - n - h, f, VEC && a.N % 4 == 0);
    }
  }
}

// ------------------------------------------------------------------ sums of outer products over a group's rows

// Lane (c, q) of a step holds four neighbouring values of row 4 s + q of the wide side and one value per 16 of the narrow
// side; product (u, b) takes value u. Eight waves take every eighth run of 32 routes, whose ids a lane each loads once, so
// that a run's rows are all in flight together; the waves are added in order through LDS. NB: 16-wide pieces of the narrow
// side, one where a second would be empty. As dW of an odd width it reads rows value by value: a training step of 1024 tokens
// of 64 experts, 2048 -> 767, takes 2153 us (dx's share with k_gather_trans) where 768 takes 271. Bound by the wait for a run's rows: 2048 routes of 8 adapters, r = 16, 8.3 to
// 11.7 us a factor (4096 or 2048 wide, bf16), 37 with one wave a block and a route id per step.
constexpr int RO_WAVES = 8, RO_V = 4, RO_RUN = 32, RO_UN = RO_RUN / 4;

template <typename T, bool VEC>
__device__ __forceinline__ void ro_ld(const T* row, int64_t i, int64_t n, float (&f)[RO_V]) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint2 w = i < n ? *(const uint2*)(row + i) : make_uint2(0u, 0u);
    f[0] = pair_lo<PairOf<T>::value>(w.x); f[1] = pair_hi<PairOf<T>::value>(w.x);
    f[2] = pair_lo<PairOf<T>::value>(w.y); f[3] = pair_hi<PairOf<T>::value>(w.y);
  } else if constexpr (VEC) {
    const float4 w = i < n ? *(const float4*)(row + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    f[0] = w.x; f[1] = w.y; f[2] = w.z; f[3] = w.w;
  } else {
#pragma unroll
    for (int u = 0; u < RO_V; ++u) f[u] = i + u < n ? to_float(row[i + u]) : 0.f;
  }
}

template <typename TI, typename TJ, typename TO, bool VEC, int NB>
__global__ __launch_bounds__(64 * RO_WAVES) void k_rows_outer(OuterArgs a) {
  __shared__ float4 red[RO_WAVES][RO_V * NB][64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t i0 = (int64_t)blockIdx.x * (16 * RO_V), j0 = (int64_t)blockIdx.y * (16 * NB), g = blockIdx.z;
  const int64_t p0 = a.offsets[g], p1 = min(p0 + a.counts[g], a.routes);
  f4 acc[RO_V][NB];
#pragma unroll
  for (int u = 0; u < RO_V; ++u)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[u][b] = f4{0.f, 0.f, 0.f, 0.f};
  const int64_t i = i0 + c * RO_V;
  for (int64_t p = p0 + RO_RUN * wv; p < p1; p += RO_RUN * RO_WAVES) {
    const int64_t at = p + (lane & (RO_RUN - 1));
    const int id = at < p1 ? a.order[at] : -1;
    float fi[RO_UN][RO_V], fj[RO_UN][NB];
#pragma unroll
    for (int d = 0; d < RO_UN; ++d) {
      const int r = __shfl(id, 4 * d + q, 64);
      const int64_t ir = r >= 0 && r < a.routes ? (int64_t)((uint32_t)r / (uint32_t)a.i_div) : -1;
      const bool ok = ir >= 0 && ir < a.i_rows;
      ro_ld<TI, VEC>((const TI*)a.i + (ok ? ir : 0) * a.i_dim, ok ? i : a.i_dim, a.i_dim, fi[d]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int64_t j = j0 + 16 * b + c;
        fj[d][b] = ok && j < a.j_dim ? to_float(((const TJ*)a.j)[r * a.j_ld + j]) : 0.f;
      }
    }
#pragma unroll
    for (int d = 0; d < RO_UN; ++d)
#pragma unroll
      for (int u = 0; u < RO_V; ++u)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[u][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(fi[d][u], fj[d][b], acc[u][b], 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < RO_V; ++u)
#pragma unroll
    for (int b = 0; b < NB; ++b)
      red[wv][u * NB + b][lane] = make_float4(acc[u][b][0], acc[u][b][1], acc[u][b][2], acc[u][b][3]);
  __syncthreads();
  // a quarter of the waves per v: the results i0 + 4 (4 q + v) + u of column j0 + 16 b + c
  const int v = wv & 3;
  const int64_t io = i0 + (4 * q + v) * RO_V;
  if (io >= a.i_dim) return;
  TO* out = (TO*)a.out + g * a.i_dim * a.j_dim;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if ((wv >> 2) != (b & 1)) continue;
    const int64_t j = j0 + 16 * b + c;
    if (j >= a.j_dim) continue;
    float f[RO_V];
#pragma unroll
    for (int u = 0; u < RO_V; ++u) {
      f[u] = 0.f;
#pragma unroll
      for (int w = 0; w < RO_WAVES; ++w) f[u] += ((const float*)&red[w][u * NB + b][lane])[v];
    }
    if (a.j_inner) {
#pragma unroll
      for (int u = 0; u < RO_V; ++u)
        if (io + u < a.i_dim) out[(io + u) * a.j_dim + j] = from_float<TO>(f[u]);
    } else {
      dense_st<TO, RO_V>(out + j * a.i_dim + io, a.i_dim - io, f, VEC);
    }
  }
}

template <typename TI, typename TJ, typename TO, int NB>
static void outer_launch(const OuterArgs& a, int64_t groups, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)((a.i_dim + 16 * RO_V - 1) / (16 * RO_V)), (unsigned)((a.j_dim + 16 * NB - 1) / (16 * NB)),
                  (unsigned)groups);
  if (vec) hipLaunchKernelGGL((k_rows_outer<TI, TJ, TO, true, NB>), grid, dim3(64 * RO_WAVES), 0, s, a);
  else hipLaunchKernelGGL((k_rows_outer<TI, TJ, TO, false, NB>), grid, dim3(64 * RO_WAVES), 0, s, a);
}

template <typename TI, typename TJ, typename TO>
static void outer_launch(const OuterArgs& a, int64_t groups, bool vec, hipStream_t s) {
  if (a.j_dim <= 16) outer_launch<TI, TJ, TO, 1>(a, groups, vec, s);
  else outer_launch<TI, TJ, TO, 2>(a, groups, vec, s);
}

int rows_outer(const OuterArgs& a, int dtype, bool j_float, int64_t groups, hipStream_t s, const char* what) {
  const bool vec = a.i_dim % RO_V == 0 && aligned(a.i, 16) && aligned(a.out, 16);
  if (dtype == KEEP_F32) outer_launch<float, float, float>(a, groups, vec, s);
  else if (dtype == KEEP_F16 && j_float) outer_launch<_Float16, float, _Float16>(a, groups, vec, s);
  else if (dtype == KEEP_F16) outer_launch<_Float16, _Float16, _Float16>(a, groups, vec, s);
  else if (j_float) outer_launch<bf16s, float, bf16s>(a, groups, vec, s);
  else outer_launch<bf16s, bf16s, bf16s>(a, groups, vec, s);
  return launch_status(what);
}

// ------------------------------------------------------------------ host side

template <typename T>
static void gather_launch(const GatherArgs& a, bool transposed, bool vec, hipStream_t s) {
  constexpr int V = Dense<T>::V;
  const int64_t strip = transposed ? 16 * V * GT_WAVES : 16;
  const dim3 grid((unsigned)((a.N + strip - 1) / strip), (unsigned)std::min(a.tiles, GATHER_Y),
                  (unsigned)((a.tiles + GATHER_Y - 1) / GATHER_Y));
  if (transposed) {
    if (vec) hipLaunchKernelGGL((k_gather_trans<T, true>), grid, dim3(64 * GT_WAVES), 0, s, a);
    else hipLaunchKernelGGL((k_gather_trans<T, false>), grid, dim3(64 * GT_WAVES), 0, s, a);
    return;
  }
  if (vec) hipLaunchKernelGGL((k_gather_few<T, true>), grid, dim3(64 * GF_WAVES), 0, s, a);
  else hipLaunchKernelGGL((k_gather_few<T, false>), grid, dim3(64 * GF_WAVES), 0, s, a);
}

}  // namespace keep

using namespace keep;

extern "C" int keep_gather_mm_tile_supported(int dtype, int transposed, int64_t N, int64_t K, int64_t tile) {
  if (!dims_ok({N, K, tile})) return 0;
  if (tile == 16) return 1;
  return (dtype == KEEP_F16 || dtype == KEEP_BF16) && dense_gemm_tile(tile) && K % 8 == 0 && (!transposed || N % 8 == 0);
}

extern "C" int keep_gather_mm(const void* x, int dtype, int64_t x_rows, const void* weight, int transposed,
                              const int32_t* rhs, const int32_t* lhs, int64_t routes, int64_t x_div,
                              int64_t num_experts, int64_t N, int64_t K, const int32_t* order, const int32_t* offsets,
                              const int32_t* counts, const int32_t* tile_expert, const int32_t* tile_offset,
                              const int32_t* tile_count, const int32_t* valid_tiles, int64_t n_tiles, int64_t tile,
                              void* out, int out_dtype, void* stream) {
  KEEP_REQUIRE_DIMS(x_rows, routes, x_div, num_experts, N, K, n_tiles, tile);
  KEEP_REQUIRE(dtype_ok(dtype) && dtype_ok(out_dtype), "bad dtype enum");
  KEEP_REQUIRE(num_experts > 0 && N > 0 && K > 0, "num_experts, N and K must be positive");
  if (routes == 0) return KEEP_OK;
  KEEP_REQUIRE(x && weight && rhs && out && x_rows > 0, "null pointer argument");
  KEEP_REQUIRE(lhs || x_div > 0, "x_div must be > 0 without lhs");
  for (const int32_t* p : {offsets, counts, tile_expert, tile_offset, tile_count, valid_tiles})
    KEEP_REQUIRE(!order == !p, "a route plan needs all of its arrays");
  KEEP_REQUIRE(!order || n_tiles > 0, "a route plan needs n_tiles > 0");
  const bool gemm = order && tile != 16;
  KEEP_REQUIRE(!gemm || keep_gather_mm_tile_supported(dtype, transposed, N, K, tile),
               "tiles of %lld routes need 16-bit rows of whole 16-byte pieces", (long long)tile);
  const int64_t size = dtype_size(dtype);
  KEEP_REQUIRE(aligned(x, size) && aligned(weight, size) && aligned(out, dtype_size(out_dtype)), "misaligned pointer");
  GatherArgs a{};
  a.x = x; a.x_rows = x_rows; a.w = weight; a.rhs = rhs; a.lhs = lhs; a.routes = routes;
  a.x_div = x_div > 0 ? x_div : 1;
  a.E = num_experts; a.N = N; a.K = K;
  a.order = order; a.te = tile_expert; a.to = tile_offset; a.tc = tile_count;
  a.out = out; a.odt = out_dtype;
  a.tiles = order ? n_tiles : routes;
  KEEP_REQUIRE(a.tiles <= 65535 * GATHER_Y && (N + 15) / 16 <= 0xffffffffLL / (64 * GF_WAVES) &&
                   routes <= (int64_t(1) << 40) / N,  // (a value each of 2^40: more than a GPU holds)
               "too many outputs");
  if (gemm) {
    KEEP_REQUIRE(aligned(x, 16) && aligned(weight, 16) && (out_dtype == dtype || out_dtype == KEEP_F32),
                 "tiles of %lld routes need x and weight 16-byte aligned, and an output of x's dtype or float32",
                 (long long)tile);
    DenseGemmArgs g{};
    g.x = x; g.x_rows = x_rows; g.x_div = a.x_div; g.lhs = lhs; g.w = weight;
    g.E = num_experts; g.ni = N; g.nk = K; g.routes = routes;
    g.order = order; g.offsets = offsets; g.counts = counts;
    g.te = tile_expert; g.to = tile_offset; g.tc = tile_count; g.n_tiles = valid_tiles; g.max_tiles = n_tiles;
    g.out = out; g.odt = out_dtype; g.wide = N % 8 == 0 && aligned(out, 16);
    return dense_gemm_rows(g, dtype, transposed, tile, (hipStream_t)stream);
  }
  const int64_t v = 16 / size;
  const bool vec = K % v == 0 && (!transposed || N % v == 0) && aligned(x, 16) && aligned(weight, 16) &&
                   aligned(out, 16);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KEEP_F32) gather_launch<float>(a, transposed, vec, s);
  else if (dtype == KEEP_F16) gather_launch<_Float16>(a, transposed, vec, s);
  else gather_launch<bf16s>(a, transposed, vec, s);
  return launch_status("keep_gather_mm");
}

extern "C" int keep_gather_mm_grad_weight(const void* x, int dtype, int64_t x_rows, const void* dy, int64_t routes,
                                          int64_t x_div, int64_t num_experts, int64_t N, int64_t K,
                                          const int32_t* order, const int32_t* offsets, const int32_t* counts,
                                          void* dw, void* stream) {
  KEEP_REQUIRE_DIMS(x_rows, routes, x_div, num_experts, N, K);
  KEEP_REQUIRE(dtype_ok(dtype), "bad dtype enum");
  KEEP_REQUIRE(num_experts > 0 && N > 0 && K > 0 && x_div > 0, "num_experts, N, K and x_div must be positive");
  KEEP_REQUIRE(num_experts <= 65535 && (N + 31) / 32 <= 65535, "too many experts or outputs");
  KEEP_REQUIRE(offsets && counts && dw && (routes == 0 || (x && dy && order && x_rows > 0)), "null pointer argument");
  const int64_t size = dtype_size(dtype);
  KEEP_REQUIRE(aligned(x, size) && aligned(dy, size) && aligned(dw, size), "misaligned pointer");
  if (dtype != KEEP_F32 && N % 8 == 0 && K % 8 == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dw, 16)) {
    KEEP_REQUIRE(num_experts <= 0x7ffffff0LL / (((N + 63) / 64) * ((K + 63) / 64)), "too many outputs");
    DenseGemmArgs g{};
    g.x = x; g.x_rows = x_rows; g.x_div = x_div; g.w = dy;
    g.E = num_experts; g.ni = K; g.nj = N; g.routes = routes;
    g.order = order; g.offsets = offsets; g.counts = counts;
    g.out = dw; g.odt = dtype; g.wide = 1;
    return dense_gemm_weight(g, dtype, (hipStream_t)stream);
  }
  OuterArgs a{};
  a.i = x; a.i_rows = x_rows; a.i_div = x_div; a.i_dim = K;
  a.j = dy; a.j_ld = N; a.j_dim = N;
  a.order = order; a.offsets = offsets; a.counts = counts; a.routes = routes;
  a.out = dw; a.j_inner = 0;
  return rows_outer(a, dtype, false, num_experts, (hipStream_t)stream, "keep_gather_mm_grad_weight");
}
