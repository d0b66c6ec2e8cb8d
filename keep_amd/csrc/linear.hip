// Dense projections with their epilogue and their gradients:
//
//   u = x W^T + b          out = round(residual + act(u))
//   du = round(dy act'(u)) dx = du W        dW = du^T x        db = sum of du's rows (before its rounding)
//
// 8-bit operands (e4m3): x W^T with a float32 scale per 128 values of a row of x and per 128 x 128 values of W, no gradients.
// Sums are held in fp32 on the matrix cores. Up to 16 rows stream W straight to the matrix cores (k_linear_few: a byte of W
// serves few products, so that HBM bounds it); more run through LDS (linear_gemm_dev.h), in slices of the summed index
// (k_linear_join) where there are fewer tiles than CUs. u is kept for the gradient in x's dtype and du rounded to it: the
// matrix cores take 16-bit operands, and both roundings are half a step of the dtype that dy has. By them dx and dW of 4096 x
// 4096 -> 2048 bf16 with silu lie 0.0024 (relative, root mean square) from their 64-bit values; rounding them alone leaves 0.0017.
#include <algorithm>

#include "linear_dev.h"
#include "parts_dev.h"

namespace keep {

void linear_gemm_bf16(const LinearGemmArgs& a, int mode, int tile, hipStream_t s);
void linear_gemm_f16(const LinearGemmArgs& a, int mode, int tile, hipStream_t s);
void linear_gemm_f32(const LinearGemmArgs& a, int mode, int tile, hipStream_t s);
void linear_gemm_e4m3(const LinearGemmArgs& a, int mode, int tile, hipStream_t s);

static void linear_gemm(const LinearGemmArgs& a, int dtype, int mode, int tile, hipStream_t s) {
  if (dtype == KEEP_BF16) linear_gemm_bf16(a, mode, tile, s);
  else if (dtype == KEEP_F16) linear_gemm_f16(a, mode, tile, s);
  else if (dtype == KEEP_F32) linear_gemm_f32(a, mode, tile, s);
  else linear_gemm_e4m3(a, mode, tile, s);
}

static int64_t linear_size(int dtype) { return dtype == KEEP_E4M3 ? 1 : dtype_size(dtype); }

// ------------------------------------------------------------------ few rows

// Rows of the kernel below. Against tiles of 64 x 64 through LDS, microseconds of bf16 in a graph, one row / 16 rows: 4096 -> 384
// 7.1 / 9.9 against 8.6 / 9.5, 4096 -> 4096 7.7 / 10.4 against 11.2 / 12.6, 4096 -> 8192 13.6 / 17.6 against 16.9 / 16.9,
// 512 -> 65536 14.1 / 18.1 against 16.6 / 17.2; 17 rows of 4096 -> 4096 take 12.6 there.
constexpr int LINEAR_FEW = 16;

// 16 bytes at any address of a value.
__device__ __forceinline__ uint4 linear_ld16_any(const char* p) {
  typedef unsigned int v4u __attribute__((ext_vector_type(4), aligned(2)));
  const v4u v = *(const __attribute__((address_space(1))) v4u*)p;
  return make_uint4(v.x, v.y, v.z, v.w);
}

// The piece at value k of a row of n values that starts at row, zeros past its end: read whole from before the end and moved
// down where the row ends inside it.
template <typename T>
__device__ __forceinline__ uint4 linear_piece_any(const char* row, int64_t k, int64_t n) {
  constexpr int SZ = sizeof(T), V = 16 / SZ;
  uint32_t m[4] = {0u, 0u, 0u, 0u};
  if (k + V <= n) return linear_ld16_any(row + k * SZ);
  if (k < n && n >= V) {
    const uint4 r = linear_ld16_any(row + (n - V) * SZ);
    m[0] = r.x; m[1] = r.y; m[2] = r.z; m[3] = r.w;
    const int down = (int)(k + V - n) * SZ;  // bytes
#pragma unroll
    for (int s = 2; s > 0; --s)
      if (down & 4 * s)
#pragma unroll
        for (int u = 0; u < 4; ++u) m[u] = u + s < 4 ? m[u + s < 4 ? u + s : 0] : 0u;
    if (down & 2)
#pragma unroll
      for (int u = 0; u < 4; ++u) m[u] = m[u] >> 16 | (u < 3 ? m[u < 3 ? u + 1 : 0] << 16 : 0u);
  } else if (k < n) {  // (k = 0)
#pragma unroll
    for (int u = 0; u < V - 1; ++u)
      if (u < n) {
        if constexpr (SZ == 4) m[u] = ((const uint32_t*)row)[u];
        else m[u / 2] |= (uint32_t)((const uint16_t*)row)[u] << (16 * (u & 1));
      }
  }
  return make_uint4(m[0], m[1], m[2], m[3]);
}

// Eight waves share 16 rows of W (and the rows of x): wave s takes the s-th share of the summed index and the shares are added
// in order through LDS. Lane (c, q) holds W row n0 + c, so that its results are outputs n0 + 4 q + v of row c. The loads of UN
// steps are in flight at a time. 4096 -> 4096 bf16, one row: 7.7 us, 4.4 TB/s of W; what is left of a call of one strip a CU
// (4096 -> 384: 7.1) is launch and the loads' latency. Sixteen waves: 7.7 and 7.1, but 512 -> 65536 22 us for 14; four or eight
// rows of W a block where there are few strips: 7.4 for 7.1.
// ANY: rows at any address and of any length (1 x 3925 -> 3510 bf16 14.1 us, of 3924 values
// 7.4; copied into whole pieces first 27).
template <typename T, bool ANY>
__global__ __launch_bounds__(512) void k_linear_few(LinearGemmArgs a) {
  constexpr int WAVES = 8;
  constexpr int SZ = sizeof(T), LB = SZ == 1 ? 32 : 16;  // bytes of a lane's piece
  constexpr int VL = LB / SZ, KS = 4 * VL, UN = SZ == 1 ? 4 : 8;
  __shared__ float4 red[WAVES][64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const char* xrow = (const char*)a.pj + min((int64_t)c, a.nj - 1) * a.ldj * SZ + q * LB;
  const char* wrow = (const char*)a.pi + min(n0 + c, a.ni - 1) * a.ldi * SZ + q * LB;
  const auto ld = [](const char* row, int at) {
    if constexpr (ANY) return linear_ld16_any(row + at);
    else return dense_ld16((const uint8_t*)row, at);
  };
  const int64_t kb = (a.nk + KS - 1) / KS;  // (8-bit: a scale's span each)
  const float* xs = SZ == 1 ? a.sj + min((int64_t)c, a.nj - 1) * kb : nullptr;
  const float* ws = SZ == 1 ? a.si + n0 / 128 * kb : nullptr;
  const int steps = (int)kb, per = (steps + WAVES - 1) / WAVES;
  const int s0 = min(steps, wv * per), s1 = min(steps, s0 + per), whole = min(s1, (int)(a.nk / KS));
  f4 acc{0.f, 0.f, 0.f, 0.f};
  const auto product = [&](const uint4* i, const uint4* j, float scale) {
    if constexpr (SZ == 1) {
      linear_h8 fi[4], fj[4];
      linear_e4m3(i[0], i[1], fi);
      linear_e4m3(j[0], j[1], fj);
      f4 p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(fi[t], fj[t], p, 0, 0, 0);
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[v] = fmaf(p[v], scale, acc[v]);
    } else {
      acc = dense_mfma<T>(i[0], j[0], acc);
    }
  };
  constexpr int P = LB / 16;
  int s = s0;
  for (; s + UN <= whole; s += UN) {
    uint4 fi[UN][P], fj[UN][P];
    float sc[UN];
#pragma unroll
    for (int d = 0; d < UN; ++d) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        fi[d][p] = ld(wrow, (s + d) * (KS * SZ) + p * 16);
        fj[d][p] = ld(xrow, (s + d) * (KS * SZ) + p * 16);
      }
      sc[d] = SZ == 1 ? xs[s + d] * ws[s + d] : 1.f;
    }
#pragma unroll
    for (int d = 0; d < UN; ++d) product(fi[d], fj[d], sc[d]);
  }
  for (; s < s1; ++s) {
    uint4 fi[P], fj[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if constexpr (ANY) {
        const int64_t k = (int64_t)s * KS + q * VL;
        fi[p] = linear_piece_any<T>(wrow - q * LB, k, a.nk);
        fj[p] = linear_piece_any<T>(xrow - q * LB, k, a.nk);
        continue;
      }
      const bool in = (int64_t)s * KS + (q * LB + p * 16) / SZ < a.nk;  // (pieces are whole or past the end)
      const int64_t at = (int64_t)s * (KS * SZ) + p * 16;
      fi[p] = in ? dense_ld16((const uint8_t*)wrow, at) : make_uint4(0u, 0u, 0u, 0u);
      fj[p] = in ? dense_ld16((const uint8_t*)xrow, at) : make_uint4(0u, 0u, 0u, 0u);
    }
    product(fi, fj, SZ == 1 ? xs[s] * ws[s] : 1.f);
  }
  red[wv][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (wv > 0) return;
  float f[4] = {0.f, 0.f, 0.f, 0.f}, b[4];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float4 p = red[w][lane];
    f[0] += p.x; f[1] += p.y; f[2] += p.z; f[3] += p.w;
  }
  const int64_t n = n0 + q * 4;
  if (c >= a.nj || n >= a.ni) return;
  a.e.load_bias<4>(n, a.ni - n, b);
  a.e.store<4>(c, a.ni, n, a.ni - n, f, b);
}

template <typename T>
static void linear_few_launch(const LinearGemmArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.ni + 15) / 16));
  if constexpr (sizeof(T) > 1) {
    if (a.any) {
      hipLaunchKernelGGL((k_linear_few<T, true>), grid, dim3(512), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((k_linear_few<T, false>), grid, dim3(512), 0, s, a);
}

static void linear_few(const LinearGemmArgs& a, int dtype, hipStream_t s) {
  if (dtype == KEEP_BF16) linear_few_launch<bf16s>(a, s);
  else if (dtype == KEEP_F16) linear_few_launch<_Float16>(a, s);
  else if (dtype == KEEP_F32) linear_few_launch<float>(a, s);
  else linear_few_launch<e4m3s>(a, s);
}

// ------------------------------------------------------------------ slices added

__global__ __launch_bounds__(256) void k_linear_join(LinearGemmArgs a) {
  const int64_t groups = (a.ni + 7) / 8, n = a.nj * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / groups, col = (i - row * groups) * 8;
    float f[8], b[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = 0.f;
    for (int s = 0; s < a.slices; ++s) {
      float p[8];
      linear_ld<float, 8>(a.part + (s * a.nj + row) * a.ni + col, a.ni - col, p, a.ni % 4 == 0);
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] += p[u];
    }
    a.e.load_bias<8>(col, a.ni - col, b);
    a.e.store<8>(row, a.ni, col, a.ni - col, f, b);
  }
}

struct LinearPlan {
  int tile, slices;
  int64_t tiles;
};

// The tile and the slices of a product. Microseconds of bf16 in a graph:
// - The largest tile that still gives the CUs about one each. Tiles of 256 x 256 / 256 x 128 / 128 x 128: 8192 x 4096 -> 8192
//   454 / 520 / 590; 4096 x 4096 -> 2048 (128, 256 and 512 tiles) 106 / 73 / 87. 128 x 128 by two groups of waves / 64 x 64:
//   1024 x 4096 -> 4096 (256 and 1024 tiles) 39 / 54, 4096 x 2048 -> 768 (192, 768) 22.3 / 26.3, 1024 x 4096 -> 2048 (128, 512)
//   35 / 28, fp16 333 x 2880 -> 1440 (36, 138) 24 / 11. One group for two: 600 x 4096 -> 2048 43 / 32.
// - float32's products take sixteen times as long, so that its tiles go by the rounds of 256 CUs, four and a half of 64 x 64
//   for one of 128 x 128: 1024 x 4096 -> 2048 (128 and 512 tiles) 241 / 133, 1024 x 2880 -> 1440 and
//   its dW (96 and 276, 368 and 1035) 225 / 174.
// - Slices take a second launch, 4 us: they pay where the sum is long and CUs have no work. 64 x 64 tiles, one slice / more:
//   512 x 4096 -> 2048 (256 tiles) 23.5 / 21.2 (two), 64 x 2880 -> 1440 (23) 11.7 / 9.9 (three), 384 x 2880 -> 1440 (138)
//   12.3 / 15.6 (two), 64 x 2048 -> 768 (12) 9.4 / 9.5 (two). Two, four and eight of 128 x 4096 -> 2048 (64 tiles, 64 steps)
//   13.5, 12.8 and 15.8; of 256 x 4096 -> 2048 in float32 (128, 128 steps) two 42, three 50, four 40. 128 x 128 tiles in two
//   slices against 64 x 64: 1024 x 7168 -> 2048 42 / 46, of 4096 inputs 30 / 28.
static LinearPlan linear_plan(int dtype, int mode, int64_t ni, int64_t nj, int64_t nk) {
  const auto tiles = [&](int64_t bi, int64_t bj) { return ((ni + bi - 1) / bi) * ((nj + bj - 1) / bj); };
  if (mode == LINEAR_FORWARD && nj <= LINEAR_FEW) return {LINEAR_TILE_FEW, 1, tiles(16, 16)};
  const bool small = dtype == KEEP_F32;
  if (!small && dtype != KEEP_E4M3 && tiles(256, 256) >= 224) return {LINEAR_TILE_256, 1, tiles(256, 256)};
  if (!small && tiles(256, 128) >= 192) return {LINEAR_TILE_256_128, 1, tiles(256, 128)};
  const int64_t n = tiles(128, 128), m = tiles(64, 64), rn = (n + 255) / 256, rm = (m + 255) / 256;
  const int64_t steps = (nk * std::max<int64_t>(linear_size(dtype), 2) + 127) / 128;  // (8-bit values are 16-bit ones' work)
  if (nj > 64 && ni > 64) {
    if (small ? 32 * rn <= 9 * rm : n >= 160) return {n <= 256 ? LINEAR_TILE_128_2 : LINEAR_TILE_128, 1, n};
    if (!small && n >= 96 && n <= 128 && steps >= 96) return {LINEAR_TILE_128_2, 2, n};
  }
  const int64_t room = (small || steps <= 48 ? 256 : 512) / m;
  const int64_t slices = steps < 40 ? 1 : std::max<int64_t>(1, std::min<int64_t>({room, steps / 14, 32}));
  return {LINEAR_TILE_64, (int)slices, m};
}

static int64_t linear_part_bytes(const LinearPlan& p, int64_t ni, int64_t nj) {
  return p.slices > 1 ? p.slices * ni * nj * 4 : 0;
}

// Blocks of a launch: it holds 2^32 threads.
static bool linear_gemm_fits(const LinearPlan& p) { return p.tiles <= (int64_t(1) << 22) / p.slices; }

static void linear_product(LinearGemmArgs a, int dtype, int mode, const LinearPlan& p, void* part, hipStream_t s) {
  a.slices = p.slices;
  a.part = (float*)part;
  if (p.tile == LINEAR_TILE_FEW) {
    linear_few(a, dtype, s);
    return;
  }
  linear_gemm(a, dtype, mode, p.tile, s);
  if (p.slices > 1) {
    const int64_t n = a.nj * ((a.ni + 7) / 8);
    hipLaunchKernelGGL(k_linear_join, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, s, a);
  }
}

// ------------------------------------------------------------------ the gradient before the products

struct LinearDuArgs {
  const void *dy, *u;
  int act;
  int64_t M, N, ld;  // ld: of du, whole 16-byte pieces, zeros behind the columns
  void* du;          // or null
  float* part;       // [gridDim.y][N] sums of du, or null
  void* db;          // one block of rows: their sum at once, in part's place
  int bdt;
  int64_t rows;      // of a block
};

// Threads of 8 neighbouring columns, 8 rows at a time.
template <typename T>
__global__ __launch_bounds__(256) void k_linear_du(LinearDuArgs a) {
  __shared__ float red[8][32][8 + 1];
  const int cg = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const int64_t col = ((int64_t)blockIdx.x * 32 + cg) * 8;
  const int64_t r0 = (int64_t)blockIdx.y * a.rows, r1 = min(a.M, r0 + a.rows);
  const bool vec = a.N % 8 == 0 && ((uintptr_t)a.dy & 15) == 0 && (!a.u || ((uintptr_t)a.u & 15) == 0);
  float sum[8] = {};
  if (col < a.ld) {
    for (int64_t r = r0 + rg; r < r1; r += 8) {
      float d[8], u[8];
      const int64_t left = max(a.N - col, (int64_t)0);
      linear_ld<T, 8>((const T*)a.dy + r * a.N + col, left, d, vec);
      if (a.act) {
        linear_ld<T, 8>((const T*)a.u + r * a.N + col, left, u, vec);
        linear_slope<8>(d, u, a.act);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += d[i];
      if (a.du) {
        if (left < 8)
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = i < left ? d[i] : 0.f;
        linear_st<T, 8>((T*)a.du + r * a.ld + col, a.ld - col, d, true);
      }
    }
  }
  if (!a.part && !a.db) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[rg][cg][i] = sum[i];
  __syncthreads();
  // a thread a column: the block's 256
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += red[k][threadIdx.x >> 3][threadIdx.x & 7];
  if (a.part) a.part[blockIdx.y * a.N + n] = v;
  else if (a.bdt == KEEP_F32) ((float*)a.db)[n] = v;
  else if (a.bdt == KEEP_BF16) ((bf16s*)a.db)[n] = from_float<bf16s>(v);
  else ((_Float16*)a.db)[n] = from_float<_Float16>(v);
}

constexpr int64_t LINEAR_MAX = int64_t(1) << 20;  // N and K: a tile's rows then lie within 32-bit offsets

// Row blocks of k_linear_du: enough for the CUs, a few thousand rows at most each.
static int64_t linear_du_blocks(int64_t M, int64_t N) {
  const int64_t strips = (N + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>({(M + 31) / 32, (1024 + strips - 1) / strips, 512}));
}

static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
static int64_t linear_pitch(int64_t n, int64_t size) { return (n * size + 15) / 16 * 16 / size; }

struct LinearGradPlan {
  LinearPlan rows, weight;
  int64_t du, part, db, bytes;  // offsets
};

static LinearGradPlan linear_grad_plan(int dtype, int64_t M, int64_t N, int64_t K) {
  LinearGradPlan p{};
  const int64_t size = linear_size(dtype);
  p.rows = linear_plan(dtype, LINEAR_ROWS, K, M, N);
  p.weight = linear_plan(dtype, LINEAR_WEIGHT, K, N, M);
  p.part = up256(M * linear_pitch(N, size) * size);
  p.db = p.part + up256(std::max(linear_part_bytes(p.rows, K, M), linear_part_bytes(p.weight, K, N)));
  p.bytes = p.db + up256(linear_du_blocks(M, N) * N * 4);
  return p;
}

static bool linear_vec(std::initializer_list<const void*> ps, int64_t n) {
  if (n % 8) return false;
  for (const void* p : ps)
    if (!aligned(p, 16)) return false;
  return true;
}

// What forward calls ask beside their operands.
static int linear_epilogue(LinearEpilogue& e, int64_t M, int64_t N, const void* bias, int bdt, int act, const void* res,
                           int rdt, void* u, int udt, void* out, int odt) {
  KEEP_REQUIRE((!bias || dtype_ok(bdt)) && (!res || dtype_ok(rdt)) && dtype_ok(odt), "bad dtype enum");
  KEEP_REQUIRE(act >= LINEAR_NONE && act <= LINEAR_GELU_TANH, "bad activation %d", act);
  KEEP_REQUIRE(aligned(out, dtype_size(odt)) && (!bias || aligned(bias, dtype_size(bdt))) &&
                   (!res || aligned(res, dtype_size(rdt))) && (!u || aligned(u, dtype_size(udt))),
               "misaligned pointer");
  e.bias = bias; e.bdt = bdt; e.act = act; e.res = res; e.rdt = rdt; e.u = u; e.udt = udt; e.out = out; e.odt = odt;
  e.vec = linear_vec({bias, res, u, out}, N);
  return KEEP_OK;
}

static int linear_sizes(int64_t M, int64_t N, int64_t K) {
  KEEP_REQUIRE_DIMS(M, N, K);
  KEEP_REQUIRE(N >= 1 && K >= 1 && N <= LINEAR_MAX && K <= LINEAR_MAX, "N and K must be in 1..2^20");
  KEEP_REQUIRE(M <= (int64_t(1) << 40) / std::max(N, K) / 4, "too many values");  // more than a GPU holds
  return KEEP_OK;
}

// Rows of n values at a pitch of ld: the kernels read whole 16-byte pieces.
#define KEEP_REQUIRE_PITCH(p, ld, n, size, what)                                                         \
  KEEP_REQUIRE(aligned(p, 16) && (ld) >= (n) && (ld) < KEEP_DIM_LIMIT && (ld) <= 4 * LINEAR_MAX &&       \
                   ((ld) * (size)) % 16 == 0,                                                            \
               what " must be 16-byte aligned, its pitch at least a row and a multiple of 16 bytes")

}  // namespace keep

using namespace keep;

extern "C" int64_t keep_linear_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  if (!(dtype_ok(dtype) || dtype == KEEP_E4M3) || linear_sizes(M, N, K) != KEEP_OK || M == 0) return 0;
  return linear_part_bytes(linear_plan(dtype, LINEAR_FORWARD, N, M, K), N, M);
}

static int linear_forward(LinearGemmArgs& a, int dtype, void* ws, int64_t ws_bytes, hipStream_t s) {
  const LinearPlan p = linear_plan(dtype, LINEAR_FORWARD, a.ni, a.nj, a.nk);
  const int64_t need = linear_part_bytes(p, a.ni, a.nj);
  KEEP_REQUIRE(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need),
               "the workspace must hold %lld bytes, 16-byte aligned", (long long)need);
  KEEP_REQUIRE(linear_gemm_fits(p), "too many outputs");
  linear_product(a, dtype, LINEAR_FORWARD, p, ws, s);
  return KEEP_OK;
}

extern "C" int keep_linear(const void* x, int64_t x_ld, int dtype, int64_t M, const void* weight, int64_t w_ld, int64_t N,
                           int64_t K, const void* bias, int bias_dtype, int act, const void* residual,
                           int residual_dtype, void* u, void* out, int out_dtype, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  if (const int rc = linear_sizes(M, N, K)) return rc;
  KEEP_REQUIRE(dtype_ok(dtype), "bad dtype enum");
  if (M == 0) return KEEP_OK;
  KEEP_REQUIRE(x && weight && out, "null pointer argument");
  LinearGemmArgs a{};
  const int64_t size = linear_size(dtype);
  if (M <= LINEAR_FEW) {
    KEEP_REQUIRE(aligned(x, size) && aligned(weight, size) && x_ld >= K && w_ld >= K && x_ld <= 4 * LINEAR_MAX &&
                     w_ld <= 4 * LINEAR_MAX,
                 "x and weight must be aligned to their dtype, their pitch at least a row");
    a.any = !aligned(x, 16) || !aligned(weight, 16) || (x_ld | w_ld | K) * size % 16 != 0;
  } else {
    KEEP_REQUIRE_PITCH(x, x_ld, K, size, "x");
    KEEP_REQUIRE_PITCH(weight, w_ld, K, size, "weight");
  }
  a.pi = weight; a.pj = x; a.ldi = w_ld; a.ldj = x_ld; a.ni = N; a.nj = M; a.nk = K;
  if (const int rc = linear_epilogue(a.e, M, N, bias, bias_dtype, act, residual, residual_dtype, u, dtype, out, out_dtype))
    return rc;
  if (const int rc = linear_forward(a, dtype, workspace, workspace_bytes, (hipStream_t)stream)) return rc;
  return launch_status("keep_linear");
}

extern "C" int keep_linear_q8(const void* x, int64_t x_ld, const float* x_scales, int64_t M, const void* weight,
                              int64_t w_ld, const float* w_scales, int64_t N, int64_t K, const void* bias,
                              int bias_dtype, int act, const void* residual, int residual_dtype, void* out,
                              int out_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = linear_sizes(M, N, K)) return rc;
  if (M == 0) return KEEP_OK;
  KEEP_REQUIRE(x && weight && x_scales && w_scales && out, "null pointer argument");
  KEEP_REQUIRE(aligned(x_scales, 4) && aligned(w_scales, 4), "misaligned pointer");
  KEEP_REQUIRE_PITCH(x, x_ld, K, 1, "x");
  KEEP_REQUIRE_PITCH(weight, w_ld, K, 1, "weight");
  LinearGemmArgs a{};
  a.pi = weight; a.pj = x; a.ldi = w_ld; a.ldj = x_ld; a.ni = N; a.nj = M; a.nk = K;
  a.si = w_scales; a.sj = x_scales;
  if (const int rc = linear_epilogue(a.e, M, N, bias, bias_dtype, act, residual, residual_dtype, nullptr, 0, out, out_dtype))
    return rc;
  if (const int rc = linear_forward(a, KEEP_E4M3, workspace, workspace_bytes, (hipStream_t)stream)) return rc;
  return launch_status("keep_linear_q8");
}

extern "C" int64_t keep_linear_grad_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  if (!dtype_ok(dtype) || linear_sizes(M, N, K) != KEEP_OK || M == 0) return 0;
  return linear_grad_plan(dtype, M, N, K).bytes;
}

extern "C" int keep_linear_grad(const void* dy, const void* u, int act, const void* x, int64_t x_ld, const void* weight,
                                int64_t w_ld, int dtype, int64_t M, int64_t N, int64_t K, void* dx, void* dweight,
                                void* dbias, int bias_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = linear_sizes(M, N, K)) return rc;
  KEEP_REQUIRE(dtype_ok(dtype) && (!dbias || dtype_ok(bias_dtype)), "bad dtype enum");
  KEEP_REQUIRE(act >= LINEAR_NONE && act <= LINEAR_GELU_TANH, "bad activation %d", act);
  if (M == 0) return KEEP_OK;
  const int64_t size = linear_size(dtype);
  KEEP_REQUIRE(dy && (dx || dweight || dbias) && (u || !act) && (x || !dweight) && (weight || !dx),
               "null pointer argument");
  KEEP_REQUIRE(aligned(dy, size) && aligned(u, size) && aligned(dx, size) && aligned(dweight, size) &&
                   (!dbias || aligned(dbias, dtype_size(bias_dtype))),
               "misaligned pointer");
  if (dweight) KEEP_REQUIRE_PITCH(x, x_ld, K, size, "x");
  if (dx) KEEP_REQUIRE_PITCH(weight, w_ld, K, size, "weight");
  const LinearGradPlan p = linear_grad_plan(dtype, M, N, K);
  KEEP_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= p.bytes,
               "the workspace must hold %lld bytes, 256-byte aligned", (long long)p.bytes);
  KEEP_REQUIRE(linear_gemm_fits(p.rows) && linear_gemm_fits(p.weight), "too many outputs");
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  // du: dy itself where no activation changes it and its rows are whole pieces
  const bool same = !act && (N * size) % 16 == 0 && aligned(dy, 16);
  const bool products = dx || dweight;
  const void* du = same ? dy : ws + p.du;
  if (dbias || (products && !same)) {
    LinearDuArgs d{};
    d.dy = dy; d.u = u; d.act = act; d.M = M; d.N = N; d.ld = linear_pitch(N, size);
    d.du = products && !same ? ws + p.du : nullptr;
    const int64_t blocks = linear_du_blocks(M, N);
    d.part = dbias && blocks > 1 ? (float*)(ws + p.db) : nullptr;
    d.db = blocks > 1 ? nullptr : dbias;
    d.bdt = bias_dtype;
    d.rows = (M + blocks - 1) / blocks;
    const dim3 grid((unsigned)((N + 255) / 256), (unsigned)blocks);
    if (dtype == KEEP_F32) hipLaunchKernelGGL(k_linear_du<float>, grid, dim3(256), 0, s, d);
    else if (dtype == KEEP_F16) hipLaunchKernelGGL(k_linear_du<_Float16>, grid, dim3(256), 0, s, d);
    else hipLaunchKernelGGL(k_linear_du<bf16s>, grid, dim3(256), 0, s, d);
    if (d.part) parts_sum(d.part, blocks, N, dbias, bias_dtype, s);
  }
  LinearGemmArgs a{};
  a.e.odt = dtype;
  if (dx) {
    a.pi = weight; a.ldi = w_ld; a.pj = du; a.ldj = linear_pitch(N, size);
    a.ni = K; a.nj = M; a.nk = N;
    a.e.out = dx;
    a.e.vec = linear_vec({dx}, K);
    linear_product(a, dtype, LINEAR_ROWS, p.rows, ws + p.part, s);
  }
  if (dweight) {
    a.pi = x; a.ldi = x_ld; a.pj = du; a.ldj = linear_pitch(N, size);
    a.ni = K; a.nj = N; a.nk = M;
    a.e.out = dweight;
    a.e.vec = linear_vec({dweight}, K);
    linear_product(a, dtype, LINEAR_WEIGHT, p.weight, ws + p.part, s);
  }
  return launch_status("keep_linear_grad");
}
