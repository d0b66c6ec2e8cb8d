// Routed products with dense 16-bit expert weights through LDS: prefill and
// training. The routes come sorted by expert (a route plan).
//
//   FORWARD  out[r] = W[e] x[row_r]                    W [E][N][K], one tile of a plan per block row
//   TRANS    out[r] = W[e]^T x[row_r]                  W [E][K][N], the same tiles
//   WEIGHT   dW[e][n][k] = sum_r dy[r][n] x[row_r][k]  one expert per block row, its routes the summed index
//
// Both operands of a 64-wide step are copied to LDS by the DMA path (16 bytes a
// lane, no registers), into the other of two buffers while the matrix cores
// work on this one; one barrier per step. The side whose index is contiguous in
// the output ("I") is the first MFMA operand, so a lane ends with 16
// neighbouring outputs of a row (see dense_dev.h).
//
// An operand whose rows run along the summed index is stored as it is, 128 bytes
// a row, its eight 16-byte slots permuted so that the 16 rows of a fragment fall
// on all banks. An operand that has the summed index across its rows is stored
// as it is too, rows of the tile's width, and read with the transposing LDS
// loads (four rows of 16 columns a time), its 32-byte pairs permuted likewise.
// Past an operand's end, lanes copy a zero instead.
#include <algorithm>

#include "dense_dev.h"
#include "dense_gemm.h"

namespace keep {

__device__ __attribute__((aligned(16))) uint4 g_zero16;

constexpr int DG_K = 64;  // summed index per step

enum { DG_FORWARD = 0, DG_TRANS = 1, DG_WEIGHT = 2 };

// Slot permutations: rows 2 m and 2 m + 1 share 256 bytes (all banks), so the eight row pairs of a fragment get eight
// different slots. J fragments hold 16 neighbouring rows, I fragments rows 16 a + 4 u + b (a, b = 0..3) of a group of 64.
__device__ __forceinline__ int dg_swz_j(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int dg_swz_i(int row) { return ((row >> 1) & 1) | (((row >> 4) & 3) << 1); }
// Pair permutation of a transposed operand: a read takes rows 8 q .. 8 q + 3 of all four quarters q.
template <int COLS>
__device__ __forceinline__ int dg_swz_t(int row) {
  return ((row & 3) | (((row >> 3) & 1) << 2)) & (COLS / 16 - 1);
}

// Fragment of 8 summed values at step ks: row `row` of a plain operand.
template <int SWZ_I>
__device__ __forceinline__ uint4 dg_frag(const char* s, int row, int ks, int q) {
  const int slot = (ks * 4 + q) ^ (SWZ_I ? dg_swz_i(row) : dg_swz_j(row));
  return *(const uint4*)(s + row * 128 + slot * 16);
}

// ... and column 16 ct + c of a transposed operand of COLS columns: two transposing loads of four rows each.
template <int COLS>
__device__ __forceinline__ uint4 dg_frag_t(const char* s, int ct, int ks, int lane) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  const int q = lane >> 4, m = lane & 15;
  const int row = ks * 32 + q * 8 + (m >> 2);
  const char* p = s + row * (2 * COLS) + ((ct ^ dg_swz_t<COLS>(row)) * 32 + (m & 3) * 8);
  union {
    s4 h[2];
    uint4 v;
  } f;
  f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
  f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 4 * (2 * COLS)));
  return f.v;
}

// 16 bytes per lane from g to lds_wave_base + 16 lane. Written out, since the compiler waits for every copy in flight
// before any LDS read that follows the builtin: here the reads are of the other buffer, and the loop's own wait and
// barrier stand between a copy and its readers. (No register is written, so none can be reused early.)
__device__ __forceinline__ void dg_dma(const void* g, uint32_t lds_wave_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_wave_base), "v"(g)
               : "memory");
}

template <typename T, int BI, int BJ, int WI, int WJ, int MODE>
__global__ __launch_bounds__(64 * WI * WJ) void k_dense_gemm(DenseGemmArgs a) {
  constexpr int NT = 64 * WI * WJ, TI = BI / WI, TJ = BJ / WJ, FI = TI / 16, FJ = TJ / 16;
  constexpr int LI = BI * 8 / NT, LJ = BJ * 8 / NT;  // 16-byte copies per thread and step
  constexpr int SI = BI * 128, SJ = BJ * 128;        // bytes of a buffer's operands
  constexpr bool TRI = MODE != DG_FORWARD, TRJ = MODE == DG_WEIGHT;
  __shared__ __attribute__((aligned(16))) char smem[2 * (SI + SJ)];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wv % WI, wj = wv / WI;

  // work item: (j tile or expert and row block, i block), dealt to the XCDs in contiguous runs
  int64_t e, jt, ib;
  int count = 0;
  int64_t off = 0;
  {
    const int64_t nib = (a.ni + BI - 1) / BI;
    int64_t total;
    if constexpr (MODE == DG_WEIGHT) total = a.E * ((a.nj + BJ - 1) / BJ) * nib;
    else {
      int64_t tiles = a.n_tiles[0];  // tiles of valid experts; those of invalid routes follow
      const int64_t valid = (int64_t)a.offsets[a.E - 1] + a.counts[a.E - 1];
      tiles = min(tiles + (a.routes - valid + BJ - 1) / BJ, a.max_tiles);
      total = tiles * nib;
    }
    const int64_t per = (total + 7) / 8;
    const int64_t slot = blockIdx.x >> 3;
    if (slot >= per) return;
    const int64_t item = (blockIdx.x & 7) * per + slot;
    if (item >= total) return;
    if constexpr (MODE == DG_WEIGHT) {
      const int64_t njb = (a.nj + BJ - 1) / BJ;
      e = item / (njb * nib);
      const int64_t r = item - e * (njb * nib);
      jt = r / nib;
      ib = r - jt * nib;
      off = a.offsets[e];
      count = (int)min((int64_t)a.counts[e], a.routes - off);
    } else {
      jt = item / nib;
      ib = item - jt * nib;
      e = a.te[jt];
      count = min(a.tc[jt], BJ);
      off = a.to[jt];
      if (count <= 0 || off < 0 || off + count > a.routes) return;
      if (e < 0 || e >= a.E) e = -1;
    }
  }
  const int64_t i0 = ib * BI, j0 = MODE == DG_WEIGHT ? jt * BJ : 0;
  const int64_t kn = MODE == DG_WEIGHT ? count : a.nk;
  const int steps = e < 0 ? 0 : (int)((kn + DG_K - 1) / DG_K);

  // ---- the copies of a step
  const T* wbase = (const T*)a.w + (MODE == DG_WEIGHT || e < 0 ? 0 : e * a.ni * a.nk);
  const char* pi[TRI ? 1 : LI];  // FORWARD: this thread's rows of W
  const char* pj[TRJ ? 1 : LJ];  // FORWARD, TRANS: this thread's rows of x
  if constexpr (!TRI) {
#pragma unroll
    for (int i = 0; i < LI; ++i) {
      const int L = tid + i * NT, row = L >> 3, s = (L & 7) ^ dg_swz_i(row);
      pi[i] = (const char*)(wbase + min(i0 + row, a.ni - 1) * a.nk + s * 8);
    }
  }
  if constexpr (!TRJ) {
#pragma unroll
    for (int i = 0; i < LJ; ++i) {
      const int L = tid + i * NT, row = L >> 3, s = (L & 7) ^ dg_swz_j(row);
      const int64_t r = a.order[off + min(row, count - 1)];
      int64_t xr = a.lhs ? (int64_t)a.lhs[r] : (int64_t)((uint32_t)r / (uint32_t)a.x_div);
      if (xr < 0 || xr >= a.x_rows) xr = 0;
      pj[i] = (const char*)((const T*)a.x + xr * a.nk + s * 8);
    }
  }
  // WEIGHT: the routes of this thread's copies in the next step (-1: past the expert's last)
  constexpr int RI = BI / 8, RJ = BJ / 8;  // 16-byte slots of a transposed row
  int ri[TRJ ? LI : 1], rj[TRJ ? LJ : 1];
  auto fetch = [&](int step) {
    if constexpr (TRJ) {
#pragma unroll
      for (int i = 0; i < LI; ++i) {
        const int at = step * DG_K + (tid + i * NT) / RI;
        ri[i] = at < count ? a.order[off + at] : -1;
      }
#pragma unroll
      for (int i = 0; i < LJ; ++i) {
        const int at = step * DG_K + (tid + i * NT) / RJ;
        rj[i] = at < count ? a.order[off + at] : -1;
      }
    }
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wv * 1024;
  auto issue = [&](int step, int buf) {
    const uint32_t bi = lds0 + buf * (SI + SJ), bj = bi + SI;
    const bool tail = (step + 1) * (int64_t)DG_K > kn;
#pragma unroll
    for (int i = 0; i < LI; ++i) {
      const int L = tid + i * NT;
      const void* g;
      if constexpr (!TRI) {
        const int s = (L & 7) ^ dg_swz_i(L >> 3);
        g = tail && step * (int64_t)DG_K + s * 8 >= a.nk ? (const void*)&g_zero16 : pi[i] + (int64_t)step * (DG_K * 2);
      } else {
        const int row = L / RI, sl = L % RI;
        const int64_t col = i0 + (((sl >> 1) ^ dg_swz_t<BI>(row)) * 2 + (sl & 1)) * 8;
        if constexpr (MODE == DG_TRANS) {
          const int64_t k = (int64_t)step * DG_K + row;
          g = col < a.ni && k < a.nk ? (const void*)(wbase + k * a.ni + col) : (const void*)&g_zero16;
        } else {
          const int64_t xr = (uint32_t)ri[i] / (uint32_t)a.x_div;
          g = col < a.ni && ri[i] >= 0 && xr < a.x_rows ? (const void*)((const T*)a.x + xr * a.ni + col)
                                                        : (const void*)&g_zero16;
        }
      }
      dg_dma(g, bi + i * (NT * 16));
    }
#pragma unroll
    for (int i = 0; i < LJ; ++i) {
      const int L = tid + i * NT;
      const void* g;
      if constexpr (!TRJ) {
        const int s = (L & 7) ^ dg_swz_j(L >> 3);
        g = tail && step * (int64_t)DG_K + s * 8 >= a.nk ? (const void*)&g_zero16 : pj[i] + (int64_t)step * (DG_K * 2);
      } else {
        const int row = L / RJ, sl = L % RJ;
        const int64_t col = j0 + (((sl >> 1) ^ dg_swz_t<BJ>(row)) * 2 + (sl & 1)) * 8;
        g = col < a.nj && rj[i] >= 0 && rj[i] < a.routes ? (const void*)((const T*)a.w + (int64_t)rj[i] * a.nj + col)
                                                        : (const void*)&g_zero16;
      }
      dg_dma(g, bj + i * (NT * 16));
    }
  };

  f4 acc[FJ][FI];
#pragma unroll
  for (int j = 0; j < FJ; ++j)
#pragma unroll
    for (int i = 0; i < FI; ++i) acc[j][i] = f4{0.f, 0.f, 0.f, 0.f};
  if (steps > 0) {
    fetch(0);
    issue(0, 0);
    fetch(1);
  }
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this step's copies
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();        // everybody's, and nobody reads the other buffer any more
    asm volatile("" ::: "memory");
    if (s + 1 < steps) {
      issue(s + 1, (s + 1) & 1);
      fetch(s + 2);
    }
    const char* bi = smem + (s & 1) * (SI + SJ);
    const char* bj = bi + SI;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      uint4 fi[FI], fj[FJ];
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        // results of fragments 4 g + u are columns 64 g + 16 q + 4 u + v
        if constexpr (TRI) fi[i] = dg_frag_t<BI>(bi, wi * FI + i, ks, lane);
        else fi[i] = dg_frag<1>(bi, wi * TI + (i >> 2) * 64 + (c >> 2) * 16 + (i & 3) * 4 + (c & 3), ks, q);
      }
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        if constexpr (TRJ) fj[j] = dg_frag_t<BJ>(bj, wj * FJ + j, ks, lane);
        else fj[j] = dg_frag<0>(bj, wj * TJ + j * 16 + c, ks, q);
      }
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int i = 0; i < FI; ++i) acc[j][i] = dense_mfma<T>(fi[i], fj[j], acc[j][i]);
    }
  }

  // ---- results: row j (route or n) of this lane, columns as above (TRANS, WEIGHT: 16 i + 4 q + v)
  const bool wide = a.wide;
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int row = wj * TJ + j * 16 + c;
    int64_t at;
    bool ok = true;
    if constexpr (MODE == DG_WEIGHT) {
      if (j0 + row >= a.nj) continue;
      at = (e * a.nj + j0 + row) * a.ni;
    } else {
      if (row >= count) continue;
      const int64_t r = a.order[off + row];
      const int64_t xr = a.lhs ? (int64_t)a.lhs[r] : (int64_t)((uint32_t)r / (uint32_t)a.x_div);
      ok = e >= 0 && xr >= 0 && xr < a.x_rows;
      at = r * a.ni;
    }
    if constexpr (!TRI) {
#pragma unroll
      for (int g = 0; g < FI / 4; ++g) {
        const int64_t col = i0 + wi * TI + g * 64 + q * 16;
        if (col >= a.ni) continue;
        float f[16];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int v = 0; v < 4; ++v) f[4 * u + v] = ok ? acc[j][4 * g + u][v] : __builtin_nanf("");
        if (a.odt == KEEP_F32) dense_st<float, 16>((float*)a.out + at + col, a.ni - col, f, wide);
        else dense_st<T, 16>((T*)a.out + at + col, a.ni - col, f, wide);
      }
    } else {
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int64_t col = i0 + wi * TI + i * 16 + q * 4;
        if (col >= a.ni) continue;
        float f[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) f[v] = ok ? acc[j][i][v] : __builtin_nanf("");
        if (a.odt == KEEP_F32) dense_st<float, 4>((float*)a.out + at + col, a.ni - col, f, wide);
        else dense_st<T, 4>((T*)a.out + at + col, a.ni - col, f, wide);
      }
    }
  }
}

template <typename T, int BI, int BJ, int WI, int WJ, int MODE>
static void dg_launch(const DenseGemmArgs& a, hipStream_t s) {
  const int64_t nib = (a.ni + BI - 1) / BI;
  const int64_t items = MODE == DG_WEIGHT ? a.E * ((a.nj + BJ - 1) / BJ) * nib : a.max_tiles * nib;
  const dim3 grid((unsigned)((items + 7) / 8 * 8));
  hipLaunchKernelGGL((k_dense_gemm<T, BI, BJ, WI, WJ, MODE>), grid, dim3(64 * WI * WJ), 0, s, a);
}

template <typename T, int MODE>
static void dg_rows(const DenseGemmArgs& a, int64_t tile, hipStream_t s) {
  if (tile == 64) dg_launch<T, 256, 64, 4, 1, MODE>(a, s);
  else if (tile == 128) dg_launch<T, 128, 128, 2, 2, MODE>(a, s);
  else dg_launch<T, 256, 256, 4, 2, MODE>(a, s);
}

bool dense_gemm_tile(int64_t tile) { return tile == 64 || tile == 128 || tile == 256; }

int dense_gemm_rows(const DenseGemmArgs& a, int dtype, bool transposed, int64_t tile, hipStream_t s) {
  if (dtype == KEEP_F16) {
    if (transposed) dg_rows<_Float16, DG_TRANS>(a, tile, s);
    else dg_rows<_Float16, DG_FORWARD>(a, tile, s);
  } else {
    if (transposed) dg_rows<bf16s, DG_TRANS>(a, tile, s);
    else dg_rows<bf16s, DG_FORWARD>(a, tile, s);
  }
  return launch_status("keep_gather_mm");
}

int dense_gemm_weight(const DenseGemmArgs& a, int dtype, hipStream_t s) {
  if (dtype == KEEP_F16) dg_launch<_Float16, 128, 128, 2, 2, DG_WEIGHT>(a, s);
  else dg_launch<bf16s, 128, 128, 2, 2, DG_WEIGHT>(a, s);
  return launch_status("keep_gather_mm_grad_weight");
}

}  // namespace keep
