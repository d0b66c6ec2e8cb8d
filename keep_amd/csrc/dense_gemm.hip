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
//
// A step of a 256 x 256 tile is 512 products of 16 clocks on four SIMDs, 2048
// clocks (0.85 us at 2.4 GHz), and its 64 KiB of copies and 192 KiB of fragments
// (each read by two or four waves, half a step ahead of its products, without
// bank conflicts) are as many clocks of LDS at 128 bytes each. Measured, a step
// takes 1.6 us: waves wait 32 to 44 % of their cycles. First copies and stores
// add 10 to 14 us a tile: 115 us for 4096 summed values. bf16: 8192 x 8192 x 8192
// forward 848 us (1297 TFLOP/s), dx 865 to 907, dW 1013; 65536 routes of 32
// experts, 4096 -> 2048, 1039 to 1058 us (1058 to 1039 TFLOP/s). The last round
// of tiles fills part of the CUs.
// Eight waves of 64 x 128 results each and four of 128 x 128 hold the same tile:
// the eight hide each other's waits. Tiles in turn on a resident workgroup, the
// next one's copies under the stores, took 66 to 86 registers more than there are.
// Below about 48 routes an expert the weights' bytes bound it: 256 x 64 tiles
// stream 384 experts of 4096 -> 2048 (6.4 GB) in 1.1 to 1.23 ms, 5.3 to 5.8 TB/s.
#include <algorithm>
#include <type_traits>

#include "dense_dev.h"
#include "dense_gemm.h"
#include "dense_lds.h"

namespace keep {

__device__ __attribute__((aligned(16))) uint4 g_zero16;

constexpr int DG_K = 64;  // summed index per step

enum { DG_FORWARD = 0, DG_TRANS = 1, DG_WEIGHT = 2 };

// r / x_div for 0 <= r < 2^31: (2 r m) >> (32 + l) with l = ceil(log2 x_div), m = ceil(2^(31 + l) / x_div), exact since
// m x_div - 2^(31 + l) < x_div <= 2^l.
__device__ __forceinline__ int64_t dg_row(const DenseGemmArgs& a, int r) {
  return (int64_t)(__umulhi(2u * (uint32_t)r, a.div_mul) >> a.div_shift);
}

// Row tiles that an XCD takes in turn (0: a contiguous run of all items). With few routes an expert most tiles read weights
// of their own, and an XCD whose run has experts of several tiles is done early: 384 experts of 4096 -> 2048, 8192 routes
// 1213 us in runs, 1110 in turns of 2 (1, 4: the same); 12288 routes of Zipf popularity 1293 against 1226; 64 experts of
// 2048 -> 768 38.5 against 40. Large tiles share operands with their neighbours instead (128: 384 experts 1597 against 1440,
// 256 experts 870 against 944, the same elsewhere).
constexpr int dg_turn(int bj) { return bj == 64 ? 2 : 0; }

template <typename T, int BI, int BJ, int WI, int WJ, int MODE>
__global__ __launch_bounds__(64 * WI * WJ) void k_dense_gemm(DenseGemmArgs a) {
  constexpr int NT = 64 * WI * WJ, TI = BI / WI, TJ = BJ / WJ, FI = TI / 16, FJ = TJ / 16;
  constexpr int LI = BI * 8 / NT, LJ = BJ * 8 / NT;  // 16-byte copies per thread and step
  constexpr int SI = BI * 128, SJ = BJ * 128;        // bytes of a buffer's operands
  constexpr bool TRI = MODE != DG_FORWARD, TRJ = MODE == DG_WEIGHT;
  constexpr int G = dg_turn(BJ);
  __shared__ __attribute__((aligned(16))) char smem[2 * (SI + SJ)];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wv % WI, wj = wv / WI;

  // work item: (j tile or expert and row block, i block)
  int64_t e;
  uint32_t jt, ib;
  int count = 0;
  int64_t off = 0;
  {
    const uint32_t nib = (uint32_t)((a.ni + BI - 1) / BI);
    uint32_t total, ntiles = 0;
    if constexpr (MODE == DG_WEIGHT) {
      total = (uint32_t)a.E * (uint32_t)((a.nj + BJ - 1) / BJ) * nib;
    } else {
      // tiles of valid experts; those of invalid routes follow
      const int64_t valid = (int64_t)a.offsets[a.E - 1] + a.counts[a.E - 1];
      ntiles = (uint32_t)min(a.n_tiles[0] + (a.routes - valid + BJ - 1) / BJ, a.max_tiles);
      total = ntiles * nib;
    }
    const uint32_t slot = blockIdx.x >> 3, xcd = blockIdx.x & 7;
    uint32_t item = 0;  // dealt to the XCDs in contiguous runs, or in turns of G row tiles
    if constexpr (G == 0) {
      const uint32_t per = (total + 7) / 8;
      item = xcd * per + slot;
      if (slot >= per || item >= total) return;
    }
    if constexpr (MODE == DG_WEIGHT) {
      const uint32_t njb = (uint32_t)((a.nj + BJ - 1) / BJ), ex = item / (njb * nib), r = item - ex * (njb * nib);
      jt = r / nib;
      ib = r - jt * nib;
      e = ex;
      off = a.offsets[ex];
      count = (int)max((int64_t)0, min((int64_t)a.counts[ex], a.routes - off));
    } else {
      // groups of up to 8 row tiles, within a group column block by column block: the 32 items that an XCD's CUs work on
      // share 8 + 4 operand blocks where N is wide
      if constexpr (G == 0) {
        const uint32_t group = item / (8 * nib), in = item - group * (8 * nib), rows = min(8u, ntiles - group * 8);
        ib = in / rows;
        jt = group * 8 + in - ib * rows;
      } else {
        const uint32_t turn = slot / (G * nib), in = slot - turn * (G * nib), j = (turn * 8 + xcd) * G;
        if (j >= ntiles) return;
        const uint32_t rows = min((uint32_t)G, ntiles - j);
        ib = in / rows;
        jt = j + in - ib * rows;
        if (ib >= nib) return;
      }
      e = a.te[jt];
      count = min(a.tc[jt], BJ);
      off = a.to[jt];
      if (count <= 0 || off < 0 || off + count > a.routes) return;
      if (e < 0 || e >= a.E) e = -1;
    }
  }
  const int64_t i0 = (int64_t)ib * BI, j0 = MODE == DG_WEIGHT ? (int64_t)jt * BJ : 0;
  const int64_t kn = MODE == DG_WEIGHT ? count : a.nk;
  const int steps = e < 0 ? 0 : (int)((kn + DG_K - 1) / DG_K);

  // ---- the copies of a step. Common case: 32-bit offsets off a base that moves on with the steps. The last step of a
  // summed index that is no multiple of 64, and operands of 4 GiB and more, take an address per lane, past the end that of
  // a zero. Columns past the output's are copies of its last ones: their results are not stored.
  const T* wbase = (const T*)a.w + (MODE == DG_WEIGHT || e < 0 ? 0 : e * a.ni * a.nk);
  constexpr int RI = BI / 8, RJ = BJ / 8;  // 16-byte slots of a transposed row
  auto col_t = [&](int L, bool jside) -> int64_t {  // first column of slot L of a transposed operand
    const int R = jside ? RJ : RI, row = L / R, sl = L % R;
    const int swz = jside ? dg_swz_t<BJ>(row) : dg_swz_t<BI>(row);
    return (((sl >> 1) ^ swz) * 2 + (sl & 1)) * 8;
  };
  auto x_row = [&](int row) -> int64_t {  // of the tile's row; rows past the last repeat it
    const int64_t r = a.order[off + min(row, count - 1)];
    const int64_t xr = a.lhs ? (int64_t)a.lhs[r] : dg_row(a, (int)r);
    return xr < 0 || xr >= a.x_rows ? 0 : xr;
  };
  uint32_t oi[LI], oj[LJ];  // offsets in bytes (WEIGHT: of the columns alone)
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int L = tid + i * NT;
    if constexpr (!TRI) {
      const int row = L >> 3;
      oi[i] = (uint32_t)((min(i0 + row, a.ni - 1) - i0) * a.nk + ((L & 7) ^ dg_swz_i(row)) * 8) * 2u;
    } else {
      const int64_t col = min(i0 + col_t(L, false), a.ni - 8);
      oi[i] = (uint32_t)((MODE == DG_TRANS ? (int64_t)(L / RI) * a.ni : 0) + col) * 2u;
    }
  }
#pragma unroll
  for (int i = 0; i < LJ; ++i) {
    const int L = tid + i * NT;
    if constexpr (!TRJ) {
      const int row = L >> 3;
      oj[i] = (uint32_t)(x_row(row) * a.nk + ((L & 7) ^ dg_swz_j(row)) * 8) * 2u;
    } else {
      oj[i] = (uint32_t)min(j0 + col_t(L, true), a.nj - 8) * 2u;
    }
  }
  // WEIGHT: the routes of this thread's copies in a step to come (-1: past the expert's last)
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
  const T* ibase = MODE == DG_FORWARD ? wbase + i0 * a.nk : MODE == DG_TRANS ? wbase : (const T*)a.x;
  const T* jbase = MODE == DG_WEIGHT ? (const T*)a.w : (const T*)a.x;
  const int64_t istep = MODE == DG_FORWARD ? DG_K : MODE == DG_TRANS ? DG_K * a.ni : 0;
  const int64_t jstep = MODE == DG_WEIGHT ? 0 : DG_K;
  // copy i of the step (the I side's first)
  auto copy = [&](int i, int step, bool part) {
    const uint32_t to = lds0 + (step & 1) * (SI + SJ) + i * (NT * 16);
    const bool plain = !a.far && (step + 1) * (int64_t)DG_K <= kn;
    if (i < LI) {
      if (plain) {
        uint32_t o = oi[i];
        if constexpr (MODE == DG_WEIGHT) {
          const int64_t xr = dg_row(a, ri[i]);
          o += (uint32_t)min(xr, a.x_rows - 1) * (uint32_t)(a.ni * 2);
        }
        dg_dma(ibase + step * istep, o, to);
      } else {
        int L = tid + i * NT;
        asm volatile("" : "+v"(L));  // the addresses are made here, not kept over the loop
        const void* g;
        if constexpr (MODE == DG_FORWARD) {
          const int row = L >> 3;
          const int64_t k = step * (int64_t)DG_K + ((L & 7) ^ dg_swz_i(row)) * 8;
          g = k < a.nk ? (const void*)(wbase + min(i0 + row, a.ni - 1) * a.nk + k) : (const void*)&g_zero16;
        } else if constexpr (MODE == DG_TRANS) {
          const int64_t k = step * (int64_t)DG_K + L / RI, col = min(i0 + col_t(L, false), a.ni - 8);
          g = k < a.nk ? (const void*)(wbase + k * a.ni + col) : (const void*)&g_zero16;
        } else {
          const int64_t xr = dg_row(a, ri[i]), col = min(i0 + col_t(L, false), a.ni - 8);
          g = ri[i] >= 0 && xr < a.x_rows ? (const void*)((const T*)a.x + xr * a.ni + col) : (const void*)&g_zero16;
        }
        dg_dma(g, to);
      }
    } else {
      i -= LI;
      if (part && (wv * 64 + i * NT) / 8 >= count) return;  // eight rows past the tile's last: their results are not stored
      if (plain) {
        uint32_t o = oj[i];
        if constexpr (MODE == DG_WEIGHT) o += min((uint32_t)rj[i], (uint32_t)(a.routes - 1)) * (uint32_t)(a.nj * 2);
        dg_dma(jbase + step * jstep, o, to);
      } else {
        int L = tid + i * NT;
        asm volatile("" : "+v"(L));  // the addresses are made here, not kept over the loop
        const void* g;
        if constexpr (MODE != DG_WEIGHT) {
          const int64_t k = step * (int64_t)DG_K + ((L & 7) ^ dg_swz_j(L >> 3)) * 8;
          g = k < a.nk ? (const void*)((const T*)a.x + x_row(L >> 3) * a.nk + k) : (const void*)&g_zero16;
        } else {
          const int64_t col = min(j0 + col_t(L, true), a.nj - 8);
          g = rj[i] >= 0 && rj[i] < a.routes ? (const void*)((const T*)a.w + (int64_t)rj[i] * a.nj + col) : (const void*)&g_zero16;
        }
        dg_dma(g, to);
      }
    }
  };

  // ---- products, half a step (32 of the summed index) at a time; the next half's fragments are read while this one's
  // products run, and the copies of the step after next start with the second half
  f4 acc[FJ][FI];
#pragma unroll
  for (int j = 0; j < FJ; ++j)
#pragma unroll
    for (int i = 0; i < FI; ++i) acc[j][i] = f4{0.f, 0.f, 0.f, 0.f};
  struct Half {
    uint4 f[FI + FJ];
  };
  auto read = [&](Half& h, int n, int step, int ks) {  // fragment n, the I side's first
    const char* bi = smem + (step & 1) * (SI + SJ);
    const char* bj = bi + SI;
    if (n < FI) {
      // results of fragments 4 g + u are columns 64 g + 16 q + 4 u + v
      if constexpr (TRI) h.f[n] = dg_frag_t<BI>(bi, wi * FI + n, ks, lane);
      else h.f[n] = dg_frag<1>(bi, wi * TI + (n >> 2) * 64 + (c >> 2) * 16 + (n & 3) * 4 + (c & 3), ks, q);
    } else {
      if constexpr (TRJ) h.f[n] = dg_frag_t<BJ>(bj, wj * FJ + n - FI, ks, lane);
      else h.f[n] = dg_frag<0>(bj, wj * TJ + (n - FI) * 16 + c, ks, q);
    }
  };
  constexpr int NR = FI + FJ, NC = LI + LJ;
  // this wave's fragments that hold rows
  const int live = max(0, min(FJ, (count - wj * TJ + 15) / 16));
  constexpr int CC = (NC * 2 + FJ - 1) / FJ;  // copies per group of products: all in the first half of the groups
  auto half = [&](const Half& use, Half& next, int nstep, int nks, bool copies, int cstep, bool part) {
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      if (copies) {
#pragma unroll
        for (int i = j * CC; i < (j + 1) * CC && i < NC; ++i) copy(i, cstep, part);
      }
#pragma unroll
      for (int n = j * NR / FJ; n < (j + 1) * NR / FJ; ++n) read(next, n, nstep, nks);
      if (!part || j < live)
#pragma unroll
        for (int i = 0; i < FI; ++i) acc[j][i] = dense_mfma<T>(use.f[i], use.f[FI + j], acc[j][i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto landed = [&]() {  // this wave's reads are done and its copies landed, then everybody's
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // PART: a tile with fewer rows than BJ leaves out the copies and products of fragments without rows
  auto sum = [&](auto part_c) {
    constexpr bool PART = decltype(part_c)::value;
    Half h0, h1;
    fetch(0);
#pragma unroll
    for (int i = 0; i < NC; ++i) copy(i, 0, PART);
    fetch(1);
    landed();
    if (steps > 1) {
#pragma unroll
      for (int i = 0; i < NC; ++i) copy(i, 1, PART);
      fetch(2);
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) read(h0, n, 0, 0);
    for (int s = 0; s < steps; ++s) {
      half(h0, h1, s, 1, false, 0, PART);
      landed();  // step s is read by everybody, step s + 1 is there
      // (after the last step h0 takes the buffer's old bytes, not used)
      half(h1, h0, s + 1, 0, s + 2 < steps, s + 2, PART);
      if (s + 2 < steps) fetch(s + 3);
    }
  };
  // the routes of this lane's rows, read before the sums: -1 none, -2 - r a NaN row
  int ro[MODE == DG_WEIGHT ? 1 : FJ];
  if constexpr (MODE != DG_WEIGHT) {
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int row = wj * TJ + j * 16 + c;
      const int r = a.order[off + min(row, count - 1)];
      const int64_t xr = a.lhs ? (int64_t)a.lhs[r] : dg_row(a, r);
      ro[j] = row >= count || r < 0 || r >= a.routes ? -1 : e >= 0 && xr >= 0 && xr < a.x_rows ? r : -2 - r;
    }
  }
  if (steps > 0) {
    if (MODE == DG_WEIGHT || count == BJ) sum(std::false_type{});
    else if constexpr (MODE != DG_WEIGHT) sum(std::true_type{});
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
      if (ro[j] == -1) continue;
      ok = ro[j] >= 0;
      at = (int64_t)(ok ? ro[j] : -2 - ro[j]) * a.ni;
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
static void dg_launch(DenseGemmArgs a, hipStream_t s) {
  int l = 0;
  while ((int64_t(1) << l) < a.x_div) ++l;
  a.div_shift = l;
  a.div_mul = (uint32_t)(((uint64_t(1) << (31 + l)) + a.x_div - 1) / a.x_div);
  const int64_t most = int64_t(1) << 31;  // of 16-bit values (256 rows past a block's first too)
  a.far = MODE == DG_WEIGHT ? a.x_rows * a.ni >= most || a.routes * a.nj >= most
                            : a.x_rows * a.nk >= most || 256 * (MODE == DG_TRANS ? a.ni : a.nk) >= most;
  const int64_t nib = (a.ni + BI - 1) / BI;
  const int64_t items = MODE == DG_WEIGHT ? a.E * ((a.nj + BJ - 1) / BJ) * nib : a.max_tiles * nib;
  constexpr int64_t G = dg_turn(BJ);
  const dim3 grid((unsigned)(G ? (a.max_tiles + 8 * G - 1) / (8 * G) * (8 * G) * nib : (items + 7) / 8 * 8));
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

// Tiles of 256 x 256 where both sides fill three quarters of one (32 experts of 4096 x 2048, 65536 routes: 1178 us against
// 1752 with 128 x 128; 64 of 2048 x 768, 32768 routes: 162 against 203).
int dense_gemm_weight(const DenseGemmArgs& a, int dtype, hipStream_t s) {
  const bool large = a.ni >= 192 && a.nj >= 192;
  if (dtype == KEEP_F16) {
    if (large) dg_launch<_Float16, 256, 256, 4, 2, DG_WEIGHT>(a, s);
    else dg_launch<_Float16, 128, 128, 2, 2, DG_WEIGHT>(a, s);
  } else {
    if (large) dg_launch<bf16s, 256, 256, 4, 2, DG_WEIGHT>(a, s);
    else dg_launch<bf16s, 128, 128, 2, 2, DG_WEIGHT>(a, s);
  }
  return launch_status("keep_gather_mm_grad_weight");
}

}  // namespace keep
