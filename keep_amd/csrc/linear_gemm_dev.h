#pragma once
// Products of two dense matrices through LDS: the dense projection and its gradients.
//
//   FORWARD  out[m][n] = sum_k x[m][k] W[n][k], then the epilogue   both sides run along the summed index
//   ROWS     dx[m][k] = sum_n du[m][n] W[n][k]                      W across it
//   WEIGHT   dW[n][k] = sum_m du[m][n] x[m][k]                      both across it
//
// The side whose index is contiguous in the output is "I", the first MFMA operand (dense_dev.h), the other "J". A step sums
// 128 bytes of a row: 64 16-bit values, 32 floats, 128 8-bit ones. Its operands are copied to LDS by the DMA path into one of
// two buffers while the matrix cores work on the other; one barrier a step. Where there are few tiles G groups of waves of a
// block take a part of the summed index each, in buffers of their own, and their sums are added in LDS; where there are fewer
// still it is cut into slices too, whose float32 sums k_linear_join adds. Both in order.
//
// Bound by the matrix cores' power and by LDS: 8192 x 8192 x 8192 bf16 1372 TFLOP/s, 8192 x 4096 -> 8192 with silu 410 to 436 us
// (1340 to 1260 TFLOP/s), during which the clock falls to about 1.8 GHz: a step's products take 2048 clocks of a SIMD, 62 % of
// what a step takes, and four buffers for two, which cut the waits, left the time as it was. 4096 x 4096 -> 2048 (256 tiles of 256 x 128, one
// a CU) 73 us with its epilogue, 65 for dx and 68 for dW: a step of this tile reads 128 KB of LDS and writes 48 for 1024 clocks
// of products, and a tile's first copies and its stores are not overlapped. float32 (16x16x4 products) 142 TFLOP/s of 157.
//
// 8-bit values (e4m3) come with a scale per 128 of a row of x and per 128 x 128 of W: a step is one scale's span, so its
// products start from zero and enter the sums times both scales, one multiply-add a value. 4096 x 7168 -> 2048 115 us, 1045
// TFLOP/s by either tile; with conversions and scaling spread between the products it took 117.
#include <algorithm>
#include <type_traits>

#include "dense_lds.h"
#include "linear_dev.h"

namespace keep {

__device__ __attribute__((aligned(16))) static uint4 g_linear_zero;

// Group permutation of a transposed float operand: the four quarters of a fragment read rows 4 q + s of one s at a time.
__device__ __forceinline__ int lg_swz_tf(int row) { return (row >> 2) & 3; }

// Column 16 ct + c of a transposed float operand of COLS columns: values of rows 4 q .. 4 q + 3 of half step ks.
template <int COLS>
__device__ __forceinline__ uint4 lg_frag_tf(const char* s, int ct, int ks, int lane) {
  const int q = lane >> 4, c = lane & 15;
  const int row = ks * 16 + q * 4;
  const uint32_t* p = (const uint32_t*)(s + row * (4 * COLS) + (((ct ^ lg_swz_tf(row)) * 16 + c) * 4));
  return make_uint4(p[0], p[COLS], p[2 * COLS], p[3 * COLS]);
}

template <typename T>
struct LinearStep {
  static constexpr int V = 16 / sizeof(T);   // values of a 16-byte slot
  static constexpr int K = 128 / sizeof(T);  // summed values of a step
};

// TAIL: the summed index may end inside the last step. (The choice costs every copy of the loop a branch, 8 % of a step.)
template <typename T, int BI, int BJ, int WI, int WJ, int G, int MODE, bool TAIL>
__global__ __launch_bounds__(64 * WI * WJ * G) void k_linear_gemm(LinearGemmArgs a) {
  constexpr int NT = 64 * WI * WJ, TI = BI / WI, TJ = BJ / WJ, FI = TI / 16, FJ = TJ / 16;
  constexpr int LI = BI * 8 / NT, LJ = BJ * 8 / NT;  // 16-byte copies per thread and step
  constexpr int SI = BI * 128, SJ = BJ * 128;        // bytes of a buffer's operands
  constexpr int V = LinearStep<T>::V, KS = LinearStep<T>::K, SZ = sizeof(T);
  constexpr bool TRI = MODE != LINEAR_FORWARD, TRJ = MODE == LINEAR_WEIGHT;
  constexpr bool Q8 = sizeof(T) == 1;
  static_assert(!Q8 || MODE == LINEAR_FORWARD, "8-bit values have no gradient");
  constexpr int FP = FJ > 4 ? 4 : FJ, ROWS = WJ * FP * 16, PITCH = BI + 4, CG = BI / 8;
  constexpr int LDS = G * 2 * (SI + SJ) > G * ROWS * PITCH * 4 ? G * 2 * (SI + SJ) : G * ROWS * PITCH * 4;
  __shared__ __attribute__((aligned(16))) char smem_all[LDS];
  const int gr = G > 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT) : 0;  // group
  char* smem = smem_all + gr * (2 * (SI + SJ));
  const int tid = threadIdx.x - gr * NT, lane = tid & 63, c = lane & 15, q = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wv % WI, wj = wv / WI;

  // ---- work item (slice, j tile, i tile): items go to the XCDs in contiguous runs; inside a slice, groups of up to 8 j
  // tiles are walked i tile by i tile, so that the items that an XCD's CUs work on share operands
  const uint32_t nib = (uint32_t)((a.ni + BI - 1) / BI), njb = (uint32_t)((a.nj + BJ - 1) / BJ);
  const uint32_t total = nib * njb * (uint32_t)a.slices, per = (total + 7) / 8;
  const uint32_t item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || item >= total) return;
  const uint32_t slice = item / (nib * njb), rem = item - slice * (nib * njb);
  const uint32_t group = rem / (8 * nib), in = rem - group * (8 * nib), rows = min(8u, njb - group * 8);
  const uint32_t ib = in / rows, jb = group * 8 + in - ib * rows;
  const int64_t i0 = (int64_t)ib * BI, j0 = (int64_t)jb * BJ;
  const int count = (int)min((int64_t)BJ, a.nj - j0);
  const int all = (int)((a.nk + KS - 1) / KS), each = (all + a.slices - 1) / a.slices;
  const int b0 = min(all, (int)slice * each), b1 = min(all, b0 + each);
  const int turns = (b1 - b0 + G - 1) / G;  // steps of a group; the last ones may have fewer
  const int s0 = min(b1, b0 + gr * turns), s1 = min(b1, s0 + turns);

  // ---- copies of a step. Common case: 32-bit offsets off a base that moves on with the steps. In the last step of a summed
  // index that ends inside it, an address per lane, past the end that of a zero. Rows and columns past the last repeat it:
  // their results are not stored.
  constexpr int RI = BI * SZ / 16, RJ = BJ * SZ / 16;  // 16-byte slots of a transposed row
  const auto col_t = [](int L, int R, int groups) -> int {  // first column of slot L of a transposed operand
    const int row = L / R, sl = L % R;
    if constexpr (SZ == 4) return (((sl >> 2) ^ lg_swz_tf(row)) * 4 + (sl & 3)) * 4;
    else return (((sl >> 1) ^ (((row & 3) | (((row >> 3) & 1) << 2)) & (groups - 1))) * 2 + (sl & 1)) * 8;
  };
  uint32_t oi[LI], oj[LJ];
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int L = tid + i * NT;
    if constexpr (!TRI) {
      const int row = L >> 3;
      oi[i] = (uint32_t)((min(i0 + row, a.ni - 1) - i0) * a.ldi * SZ) + ((L & 7) ^ dg_swz_j(row)) * 16;
    } else {
      const int64_t last = (a.ni + V - 1) / V * V - V;
      oi[i] = (uint32_t)(((L / RI) * a.ldi + min(i0 + col_t(L, RI, BI / 16), last)) * SZ);
    }
  }
#pragma unroll
  for (int i = 0; i < LJ; ++i) {
    const int L = tid + i * NT;
    if constexpr (!TRJ) {
      const int row = L >> 3;
      oj[i] = (uint32_t)(min(row, count - 1) * a.ldj * SZ) + ((L & 7) ^ dg_swz_j(row)) * 16;
    } else {
      const int64_t last = (a.nj + V - 1) / V * V - V;
      oj[i] = (uint32_t)(((L / RJ) * a.ldj + min(j0 + col_t(L, RJ, BJ / 16), last)) * SZ);
    }
  }
  const char* ibase = (const char*)a.pi + (TRI ? 0 : i0 * a.ldi * SZ);
  const char* jbase = (const char*)a.pj + (TRJ ? 0 : j0 * a.ldj * SZ);
  const int64_t istep = TRI ? (int64_t)KS * a.ldi * SZ : 128, jstep = TRJ ? (int64_t)KS * a.ldj * SZ : 128;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wv * 1024;
  // copy i of the step (the I side's first)
  const auto copy = [&](int i, int step, bool part) {
    const uint32_t to = lds0 + (step & 1) * (SI + SJ) + i * (NT * 16);
    const bool jside = i >= LI;
    if (jside && part && !TRJ && (wv * 64 + (i - LI) * NT) / 8 >= count) return;  // rows past the last: not stored
    const char* base = jside ? jbase + step * jstep : ibase + step * istep;
    const uint32_t o = jside ? oj[jside ? i - LI : 0] : oi[jside ? 0 : i];
    if (!TAIL || (int64_t)(step + 1) * KS <= a.nk) {
      dg_dma(base, o, to);
    } else {
      int L = tid + (jside ? i - LI : i) * NT;
      asm volatile("" : "+v"(L));  // made here, not kept over the loop
      const bool tr = jside ? TRJ : TRI;
      const int64_t k = (int64_t)step * KS + (tr ? L / (jside ? RJ : RI)
                                                 : ((L & 7) ^ dg_swz_j(L >> 3)) * V);
      dg_dma(k < a.nk ? (const void*)(base + o) : (const void*)&g_linear_zero, to);
    }
  };

  f4 acc[FJ][FI];
#pragma unroll
  for (int j = 0; j < FJ; ++j)
#pragma unroll
    for (int i = 0; i < FI; ++i) acc[j][i] = f4{0.f, 0.f, 0.f, 0.f};
  const auto read = [&](int n, int step, int ks) -> uint4 {  // fragment n, the I side's first
    const char* bi = smem + (step & 1) * (SI + SJ);
    const char* bj = bi + SI;
    if (n < FI) {
      if constexpr (!TRI) return dg_frag<0>(bi, wi * TI + n * 16 + c, ks, q);
      else if constexpr (SZ == 4) return lg_frag_tf<BI>(bi, wi * FI + n, ks, lane);
      else return dg_frag_t<BI>(bi, wi * FI + n, ks, lane);
    } else {
      n -= FI;
      if constexpr (!TRJ) return dg_frag<0>(bj, wj * TJ + n * 16 + c, ks, q);
      else if constexpr (SZ == 4) return lg_frag_tf<BJ>(bj, wj * FJ + n, ks, lane);
      else return dg_frag_t<BJ>(bj, wj * FJ + n, ks, lane);
    }
  };
  constexpr int NR = FI + FJ, NC = LI + LJ;
  const int live = max(0, min(FJ, (count - wj * TJ + 15) / 16));  // this wave's fragments that hold rows
  const auto landed = [&]() {  // this wave's reads are done and its copies landed, then everybody's
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // PART: a tile with fewer rows than BJ leaves out the copies and products of fragments without rows
  const auto sum = [&](auto part_c) {
    constexpr bool PART = decltype(part_c)::value;
    if constexpr (Q8) {
      const int64_t kb = (a.nk + 127) / 128;
      const float* si = a.si + (int64_t)(min(i0 + wi * TI, a.ni - 1) / 128) * kb;
      const float* sj[FJ];
#pragma unroll
      for (int j = 0; j < FJ; ++j) sj[j] = a.sj + (j0 + min(wj * TJ + j * 16 + c, count - 1)) * kb;
      if (s0 < s1) {
#pragma unroll
        for (int i = 0; i < NC; ++i) copy(i, s0, PART);
      }
      float xs[FJ], ws = s0 < s1 ? si[s0] : 0.f;
#pragma unroll
      for (int j = 0; j < FJ; ++j) xs[j] = s0 < s1 ? sj[j][s0] : 0.f;
      landed();
      for (int turn = 0; turn < turns; ++turn) {
        const int s = s0 + turn;
        if (G > 1 && s >= s1) {
          landed();
          continue;
        }
        float nxs[FJ], nws = ws;
        if (s + 1 < s1) {  // into the other buffer, which everybody has read
          nws = si[s + 1];
#pragma unroll
          for (int j = 0; j < FJ; ++j) nxs[j] = sj[j][s + 1];
#pragma unroll
          for (int i = 0; i < NC; ++i) copy(i, s + 1, PART);
        } else {
#pragma unroll
          for (int j = 0; j < FJ; ++j) nxs[j] = xs[j];
        }
        linear_h8 fi[FI][4];
#pragma unroll
        for (int i = 0; i < FI; ++i) linear_e4m3(read(i, s, 0), read(i, s, 1), fi[i]);
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
          if (PART && j >= live) continue;
          linear_h8 fj[4];
          linear_e4m3(read(FI + j, s, 0), read(FI + j, s, 1), fj);
          f4 p[FI];
#pragma unroll
          for (int i = 0; i < FI; ++i) p[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < FI; ++i) p[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fi[i][t], fj[t], p[i], 0, 0, 0);
          const float scale = xs[j] * ws;
#pragma unroll
          for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[j][i][v] = fmaf(p[i][v], scale, acc[j][i][v]);
        }
        landed();
        ws = nws;
#pragma unroll
        for (int j = 0; j < FJ; ++j) xs[j] = nxs[j];
      }
    } else {
      // half a step at a time; the next half's fragments are read while this one's products run, and the copies of the step
      // after next start with the second half
      struct Half {
        uint4 f[NR];
      };
      constexpr int CC = (NC + FJ - 1) / FJ;  // copies per group of products
      const auto half = [&](const Half& use, Half& next, int nstep, int nks, bool copies, int cstep) {
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
          if (copies) {
#pragma unroll
            for (int i = j * CC; i < (j + 1) * CC && i < NC; ++i) copy(i, cstep, PART);
          }
#pragma unroll
          for (int n = j * NR / FJ; n < (j + 1) * NR / FJ; ++n) next.f[n] = read(n, nstep, nks);
          if (!PART || j < live)
#pragma unroll
            for (int i = 0; i < FI; ++i) acc[j][i] = dense_mfma<T>(use.f[i], use.f[FI + j], acc[j][i]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      Half h0, h1;
      if (G == 1 || s0 < s1) {
#pragma unroll
        for (int i = 0; i < NC; ++i) copy(i, s0, PART);
      }
      landed();
      if (s0 + 1 < s1) {
#pragma unroll
        for (int i = 0; i < NC; ++i) copy(i, s0 + 1, PART);
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) h0.f[n] = read(n, s0, 0);
      for (int turn = 0; turn < turns; ++turn) {
        const int s = s0 + turn;
        if (G == 1 || s < s1) half(h0, h1, s, 1, false, 0);
        landed();  // step s is read by everybody, step s + 1 is there
        // (after the last step h0 takes the buffer's old bytes, not used)
        if (G == 1 || s < s1) half(h1, h0, s + 1, 0, s + 2 < s1, s + 2);
      }
    }
  };
  if (turns > 0) {
    if (TRJ || count == BJ) sum(std::false_type{});
    else if constexpr (!TRJ) sum(std::true_type{});
  }

  // ---- results, through LDS: a lane's columns of a row are few and its rows many, a thread of the epilogue takes eight
  // neighbouring columns, so that a row's pieces lie together in memory. FP fragments of every wave at a time: four of the largest tile's
  // eight (8192 x 128 -> 8192 bf16 65 us, by two 70; 8192 x 4096 -> 8192 407, 417), two where there are four (of four 1 % slower).
  static_assert(FJ % FP == 0 && NT % CG == 0, "LDS");
  float* tile = (float*)smem_all + gr * (ROWS * PITCH);
  const int64_t col = i0 + (tid % CG) * 8;
  float b[8];
  a.e.load_bias<8>(col, a.ni - col, b);
#pragma unroll
  for (int p = 0; p < FJ / FP; ++p) {
    __syncthreads();
#pragma unroll
    for (int jj = 0; jj < FP; ++jj) {
      float* row = tile + ((wj * FP + jj) * 16 + c) * PITCH + wi * TI;
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const f4 r = acc[p * FP + jj][i];
        *(float4*)(row + i * 16 + q * 4) = make_float4(r[0], r[1], r[2], r[3]);
      }
    }
    __syncthreads();
    if (col >= a.ni) continue;
#pragma unroll 4
    for (int r = threadIdx.x / CG; r < ROWS; r += G * NT / CG) {
      const int64_t row = j0 + (r / (FP * 16)) * TJ + p * (FP * 16) + r % (FP * 16);
      if (row >= a.nj) continue;
      const float* from = (const float*)smem_all + r * PITCH + (tid % CG) * 8;
      float f[8];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float4 lo = *(const float4*)(from + g * (ROWS * PITCH)), hi = *(const float4*)(from + g * (ROWS * PITCH) + 4);
        const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int u = 0; u < 8; ++u) f[u] = g == 0 ? v[u] : f[u] + v[u];
      }
      if (a.slices > 1)
        dense_st<float, 8>(a.part + ((int64_t)slice * a.nj + row) * a.ni + col, a.ni - col, f, a.ni % 4 == 0);
      else
        a.e.store<8>(row, a.ni, col, a.ni - col, f, b);
    }
  }
}

template <typename T, int BI, int BJ, int WI, int WJ, int G, int MODE>
void linear_gemm_launch(const LinearGemmArgs& a, hipStream_t s) {
  const int64_t items = ((a.ni + BI - 1) / BI) * ((a.nj + BJ - 1) / BJ) * a.slices;
  const dim3 grid((unsigned)((items + 7) / 8 * 8)), block(64 * WI * WJ * G);
  if (a.nk % LinearStep<T>::K == 0)
    hipLaunchKernelGGL((k_linear_gemm<T, BI, BJ, WI, WJ, G, MODE, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_linear_gemm<T, BI, BJ, WI, WJ, G, MODE, true>), grid, block, 0, s, a);
}

template <typename T, int MODE>
void linear_gemm_tile(const LinearGemmArgs& a, int tile, hipStream_t s) {
  if (tile == LINEAR_TILE_64) linear_gemm_launch<T, 64, 64, 2, 2, 2, MODE>(a, s);
  else if (tile == LINEAR_TILE_128_2) linear_gemm_launch<T, 128, 128, 2, 2, 2, MODE>(a, s);
  else if (sizeof(T) == 4 || tile == LINEAR_TILE_128) linear_gemm_launch<T, 128, 128, 2, 2, 1, MODE>(a, s);
  else if constexpr (sizeof(T) < 4) {
    if (sizeof(T) == 1 || tile == LINEAR_TILE_256_128) linear_gemm_launch<T, 256, 128, 4, 2, 1, MODE>(a, s);
    else if constexpr (sizeof(T) == 2) linear_gemm_launch<T, 256, 256, 4, 2, 1, MODE>(a, s);
  }
}

template <typename T>
void linear_gemm_mode(const LinearGemmArgs& a, int mode, int tile, hipStream_t s) {
  if constexpr (sizeof(T) == 1) {
    linear_gemm_tile<T, LINEAR_FORWARD>(a, tile, s);
  } else {
    if (mode == LINEAR_FORWARD) linear_gemm_tile<T, LINEAR_FORWARD>(a, tile, s);
    else if (mode == LINEAR_ROWS) linear_gemm_tile<T, LINEAR_ROWS>(a, tile, s);
    else linear_gemm_tile<T, LINEAR_WEIGHT>(a, tile, s);
  }
}

}  // namespace keep
