#pragma once
// Operands of the matrix cores in LDS (dense_gemm.hip, linear.hip): 128 bytes of the summed index a row where rows run along
// it, its eight 16-byte slots permuted; rows of the tile's width, their 32-byte pairs permuted, where the summed index runs
// across the rows (16-bit values: read with the transposing loads).
#include "common.h"

namespace keep {

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

// 16 bytes per lane to lds_wave_base + 16 lane, from an address per lane, or from one offset per lane off a common
// base. Written out, since the compiler waits for every copy in flight before any LDS read that follows the builtin: here
// the reads are of the other buffer, and the loop's own wait and barrier stand between a copy and its readers. (No
// register is written, so none can be reused early; M0 is an operand, which the compiler sets and knows.)
__device__ __forceinline__ void dg_dma(const void* g, uint32_t lds_wave_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(lds_wave_base), "v"(g) : "memory");
}
__device__ __forceinline__ void dg_dma(const void* base, uint32_t off, uint32_t lds_wave_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds_wave_base), "v"(off), "s"(base) : "memory");
}

}  // namespace keep
