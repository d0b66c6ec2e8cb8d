#pragma once
// Routed 16-bit products through LDS (dense_gemm.hip).
#include "common.h"

namespace keep {

struct DenseGemmArgs {
  const void* x;  // rows [x_rows][nk] (weight gradient: [x_rows][ni])
  int64_t x_rows, x_div;
  const int32_t* lhs;
  const void* w;  // weights (weight gradient: dy [routes][nj])
  int64_t E, ni, nj, nk;  // output columns; weight gradient: output rows; summed index
  int64_t routes;
  const int32_t *order, *offsets, *counts, *te, *to, *tc, *n_tiles;
  int64_t max_tiles;
  void* out;
  int odt, wide;
  int far;                      // an operand of 4 GiB or more (set at the launch)
  uint32_t div_mul, div_shift;  // x_div as a multiplication (set at the launch)
};

bool dense_gemm_tile(int64_t tile);  // tiles of a plan that dense_gemm_rows takes
int dense_gemm_rows(const DenseGemmArgs& a, int dtype, bool transposed, int64_t tile, hipStream_t s);
int dense_gemm_weight(const DenseGemmArgs& a, int dtype, hipStream_t s);

}  // namespace keep
