#pragma once
// Sums of outer products over the routes of each group:
//   out[g][j][i] (or [g][i][j] with j_inner) = sum over the group's routes r of J[r][j] I[r / i_div][i]
// in fp32 (dense.hip, k_rows_outer): the weight gradients of the routed products and of the adapters.
#include "common.h"

namespace keep {

struct OuterArgs {
  const void* i;  // [i_rows][i_dim], the wide side
  int64_t i_rows, i_div, i_dim;
  const void* j;  // [routes][j_ld], the first j_dim of a row
  int64_t j_ld, j_dim;
  const int32_t *order, *offsets, *counts;  // the groups' runs of sorted routes
  int64_t routes;
  void* out;
  int j_inner;
};

// dtype: of I and the output, and of J unless j_float.
int rows_outer(const OuterArgs& a, int dtype, bool j_float, int64_t groups, hipStream_t s, const char* what);

}  // namespace keep
