#pragma once
// Sums of column shares that blocks leave in float32: out[i] = round(sum over p of part[p][i]).
#include "common.h"

namespace keep {

// 32 columns a block, 32 runs of shares, each added in order and then the runs. Eight loads of a run are in flight.
template <typename W>
__global__ __launch_bounds__(1024) void k_parts_sum(const float* part, int parts, int n, W* out) {
  __shared__ float red[32][32 + 1];
  const int c = threadIdx.x & 31, s = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + c;
  const int per = (parts + 31) / 32, p0 = s * per, p1 = min(parts, p0 + per);
  float v = 0.f;
  if (i < n) {
    int p = p0;
    for (; p + 8 <= p1; p += 8) {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = part[(int64_t)(p + k) * n + i];
#pragma unroll
      for (int k = 0; k < 8; ++k) v += f[k];
    }
    for (; p < p1; ++p) v += part[(int64_t)p * n + i];
  }
  red[s][c] = v;
  __syncthreads();
  if (s > 0 || i >= n) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) v += red[k][c];
  out[i] = from_float<W>(v);
}

inline void parts_sum(const float* part, int64_t parts, int64_t n, void* out, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)((n + 31) / 32));
  if (dtype == KEEP_F32)
    hipLaunchKernelGGL(k_parts_sum<float>, grid, dim3(1024), 0, s, part, (int)parts, (int)n, (float*)out);
  else if (dtype == KEEP_F16)
    hipLaunchKernelGGL(k_parts_sum<_Float16>, grid, dim3(1024), 0, s, part, (int)parts, (int)n, (_Float16*)out);
  else
    hipLaunchKernelGGL(k_parts_sum<bf16s>, grid, dim3(1024), 0, s, part, (int)parts, (int)n, (bf16s*)out);
}

}  // namespace keep
