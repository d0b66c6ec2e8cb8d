// The routed combine on rows of any float type, and its gradients.
//
//   out[t]   = sum_j w[t, j] y[t, j]           (j in order, fp32 multiply-adds, rounded once)
//   dy[t, j] = w[t, j] dout[t]
//   dw[t, j] = <y[t, j], dout[t]>
//
// Elementwise over H beside one dot product per route: HBM-bound. The forward
// gives a thread 16 bytes of a row (eight or four values) and walks the token's
// k rows; the backward gives a wave one route, which reads its row of y once,
// writes its row of dy once and takes dout, which the k routes of a token
// share, from the caches. Measured: 2048 x 6 rows of 4096, bf16 to float32
// (134 MB) 23.8 us, 5.6 TB/s; backward of 1021 x 8 rows of 4096, bf16 (151 MB) 28 to 31 us, where a copy of as many
// bytes takes 29. Rows of no whole number of eight values go value by value: 2048 x 6 rows of 4092 66 us.
#include <algorithm>

#include "common.h"

namespace keep {

// V consecutive values of a row as floats: one load where VEC (V values, 16 or 32 bytes, aligned and all there).
template <typename T, int V, bool VEC>
__device__ __forceinline__ void ld_row(const T* p, int64_t n, float (&f)[V]) {
  if constexpr (VEC && sizeof(T) == 2) {
    static_assert(V == 8, "16 bytes");
    const uint4 q = *(const uint4*)p;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = pair_lo<PairOf<T>::value>(w[i]);
      f[2 * i + 1] = pair_hi<PairOf<T>::value>(w[i]);
    }
  } else if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 q = ((const float4*)p)[i];
      f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < n ? to_float(p[i]) : 0.f;
  }
}

template <typename T, int V, bool VEC>
__device__ __forceinline__ void st_row(T* p, int64_t n, const float (&f)[V]) {
  if constexpr (VEC && sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(f[2 * i])) |
             ((uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(f[2 * i + 1])) << 16);
    *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
  } else if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) ((float4*)p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = from_float<T>(f[i]);
  }
}

// w = null: weights of one (the sum of a token's rows).
template <typename T, typename OT, bool VEC>
__global__ __launch_bounds__(256) void k_combine_rows(const T* y, const float* w, int64_t n_tok, int k, int64_t H,
                                                      OT* out) {
  constexpr int V = 8;
  const int64_t HV = (H + V - 1) / V;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_tok * HV; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / HV, c = (i - t * HV) * V;
    float acc[V] = {};
    for (int j = 0; j < k; ++j) {
      float f[V];
      ld_row<T, V, VEC>(y + (t * k + j) * H + c, H - c, f);
      const float wt = w ? w[t * k + j] : 1.f;
#pragma unroll
      for (int u = 0; u < V; ++u) acc[u] = fmaf(wt, f[u], acc[u]);
    }
    st_row<OT, V, VEC>(out + t * H + c, H - c, acc);
  }
}

template <typename T, typename DT, bool VEC>
__global__ __launch_bounds__(256) void k_combine_grad(const T* y, const float* w, const DT* dout, int64_t routes, int k,
                                                      int64_t H, T* dy, float* dw) {
  constexpr int V = 8;
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < routes; r += (int64_t)gridDim.x * 4) {
    const int64_t t = r / k;
    const float wt = w[r];
    float dot = 0.f;
    for (int64_t c = lane * V; c < H; c += 64 * V) {
      float d[V], f[V];
      ld_row<DT, V, VEC>(dout + t * H + c, H - c, d);
      if (dw) {
        ld_row<T, V, VEC>(y + r * H + c, H - c, f);
#pragma unroll
        for (int u = 0; u < V; ++u) dot = fmaf(f[u], d[u], dot);
      }
      if (dy) {
#pragma unroll
        for (int u = 0; u < V; ++u) d[u] *= wt;
        st_row<T, V, VEC>(dy + r * H + c, H - c, d);
      }
    }
    if (dw) {
      dot = wave_sum(dot);
      if (lane == 0) dw[r] = dot;
    }
  }
}

constexpr int64_t COMBINE_VALUES = int64_t(1) << 40;  // more than a GPU holds
constexpr int64_t COMBINE_BLOCKS = 1 << 23;  // a launch holds 2^32 threads; more work goes round again

template <typename T, typename OT>
void launch_combine(const void* y, const float* w, int64_t T_, int64_t k, int64_t H, void* out, bool vec,
                    hipStream_t s) {
  const int64_t n = T_ * ((H + 7) / 8);
  const dim3 grid((unsigned)std::min((n + 255) / 256, COMBINE_BLOCKS));
  if (vec)
    hipLaunchKernelGGL((k_combine_rows<T, OT, true>), grid, dim3(256), 0, s, (const T*)y, w, T_, (int)k, H, (OT*)out);
  else
    hipLaunchKernelGGL((k_combine_rows<T, OT, false>), grid, dim3(256), 0, s, (const T*)y, w, T_, (int)k, H, (OT*)out);
}

template <typename T, typename DT>
void launch_combine_grad(const void* y, const float* w, const void* dout, int64_t routes, int64_t k, int64_t H,
                         void* dy, float* dw, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)std::min((routes + 3) / 4, COMBINE_BLOCKS));
  if (vec)
    hipLaunchKernelGGL((k_combine_grad<T, DT, true>), grid, dim3(256), 0, s, (const T*)y, w, (const DT*)dout, routes,
                       (int)k, H, (T*)dy, dw);
  else
    hipLaunchKernelGGL((k_combine_grad<T, DT, false>), grid, dim3(256), 0, s, (const T*)y, w, (const DT*)dout, routes,
                       (int)k, H, (T*)dy, dw);
}

template <typename F>
void by_dtype(int dt, F f) {
  if (dt == KEEP_F32) f(float{});
  else if (dt == KEEP_F16) f(_Float16{});
  else f(bf16s{});
}

}  // namespace keep

using namespace keep;

extern "C" int keep_route_combine_rows(const void* y, int y_dtype, const float* w, int64_t T, int64_t k, int64_t H,
                                       void* out, int out_dtype, void* stream) {
  KEEP_REQUIRE_DIMS(T, k, H);
  KEEP_REQUIRE(dtype_ok(y_dtype) && dtype_ok(out_dtype), "bad dtype enum");
  KEEP_REQUIRE(k > 0 && H > 0, "k and H must be positive");
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(y && out, "null pointer argument");
  KEEP_REQUIRE(T <= COMBINE_VALUES / k / H, "too many values");
  const bool vec = H % 8 == 0 && aligned(y, 16) && aligned(out, 16);
  by_dtype(y_dtype, [&](auto t) {
    by_dtype(out_dtype, [&](auto o) {
      launch_combine<decltype(t), decltype(o)>(y, w, T, k, H, out, vec, (hipStream_t)stream);
    });
  });
  return launch_status("keep_route_combine_rows");
}

extern "C" int keep_route_combine_grad(const void* y, int y_dtype, const float* w, const void* dout, int dout_dtype,
                                       int64_t T, int64_t k, int64_t H, void* dy, float* dw, void* stream) {
  KEEP_REQUIRE_DIMS(T, k, H);
  KEEP_REQUIRE(dtype_ok(y_dtype) && dtype_ok(dout_dtype), "bad dtype enum");
  KEEP_REQUIRE(k > 0 && H > 0, "k and H must be positive");
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(w && dout && (dy || dw) && (y || !dw), "null pointer argument");
  KEEP_REQUIRE(T <= COMBINE_VALUES / k / H, "too many values");
  const bool vec = H % 8 == 0 && aligned(y, 16) && aligned(dout, 16) && aligned(dy, 16);
  by_dtype(y_dtype, [&](auto t) {
    by_dtype(dout_dtype, [&](auto d) {
      launch_combine_grad<decltype(t), decltype(d)>(y, w, dout, T * k, k, H, dy, dw, vec, (hipStream_t)stream);
    });
  });
  return launch_status("keep_route_combine_grad");
}
