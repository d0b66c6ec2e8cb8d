// Root-mean-square norm of rows with the residual's addition on gfx950, its
// 8-bit form and its gradients.
//
//   h = round(residual + x)                      (fp32 sum, rounded to the residual's dtype; no residual: h = x)
//   r = 1 / sqrt(mean(h^2) + eps)
//   y = round(h r w)                             (w = 1 without a weight)
//   8 bits: s = max(max |h r w|, 1e-4) / 448 per block of values, q = e4m3(h r w / s)
// and with g = dy w, c = sum(g h) over the row:
//   d = r (g - h r^2 c / n) + dh,  dx = round(d),  dresidual = round(d),  dw = sum over the rows of dy h r
//
// The norm is of the rounded h: it is what the caller keeps, and what the backward pass reads again. The 8-bit values come
// from the fp32 product, so that they are rounded once. The bound of 1e-4 on a block's largest value, under which values
// lose bits, is act_quant's (scripts/runpod/v41_reap/torch_kernel.py:40-53).
//
// Bound by HBM: every value is read once, kept in registers as fp32 over the row's sum, and written once. bf16 with a
// residual, 8192 rows of 4096: 40.4 us, 6.6 TB/s; of 2048 22.1; 65536 of 512 without one 23.9 (5.6 TB/s); 4096 of 7168 37.4,
// in 8 bits 38.2; float32 4096 of 4096 42.8 (6.3 TB/s). One row of 7168: 3.5 us in a graph, a launch and the loads'
// way. The 8-bit rows multiply by the scale's reciprocal and correct the product: 2048 rows of 4096 13.9 us, without
// the correction 13.7 (and codes beside a middle a step off), with a division a value 19.5.
#include "norm_dev.h"

namespace keep {

struct NormArgs {
  const void *x, *res, *w;
  int wdt;
  int64_t T;
  int n;
  float eps;
  void *h, *y;    // h: null without a residual
  float* rstd;    // or null
  uint8_t* q;     // 8-bit form: in y's place
  float* scales;
  int qblock, pow2;
};

// 2^ceil(log2 v) of a positive normal v.
__device__ __forceinline__ float norm_pow2_ceil(float v) {
  const uint32_t b = __float_as_uint(v);
  return __uint_as_float((b + 0x7FFFFFu) & 0xFF800000u);
}

// X: type of x and y; R: of the residual (void: none).
template <typename X, typename R, int TPR, int NV, int END, bool QUANT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_rmsnorm(NormArgs a) {
  constexpr int BT = TPR < 256 ? 256 : TPR, RPB = BT / TPR;
  __shared__ float red[BT / 64];
  const int t = threadIdx.x % TPR, n = a.n;
  constexpr bool RES = !__is_same(R, void);
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.T; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool live = row < a.T;
    const int64_t at = (live ? row : 0) * n;
    float h[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) norm_ld<END>((const X*)a.x + at, (v * TPR + t) * 8, n, h[v]);
    if constexpr (RES) {
      float p[NV][8];
#pragma unroll
      for (int v = 0; v < NV; ++v) norm_ld<END>((const R*)a.res + at, (v * TPR + t) * 8, n, p[v]);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int u = 0; u < 8; u += 2) {
          h[v][u] += p[v][u];
          h[v][u + 1] += p[v][u + 1];
          if constexpr (sizeof(R) == 2) {  // the stream as it is kept
            const uint32_t w = norm_pair<R>(h[v][u], h[v][u + 1]);
            h[v][u] = pair_lo<PairOf<R>::value>(w);
            h[v][u + 1] = pair_hi<PairOf<R>::value>(w);
          }
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int u = 0; u < 8; ++u) ss = fmaf(h[v][u], h[v][u], ss);
    if constexpr (RES) {
      if (live)
#pragma unroll
        for (int v = 0; v < NV; ++v) norm_st<END>((R*)a.h + at, (v * TPR + t) * 8, n, h[v]);
    }
    ss = norm_sum<TPR, BT>(ss, red);
    const float r = 1.f / sqrtf(ss / (float)n + a.eps);
    if (live && t == 0 && a.rstd) a.rstd[row] = r;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * TPR + t) * 8;
      float w[8];
      norm_weight<END>(a.w, a.wdt, i, n, w);
#pragma unroll
      for (int u = 0; u < 8; ++u) h[v][u] = h[v][u] * r * w[u];
      if constexpr (!QUANT) {
        if (live) norm_st<END>((X*)a.y + at, i, n, h[v]);
      } else {
        // a maximum of the bits, which a NaN outranks
        uint32_t bits = 0u;
#pragma unroll
        for (int u = 0; u < 8; ++u) bits = max(bits, __float_as_uint(h[v][u]) & 0x7fffffffu);
        for (int o = 1; o < a.qblock / 8; o <<= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o, 64));
        const float top = __uint_as_float(bits);
        float s = (top < 1e-4f ? 1e-4f : top) / 448.f;
        if (a.pow2 && s < __builtin_inff()) s = norm_pow2_ceil(s);
        // The quotient by s from its product with 1 / s, corrected by what that product leaves over: float32's rounded
        // quotient without a division a value. It is at most 448 and a step, which the conversion rounds to 448.
        const float inv = 1.f / s, by = s < __builtin_inff() ? s : 0.f;  // (beside an infinite value: 0)
        float f[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float c = h[v][u] * inv;
          f[u] = fmaf(fmaf(-c, by, h[v][u]), inv, c);
        }
        uint32_t word[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          int b = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * u], f[4 * u + 1], 0, false);
          word[u] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * u + 2], f[4 * u + 3], b, true);
        }
        if (live) {
          uint8_t* to = a.q + at + i;
          if (i + 8 <= n) {
            __builtin_memcpy(to, word, 8);
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (i + u < n) to[u] = (uint8_t)(word[u >> 2] >> (8 * (u & 3)));
          }
          if (i % a.qblock == 0 && i < n) a.scales[row * ((n + a.qblock - 1) / a.qblock) + i / a.qblock] = s;
        }
      }
    }
  }
}

template <typename X, typename R, bool QUANT>
static void norm_launch(const NormArgs& a, hipStream_t s) {
  norm_by_width(a.n, [&](auto tpr, auto nv, auto end) {
    constexpr int TPR = decltype(tpr)::value, BT = TPR < 256 ? 256 : TPR;
    const dim3 grid((unsigned)std::min<int64_t>((a.T + BT / TPR - 1) / (BT / TPR), NORM_BLOCKS));
    hipLaunchKernelGGL((k_rmsnorm<X, R, TPR, decltype(nv)::value, decltype(end)::value, QUANT>), grid, dim3(BT), 0, s, a);
  });
}

template <typename X, bool QUANT>
static void norm_launch(const NormArgs& a, int rdt, hipStream_t s) {
  if (!a.res) norm_launch<X, void, QUANT>(a, s);
  else if (rdt == KEEP_F32) norm_launch<X, float, QUANT>(a, s);
  else norm_launch<X, X, QUANT>(a, s);
}

template <bool QUANT>
static void norm_launch(const NormArgs& a, int dt, int rdt, hipStream_t s) {
  if (dt == KEEP_F32) norm_launch<float, QUANT>(a, rdt, s);
  else if (dt == KEEP_F16) norm_launch<_Float16, QUANT>(a, rdt, s);
  else norm_launch<bf16s, QUANT>(a, rdt, s);
}

}  // namespace keep

using namespace keep;

extern "C" int keep_rmsnorm(const void* x, int x_dtype, const void* residual, int residual_dtype, int64_t T, int64_t n,
                            const void* weight, int weight_dtype, float eps, void* h, void* y, float* rstd,
                            void* stream) {
  KEEP_REQUIRE_NORM(T, n, eps);
  KEEP_REQUIRE(dtype_ok(x_dtype) && (!weight || dtype_ok(weight_dtype)), "bad dtype enum");
  KEEP_REQUIRE(!residual || residual_dtype == x_dtype || residual_dtype == KEEP_F32,
               "the residual must have x's dtype or float32");
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(x && y && !residual == !h, "null pointer argument");
  KEEP_REQUIRE(aligned(x, dtype_size(x_dtype)) && aligned(y, dtype_size(x_dtype)) &&
                   (!residual || (aligned(residual, dtype_size(residual_dtype)) &&
                                  aligned(h, dtype_size(residual_dtype)))) &&
                   (!weight || aligned(weight, dtype_size(weight_dtype))) && aligned(rstd, 4),
               "misaligned pointer");
  NormArgs a{};
  a.x = x; a.res = residual; a.w = weight; a.wdt = weight_dtype; a.T = T; a.n = (int)n; a.eps = eps;
  a.h = h; a.y = y; a.rstd = rstd;
  norm_launch<false>(a, x_dtype, residual_dtype, (hipStream_t)stream);
  return launch_status("keep_rmsnorm");
}

extern "C" int keep_rmsnorm_quant(const void* x, int x_dtype, const void* residual, int residual_dtype, int64_t T,
                                  int64_t n, const void* weight, int weight_dtype, float eps, int64_t quant_block,
                                  int pow2_scales, void* h, void* q, float* scales, void* stream) {
  KEEP_REQUIRE_NORM(T, n, eps);
  KEEP_REQUIRE_DIMS(quant_block);
  KEEP_REQUIRE(dtype_ok(x_dtype) && (!weight || dtype_ok(weight_dtype)), "bad dtype enum");
  KEEP_REQUIRE(!residual || residual_dtype == x_dtype || residual_dtype == KEEP_F32,
               "the residual must have x's dtype or float32");
  KEEP_REQUIRE(quant_block >= 16 && quant_block <= 512 && (quant_block & (quant_block - 1)) == 0,
               "quant_block must be a power of two in 16..512, got %lld", (long long)quant_block);
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(x && q && scales && !residual == !h, "null pointer argument");
  KEEP_REQUIRE(aligned(x, dtype_size(x_dtype)) && aligned(scales, 4) &&
                   (!residual || (aligned(residual, dtype_size(residual_dtype)) &&
                                  aligned(h, dtype_size(residual_dtype)))) &&
                   (!weight || aligned(weight, dtype_size(weight_dtype))),
               "misaligned pointer");
  NormArgs a{};
  a.x = x; a.res = residual; a.w = weight; a.wdt = weight_dtype; a.T = T; a.n = (int)n; a.eps = eps;
  a.h = h; a.q = (uint8_t*)q; a.scales = scales; a.qblock = (int)quant_block; a.pow2 = pow2_scales;
  norm_launch<true>(a, x_dtype, residual_dtype, (hipStream_t)stream);
  return launch_status("keep_rmsnorm_quant");
}
