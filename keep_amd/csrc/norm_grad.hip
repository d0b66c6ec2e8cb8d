// Gradients of the root-mean-square norm with the residual's addition (norm.hip): with g = dy w, c = sum(g h) over the row
// and dh the gradient of h,
//   d = r (g - h r^2 c / n) + dh,  dx = round(d),  dresidual = round(d),  dw = sum over the rows of dy h r
// Bound by HBM: h, dy and dh are read once, dx (and dresidual, where its dtype is another) written once. dw is summed in a
// fixed order: per block in registers, then over the blocks. bf16, 8192 rows of 4096: 45.9 us (5.8 TB/s) and 4 of k_parts_sum;
// without the row ahead 114, of which most was the wait for a row's loads between two barriers. A float32 stream (8192 x 4096:
// 110 us, 4.3 TB/s) holds twice the registers, so that fewer blocks are resident.
#include "norm_dev.h"
#include "parts_dev.h"

namespace keep {

struct NormGradArgs {
  const void *h, *w, *dy, *dh;  // dh: or null
  int wdt;
  const float* rstd;
  int64_t T;
  int n;
  void *dx, *dres;  // either null
  float* part;      // [blocks][n] sums of the weight's gradient, or null
};

// Threads of a block: two rows and more where a row has fewer than 256.
constexpr int norm_grad_block(int tpr) { return tpr < 256 ? 256 : tpr; }

// H: type of h, dh and dresidual; X: of dy and dx. A block takes every gridDim-th group of rows, reads a group's values while
// it works on the one before, and adds its share of dw in registers, so that the shares that are left for k_parts_sum are as
// many as blocks.
template <typename X, typename H, int TPR, int NV, int END>
__global__ __launch_bounds__(norm_grad_block(TPR)) void k_rmsnorm_grad(NormGradArgs a) {
  constexpr int BT = norm_grad_block(TPR), RPB = BT / TPR;
  __shared__ float red[BT / 64];
  __shared__ float other[RPB > 1 ? TPR * NV * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, n = a.n;
  float dw[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int u = 0; u < 8; ++u) dw[v][u] = 0.f;
  float w[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) norm_weight<END>(a.w, a.wdt, (v * TPR + t) * 8, n, w[v]);
  struct Row {
    NormRaw<H> h[NV], dh[NV];
    NormRaw<X> dy[NV];
    float r;
  };
  const auto load = [&](Row& o, int64_t row) {
    const int64_t at = row < a.T ? row : a.T - 1;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * TPR + t) * 8;
      o.h[v].template load<END>((const H*)a.h + at * n, i, n);
      o.dy[v].template load<END>((const X*)a.dy + at * n, i, n);
      if (a.dh) o.dh[v].template load<END>((const H*)a.dh + at * n, i, n);
    }
    o.r = a.rstd[at];
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  // 1024 threads have 128 registers each, which two rows do not fit (2048 x 16384 bf16: 98 us with spills, 76 without)
  constexpr bool AHEAD = TPR < 1024;
  Row next;
  if constexpr (AHEAD) load(next, (int64_t)blockIdx.x * RPB + sub);
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.T; r0 += step) {
    const int64_t row = r0 + sub;
    const bool live = row < a.T;
    const int64_t at = row * n;
    if constexpr (!AHEAD) load(next, row);
    const Row now = next;
    if (AHEAD && r0 + step < a.T) load(next, row + step);
    float h[NV][8], g[NV][8];
    float c = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * TPR + t) * 8;
      now.h[v].template get<END>(i, n, h[v]);
      now.dy[v].template get<END>(i, n, g[v]);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (live) dw[v][u] = fmaf(g[v][u], h[v][u] * now.r, dw[v][u]);
        g[v][u] *= w[v][u];
        c = fmaf(g[v][u], h[v][u], c);
      }
    }
    c = norm_sum<TPR, BT>(c, red);
    if (!live || !(a.dx || a.dres)) continue;
    const float k = now.r * now.r * (c / (float)n);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (v * TPR + t) * 8;
      float d[8];
      now.dh[v].template get<END>(i, n, d);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float e = now.r * fmaf(-h[v][u], k, g[v][u]);
        d[u] = a.dh ? e + d[u] : e;
      }
      if (a.dx) norm_st<END>((X*)a.dx + at, i, n, d);
      if (a.dres) norm_st<END>((H*)a.dres + at, i, n, d);
    }
  }
  if (!a.part) return;
  if constexpr (RPB > 1) {
    for (int s = 1; s < RPB; ++s) {
      __syncthreads();
      if (sub == s)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int u = 0; u < 8; ++u) other[(v * 8 + u) * TPR + t] = dw[v][u];
      __syncthreads();
      if (sub == 0)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int u = 0; u < 8; ++u) dw[v][u] += other[(v * 8 + u) * TPR + t];
    }
    if (sub > 0) return;
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) norm_st<END>(a.part + (int64_t)blockIdx.x * n, (v * TPR + t) * 8, n, dw[v]);
}

// f(TPR, NV, END) for rows of n values: two vectors a thread, whose row and the one to come are in registers.
template <typename F>
static void norm_grad_by_width(int64_t n, F f) {
  using std::integral_constant;
  constexpr integral_constant<int, 1> one;
  constexpr integral_constant<int, 2> two;
  const auto by = [&](auto end) {
    if (n <= 512) f(integral_constant<int, 64>{}, one, end);
    else if (n <= 1024) f(integral_constant<int, 64>{}, two, end);
    else if (n <= 2048) f(integral_constant<int, 128>{}, two, end);
    else if (n <= 4096) f(integral_constant<int, 256>{}, two, end);
    else if (n <= 8192) f(integral_constant<int, 512>{}, two, end);
    else f(integral_constant<int, 1024>{}, two, end);
  };
  if (n < 8) f(integral_constant<int, 64>{}, one, integral_constant<int, NORM_TINY>{});
  else if (n % 8) by(integral_constant<int, NORM_ODD>{});
  else by(integral_constant<int, NORM_EVEN>{});
}

// Rows of a block of k_rmsnorm_grad, and its blocks: three per CU, as many as their registers let in.
static int norm_rows_per_block(int64_t n) {
  int rows = 1;
  norm_grad_by_width(n, [&](auto tpr, auto, auto) { rows = norm_grad_block(decltype(tpr)::value) / decltype(tpr)::value; });
  return rows;
}
static int64_t norm_parts(int64_t T, int64_t n) {
  const int64_t rpb = norm_rows_per_block(n);
  return std::min<int64_t>((T + rpb - 1) / rpb, 768);
}

template <typename X, typename H>
static void norm_grad_launch(const NormGradArgs& a, int64_t blocks, hipStream_t s) {
  norm_grad_by_width(a.n, [&](auto tpr, auto nv, auto end) {
    constexpr int TPR = decltype(tpr)::value, BT = norm_grad_block(TPR);
    hipLaunchKernelGGL((k_rmsnorm_grad<X, H, TPR, decltype(nv)::value, decltype(end)::value>), dim3((unsigned)blocks), dim3(BT), 0, s, a);
  });
}

}  // namespace keep

using namespace keep;

extern "C" int64_t keep_rmsnorm_grad_workspace_bytes(int64_t T, int64_t n) {
  if (!dims_ok({T, n}) || n > NORM_MAX) return 0;
  return norm_parts(T, n) * n * 4;
}

extern "C" int keep_rmsnorm_grad(const void* h, int h_dtype, const void* dy, int dy_dtype, const void* dh,
                                 const float* rstd, int64_t T, int64_t n, const void* weight, int weight_dtype,
                                 void* dx, void* dresidual, void* dweight, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  KEEP_REQUIRE_NORM(T, n, 0.f);
  KEEP_REQUIRE(dtype_ok(h_dtype) && dtype_ok(dy_dtype) && (!weight || dtype_ok(weight_dtype)), "bad dtype enum");
  KEEP_REQUIRE(h_dtype == dy_dtype || h_dtype == KEEP_F32, "h must have dy's dtype or float32");
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(h && dy && rstd && (dx || dresidual || dweight) && (weight || !dweight), "null pointer argument");
  KEEP_REQUIRE(aligned(h, dtype_size(h_dtype)) && aligned(dy, dtype_size(dy_dtype)) &&
                   aligned(dh, dtype_size(h_dtype)) && aligned(rstd, 4) && aligned(dx, dtype_size(dy_dtype)) &&
                   aligned(dresidual, dtype_size(h_dtype)) &&
                   (!weight || (aligned(weight, dtype_size(weight_dtype)) &&
                                aligned(dweight, dtype_size(weight_dtype)))),
               "misaligned pointer");
  const int64_t blocks = norm_parts(T, n);
  KEEP_REQUIRE(!dweight || (workspace && aligned(workspace, 4) && workspace_bytes >= blocks * n * 4),
               "the workspace must hold %lld bytes", (long long)(blocks * n * 4));
  NormGradArgs a{};
  a.h = h; a.w = weight; a.dy = dy; a.dh = dh; a.wdt = weight_dtype; a.rstd = rstd; a.T = T; a.n = (int)n;
  a.dx = dx; a.dres = dresidual; a.part = dweight ? (float*)workspace : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (dy_dtype == KEEP_F32) norm_grad_launch<float, float>(a, blocks, s);
  else if (dy_dtype == KEEP_F16 && h_dtype == KEEP_F32) norm_grad_launch<_Float16, float>(a, blocks, s);
  else if (dy_dtype == KEEP_F16) norm_grad_launch<_Float16, _Float16>(a, blocks, s);
  else if (h_dtype == KEEP_F32) norm_grad_launch<bf16s, float>(a, blocks, s);
  else norm_grad_launch<bf16s, bf16s>(a, blocks, s);
  if (dweight) parts_sum(a.part, blocks, n, dweight, weight_dtype, s);
  return launch_status("keep_rmsnorm_grad");
}
