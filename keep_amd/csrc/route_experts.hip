// The choice of each token's experts among groups, with the weights' gradients,
// on gfx950: one wave64 per token.
//
//   s_e = score(z_e)                          softmax over the experts, sigmoid or sqrt(softplus)
//   key_e = s_e + bias_e                      the bias balances the choice and does not enter the weights
//   value of a group = the sum of its two largest keys (its only key where it has one expert)
//   chosen: the k largest keys in the topk_groups groups of the largest values
//   w_j = s_j / (sum s_i + 1e-20) scale       (without renormalisation: s_j scale)
//
// The lower index comes first among equal keys, NaN ranks as -inf, and a choice does not depend on how fp32 rounds. Without
// a bias the scores order as the logits do, and the logits are what is compared. With one (and for the groups' values) keys
// are formed in fp32, and where two that decide the outcome lie closer than fp32 is sure of, the token is chosen again with
// keys in 64 bits. Equal logits under equal biases are equal without a second look.
//
// The groups are spread over the lanes: LG lanes share a group (the largest power of two with LG groups <= 64), so that a
// group's two largest are found inside its lanes.
//
// With c = scale / (sum s_i + 1e-20) and p_j = c (g_j - sum g_i s_i / (sum s_i + 1e-20)), the gradient of s_j
// (not renormalised: p_j = scale g_j):
//   softmax: dz_e = s_e ([e chosen] p_e - sum p_j s_j);  sigmoid: p s (1 - s);  sqrt(softplus): p sigmoid(z) / (2 s)
#include "route_dev.h"

namespace keep {

struct ChooseArgs {
  const void* z;
  int zdt;
  const float* bias;
  int T, E, k, groups, topk_groups;
  int func, renorm;
  float scale;
  int32_t* idx;
  float* w;
  int32_t* load;  // or null
};

__device__ __forceinline__ float ch_load(const void* z, int dt, int64_t i) {
  if (dt == KEEP_F32) return ((const float*)z)[i];
  if (dt == KEEP_BF16) return to_float(((const bf16s*)z)[i]);
  return to_float(((const _Float16*)z)[i]);
}

// Which experts a lane holds: i-th is first + i step for i < n.
struct ChooseLane {
  int lg, group, sub, first, n;
  __device__ __forceinline__ ChooseLane(int E, int groups, int lane) {
    lg = 64 / groups;
    lg = 1 << (31 - __clz(lg));
    const int size = E / groups;
    group = lane / lg;
    sub = lane & (lg - 1);
    first = group * size + sub;
    n = group < groups && sub < size ? (size - sub + lg - 1) / lg : 0;
  }
};

__device__ __forceinline__ int ch_reduce_min(int v) { return (int)rt_wave_u32<false>((uint32_t)v); }

// Softmax scores of a row whose logits are all -inf are 0.
template <int PER>
__device__ __forceinline__ void ch_scores(const float (&z)[PER], int n, int func, float (&s)[PER]) {
  if (func == KEEP_SCORE_SOFTMAX) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmaxf(m, z[i]);
    m = wave_max(m);
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = i < n && (m > -__builtin_inff() || z[i] != z[i]) ? expf(z[i] - m) : 0.f;
      part += s[i];
    }
    const float sum = wave_sum(part);
    const float r = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] *= r;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = i < n ? rt_score_of(z[i], func) : 0.f;
  }
}

__device__ __forceinline__ double ch_wave_max_d(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmax(v, __shfl_xor(v, m, 64));
  return v;
}

// The choice in 64 bits: lane j < k gets winner j. The logits are read again: the few tokens that come here shall not cost
// the others registers.
template <int PER>
__device__ __forceinline__ int ch_exact(const ChooseArgs& a, const ChooseLane& l, int64_t t, int lane) {
  const int n = l.n, first = l.first, lg = l.lg, group = l.group;
  float z[PER];
  double key[PER];
  const double none = -__builtin_inf();
#pragma unroll
  for (int i = 0; i < PER; ++i) z[i] = i < n ? ch_load(a.z, a.zdt, t * a.E + first + i * lg) : -__builtin_inff();
  if (a.func == KEEP_SCORE_SOFTMAX) {
    double m = none;
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmax(m, i < n ? (double)z[i] : none);
    m = ch_wave_max_d(m);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = i < n && (m > none || z[i] != z[i]) ? exp((double)z[i] - m) : 0.;
      sum += key[i];
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = sum == 0. ? 0. : key[i] / sum;
  } else if (a.func == KEEP_SCORE_SIGMOID) {
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = 1. / (1. + exp(-(double)z[i]));
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      key[i] = sqrt(fmax((double)z[i], 0.) + log1p(exp(-fabs((double)z[i]))));
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (a.bias && i < n) key[i] += (double)a.bias[first + i * lg];
    if (key[i] != key[i] || i >= n) key[i] = none;
  }
  bool in = n > 0;
  if (a.topk_groups < a.groups) {
    double t1 = none, t2 = none;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      t2 = fmax(t2, fmin(t1, key[i]));
      t1 = fmax(t1, key[i]);
    }
    for (int o = 1; o < lg; o <<= 1) {
      const double o1 = __shfl_xor(t1, o, 64), o2 = __shfl_xor(t2, o, 64);
      t2 = fmax(fmin(t1, o1), fmax(t2, o2));
      t1 = fmax(t1, o1);
    }
    double v = a.E > a.groups ? t1 + t2 : t1;
    if (v != v) v = none;
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const double o = __shfl(v, h * lg, 64);
      rank += o > v || (o == v && h < group) ? 1 : 0;
    }
    in = in && rank < a.topk_groups;
  }
  if (!a.bias) {
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = z[i] == z[i] ? (double)z[i] : none;
  }
  uint32_t open = 0;  // slots that are not chosen yet
#pragma unroll
  for (int i = 0; i < PER; ++i) open |= in && i < n ? 1u << i : 0u;
  int mine = 0;
  for (int j = 0; j < a.k; ++j) {
    double best = none;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if ((open >> i & 1u) && key[i] >= best) {
        best = key[i];
        at = first + i * lg;
      }
    const double top = ch_wave_max_d(best);
    const int e = ch_reduce_min(best == top ? at : 0x7fffffff);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e == first + i * lg && i < n) open &= ~(1u << i);
    mine = lane == j ? e : mine;
  }
  return mine;
}

// How far a score formed in fp32 may be from the real one: expf and the divisions 2^-21 of it; the softmax's exponent loses
// |z - m| 2^-24 too, up to 104 before the score is 0.
__device__ __forceinline__ float ch_unsure(int func) { return func == KEEP_SCORE_SOFTMAX ? 0x1p-17f : 0x1p-20f; }

template <int PER>
__global__ __launch_bounds__(256) void k_route_experts(ChooseArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const ChooseLane l(a.E, a.groups, lane);
  float z[PER], b[PER], s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = l.first + i * l.lg;
    z[i] = i < l.n ? ch_load(a.z, a.zdt, t * a.E + e) : -__builtin_inff();
    b[i] = a.bias && i < l.n ? a.bias[e] : 0.f;
  }
  ch_scores<PER>(z, l.n, a.func, s);
  bool sure = true, in = l.n > 0;
  const bool biased = a.bias != nullptr, grouped = a.topk_groups < a.groups;
  // how far any two keys' scores may be off together
  float unsure = 0.f;
  if (biased || grouped) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmaxf(m, s[i]);
    unsure = 2.f * ch_unsure(a.func) * rt_wave_reduce(m, true);
  }
  if (grouped) {
    const float none = -__builtin_inff();
    float t1 = none, t2 = none;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float v = i < l.n ? s[i] + b[i] : none;
      t2 = fmaxf(t2, fminf(t1, v));
      t1 = fmaxf(t1, v);
    }
    for (int o = 1; o < l.lg; o <<= 1) {
      const float o1 = __shfl_xor(t1, o, 64), o2 = __shfl_xor(t2, o, 64);
      t2 = fmaxf(fminf(t1, o1), fmaxf(t2, o2));
      t1 = fmaxf(t1, o1);
    }
    const bool pair = a.E > a.groups;
    float v = pair ? t1 + t2 : t1;
    if (v != v) v = none;
    // two values' scores, and the roundings of two keys and their sum in each
    const float err = 2.f * unsure + 0x1p-21f * rt_wave_reduce(l.n > 0 ? fabsf(t1) + (pair ? fabsf(t2) : 0.f) : 0.f, true);
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), h * l.lg));
      rank += o > v || (o == v && h < l.group) ? 1 : 0;
    }
    in = in && rank < a.topk_groups;
    // the last group that is in and the first that is not
    const uint64_t ma = __ballot(l.group < a.groups && rank == a.topk_groups - 1);
    const uint64_t mb = __ballot(l.group < a.groups && rank == a.topk_groups);
    if (ma == 0 || mb == 0) {
      sure = false;
    } else {
      const int la = __builtin_ctzll(ma), lb = __builtin_ctzll(mb);
      sure = __shfl(v, la, 64) - __shfl(v, lb, 64) > err;
    }
  }
  // without a bias the logits are the keys
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = in && i < l.n ? rt_sortable(biased ? s[i] + b[i] : z[i]) : 0u;
  int mine = 0;
  float ws = 0.f, total = 0.f, pk = 0.f, pz = 0.f, pb = 0.f;
  const int rounds = biased ? a.k + 1 : a.k;
  for (int j = 0; j < rounds; ++j) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) top = max(top, key[i]);
    const uint32_t best = rt_wave_u32<true>(top);
    if (best == 0u) break;  // fewer than k + 1 experts
    int at = 0x7fffffff;
    float zs = 0.f, bs = 0.f, ss = 0.f;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == best) {
        at = l.first + i * l.lg;
        zs = z[i];
        bs = b[i];
        ss = s[i];
      }
    const uint64_t who = __ballot(top == best);
    int owner = __builtin_ctzll(who), e;
    if (who & (who - 1)) {  // several lanes: the lowest expert
      e = ch_reduce_min(at);
      owner = __builtin_ctzll(__ballot(at == e));
    }
    e = __builtin_amdgcn_readlane(at, owner);
    const auto of = [&](float v) {
      return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), owner));
    };
    const float se = of(ss);
    if (biased) {
      const float ke = rt_unsortable(best), ze = of(zs), be = of(bs);
      if (j > 0) {
        const float err = unsure + 0x1p-23f * (fabsf(ke) + fabsf(pk));  // (a key further down may be off as far)
        sure = sure && (pk - ke > err || (ze == pz && be == pb));
      }
      pk = ke; pz = ze; pb = be;
    }
    if (j == a.k) break;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == e && key[i] == best && l.first + i * l.lg == e) key[i] = 0u;
    if (lane == j) {
      mine = e;
      ws = se;
    }
    total += se;
  }
  if (!sure) {
    mine = ch_exact<PER>(a, l, t, lane);
    total = 0.f;
    for (int j = 0; j < a.k; ++j) {  // the scores of the choice, in its order
      const int e = __builtin_amdgcn_readlane(mine, j);
      float v = 0.f;
      bool here = false;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < l.n && l.first + i * l.lg == e) {
          v = s[i];
          here = true;
        }
      const int owner = __builtin_ctzll(__ballot(here));
      const float se = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), owner));
      if (lane == j) ws = se;
      total += se;
    }
  }
  if (lane < a.k) {
    a.idx[t * a.k + lane] = mine;
    a.w[t * a.k + lane] = (a.renorm ? ws / (total + 1e-20f) : ws) * a.scale;
    if (a.load) atomicAdd(a.load + mine, 1);
  }
}

struct ChooseGradArgs {
  const void* z;
  int zdt;
  const int32_t* idx;
  const float* dw;
  int T, E, k;
  int func, renorm;
  float scale;
  void* dz;
};

__device__ __forceinline__ void ch_store(void* p, int dt, int64_t i, float v) {
  if (dt == KEEP_F32) ((float*)p)[i] = v;
  else if (dt == KEEP_BF16) ((bf16s*)p)[i] = from_float<bf16s>(v);
  else ((_Float16*)p)[i] = from_float<_Float16>(v);
}

template <int PER>
__global__ __launch_bounds__(256) void k_route_experts_grad(ChooseGradArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int n = lane < a.E ? (a.E - lane + 63) / 64 : 0;
  float z[PER], s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) z[i] = i < n ? ch_load(a.z, a.zdt, t * a.E + lane + 64 * i) : -__builtin_inff();
  ch_scores<PER>(z, n, a.func, s);
  // lane j < k: the j-th choice
  const bool chosen = lane < a.k;
  const int e = chosen ? a.idx[t * a.k + lane] : 0;
  const float g = chosen ? a.dw[t * a.k + lane] : 0.f;
  float se = 0.f, ze = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float sv = __shfl(s[i], e & 63, 64), zv = __shfl(z[i], e & 63, 64);
    if ((e >> 6) == i) {
      se = sv;
      ze = zv;
    }
  }
  if (!chosen) se = 0.f;
  float p = a.scale * g;
  if (a.renorm) {
    const float total = wave_sum(se) + 1e-20f;
    p = a.scale / total * (g - wave_sum(g * se) / total);
  }
  float dot = 0.f;
  if (a.func == KEEP_SCORE_SOFTMAX) {
    dot = wave_sum(chosen ? p * se : 0.f);
  } else if (a.func == KEEP_SCORE_SIGMOID) {
    p *= 1.f - se;  // (times the score below)
  } else {
    // sigmoid(z) / (2 s) over s; where both vanish, s^2 -> e^z and the slope is s / 2
    p *= se > 0.f ? 0.5f * rt_score_of(ze, KEEP_SCORE_SIGMOID) / se / se : 0.f;
  }
  float d[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) d[i] = a.func == KEEP_SCORE_SOFTMAX ? -dot : 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int ej = __builtin_amdgcn_readlane(e, j);
    const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j));
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (ej == lane + 64 * i) d[i] += pj;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i < n) ch_store(a.dz, a.zdt, t * a.E + lane + 64 * i, s[i] * d[i]);
}

}  // namespace keep

using namespace keep;

static int choose_sizes(int64_t T, int64_t E, int64_t k, int score_func) {
  KEEP_REQUIRE_DIMS(T, E, k);
  KEEP_REQUIRE(E >= 1 && E <= 64 * RT_MAX_PER_LANE, "E must be in 1..%d, got %lld", 64 * RT_MAX_PER_LANE,
               (long long)E);
  KEEP_REQUIRE(k >= 1 && k <= 32 && k <= E, "k must be in 1..min(32, E), got %lld", (long long)k);
  KEEP_REQUIRE(score_func >= 0 && score_func <= 2, "bad score_func %d", score_func);
  KEEP_REQUIRE(T <= (int64_t(1) << 25), "at most 2^25 tokens");  // a launch holds 2^32 threads, 64 a token
  return KEEP_OK;
}

extern "C" int keep_route_experts(const void* logits, int dtype, int64_t T, int64_t E, int64_t k, const float* bias,
                                  int64_t groups, int64_t topk_groups, int score_func, int renormalize,
                                  float route_scale, int32_t* idx, float* w, int32_t* load, void* stream) {
  if (const int rc = choose_sizes(T, E, k, score_func)) return rc;
  KEEP_REQUIRE_DIMS(groups, topk_groups);
  KEEP_REQUIRE(dtype_ok(dtype), "bad dtype enum");
  KEEP_REQUIRE(groups >= 1 && groups <= 64 && E % groups == 0, "groups must be in 1..64 and divide E");
  KEEP_REQUIRE(topk_groups >= 1 && topk_groups <= groups && k <= topk_groups * (E / groups),
               "topk_groups must be in 1..groups and hold k experts");
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(logits && idx && w, "null pointer argument");
  KEEP_REQUIRE(aligned(logits, dtype_size(dtype)) && aligned(bias, 4) && aligned(idx, 4) && aligned(w, 4) &&
                   aligned(load, 4),
               "misaligned pointer");
  ChooseArgs a{logits, dtype, bias, (int)T, (int)E, (int)k, (int)groups, (int)topk_groups, score_func, renormalize,
               route_scale, idx, w, load};
  int lg = 1;
  while (lg * 2 * groups <= 64) lg *= 2;
  const int64_t per = (E / groups + lg - 1) / lg;
  const dim3 grid((unsigned)((T + 3) / 4)), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (per <= 1) hipLaunchKernelGGL(k_route_experts<1>, grid, block, 0, s, a);
  else if (per <= 2) hipLaunchKernelGGL(k_route_experts<2>, grid, block, 0, s, a);
  else if (per <= 4) hipLaunchKernelGGL(k_route_experts<4>, grid, block, 0, s, a);
  else if (per <= 6) hipLaunchKernelGGL(k_route_experts<6>, grid, block, 0, s, a);
  else if (per <= 8) hipLaunchKernelGGL(k_route_experts<8>, grid, block, 0, s, a);
  else if (per <= 16) hipLaunchKernelGGL(k_route_experts<16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(k_route_experts<32>, grid, block, 0, s, a);  // groups one more than a power of two
  return launch_status("keep_route_experts");
}

extern "C" int keep_route_experts_grad(const void* logits, int dtype, int64_t T, int64_t E, int64_t k,
                                       const int32_t* idx, const float* dw, int score_func, int renormalize,
                                       float route_scale, void* dlogits, void* stream) {
  if (const int rc = choose_sizes(T, E, k, score_func)) return rc;
  KEEP_REQUIRE(dtype_ok(dtype), "bad dtype enum");
  if (T == 0) return KEEP_OK;
  KEEP_REQUIRE(logits && idx && dw && dlogits, "null pointer argument");
  KEEP_REQUIRE(aligned(logits, dtype_size(dtype)) && aligned(idx, 4) && aligned(dw, 4) &&
                   aligned(dlogits, dtype_size(dtype)),
               "misaligned pointer");
  ChooseGradArgs a{logits, dtype, idx, dw, (int)T, (int)E, (int)k, score_func, renormalize, route_scale, dlogits};
  const int64_t per = (E + 63) / 64;
  const dim3 grid((unsigned)((T + 3) / 4)), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (per <= 2) hipLaunchKernelGGL(k_route_experts_grad<2>, grid, block, 0, s, a);
  else if (per <= 4) hipLaunchKernelGGL(k_route_experts_grad<4>, grid, block, 0, s, a);
  else if (per <= 6) hipLaunchKernelGGL(k_route_experts_grad<6>, grid, block, 0, s, a);
  else if (per <= 8) hipLaunchKernelGGL(k_route_experts_grad<8>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(k_route_experts_grad<16>, grid, block, 0, s, a);
  return launch_status("keep_route_experts_grad");
}
