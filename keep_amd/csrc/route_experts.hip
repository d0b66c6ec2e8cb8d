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
// keys in 64 bits. Equal logits under equal biases are equal without a second look; where such a pair is the last winner and the
// first that is not chosen, every key behind them that comes as close has to be their equal too.
//
// The groups are spread over the lanes: LG lanes share a group (the largest power of two with LG groups <= 64), so that a
// group's two largest are found inside its lanes.
//
// Bound by what a wave issues one after another: 8192 tokens read 8.9 MB in all (1.7 us of HBM), and take 8.7 us (256 experts, 8
// of them, sigmoid), of which 2.8 are the rounds of the selection, 12.5 with a bias (one for all and 16-bit logits, whose
// boundaries cut runs of equals: 11.1, and 10.4 without the look behind them), 14 to 15.5 with 8 groups too, of which 4 are kept
// (sqrt(softplus) without either 14.3); 4096 of 384 softmax 6.8, with loads 10.4; one token 4.1 to 4.5. A round is one maximum
// of the wave by lane moves and scalar reads, no LDS: with a round that looked through all of a lane's keys again 8192 tokens
// took 23. Keys in 64 bits throughout would double every move of the selection; so only the tokens that need them take them.
//
// With c = scale / (sum s_i + 1e-20) and p_j = c (g_j - sum g_i s_i / (sum s_i + 1e-20)), the gradient of s_j
// (not renormalised: p_j = scale g_j):
//   softmax: dz_e = s_e ([e chosen] p_e - sum p_j s_j);  sigmoid: p s (1 - s);  sqrt(softplus): p sigmoid(z) / (2 s)
#include "route_dev.h"

namespace keep {

struct ChooseArgs {
  const void* z;
  const float* bias;
  int T, E, k, groups, topk_groups;
  int func, renorm;
  float scale;
  int32_t* idx;
  float* w;
  int32_t* load;  // or null: cleared for k_route_load
};

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

// op over groups of `n` lanes (a power of two), in every one of them.
template <typename Op>
__device__ __forceinline__ void ch_lanes(int n, Op op) {
  // quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror: after each step the lanes so far hold the same value
  if (n > 1) op([](float v) { return rt_dpp_f<0xB1>(v); });
  if (n > 2) op([](float v) { return rt_dpp_f<0x4E>(v); });
  if (n > 4) op([](float v) { return rt_dpp_f<0x141>(v); });
  if (n > 8) op([](float v) { return rt_dpp_f<0x140>(v); });
  if (n > 16) op([](float v) { return __shfl_xor(v, 16, 64); });
  if (n > 32) op([](float v) { return __shfl_xor(v, 32, 64); });
}

__device__ __forceinline__ int ch_min(int v) { return (int)rt_wave_u32<false>((uint32_t)v); }
__device__ __forceinline__ float ch_lane(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// The largest of the lanes' values, as a scalar.
__device__ __forceinline__ uint32_t ch_max(uint32_t v) {
  v = rt_dpp_u32<true, 0xB1>(v);
  v = rt_dpp_u32<true, 0x4E>(v);
  v = rt_dpp_u32<true, 0x141>(v);
  v = rt_dpp_u32<true, 0x140>(v);
  const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return max(max(a, b), max(c, d));
}

// What turns a logit into a score: for the softmax its largest logit and the sum's reciprocal.
struct ChooseScore {
  float m, r;
  __device__ __forceinline__ float of(float z, int func) const {
    if (func == KEEP_SCORE_SOFTMAX) return expf(z - m) * r;
    if (func == KEEP_SCORE_SIGMOID) return __builtin_amdgcn_rcpf(1.f + expf(-z));
    return sqrtf(fmaxf(z, 0.f) + log1pf(expf(-fabsf(z))));
  }
};

// The scores of a lane's n logits (those behind them 0). Those of a softmax row whose logits are all -inf are 0.
template <int PER>
__device__ __forceinline__ ChooseScore ch_scores(const float (&z)[PER], int n, int func, float (&s)[PER]) {
  ChooseScore c{0.f, 0.f};
  if (func == KEEP_SCORE_SOFTMAX) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmaxf(m, z[i]);
    m = rt_wave_reduce(m, true);
    c.m = m == -__builtin_inff() ? 0.f : m;
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = i < n ? expf(z[i] - c.m) : 0.f;
      part += s[i];
    }
    const float sum = rt_wave_reduce(part, false);
    c.r = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] *= c.r;
  } else if (func == KEEP_SCORE_SIGMOID) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = i < n ? c.of(z[i], KEEP_SCORE_SIGMOID) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = i < n ? c.of(z[i], KEEP_SCORE_SQRTSOFTPLUS) : 0.f;
  }
  return c;
}

// The lanes' doubles combined, without the LDS pipe: a token that is chosen in 64 bits shall not hold up the launch (by way of
// LDS, 5 us behind 8192 tokens; 1 to 2).
__device__ __forceinline__ double ch_lane_d(double v, int lane) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
template <typename Op>
__device__ __forceinline__ void ch_rows_d(int n, Op op) {  // inside 16 lanes, as ch_lanes
  if (n > 1) op([](double v) { return rt_dpp_d<0xB1, 0xF>(v); });
  if (n > 2) op([](double v) { return rt_dpp_d<0x4E, 0xF>(v); });
  if (n > 4) op([](double v) { return rt_dpp_d<0x141, 0xF>(v); });
  if (n > 8) op([](double v) { return rt_dpp_d<0x140, 0xF>(v); });
}
__device__ __forceinline__ double ch_wave_max_d(double v) {
  ch_rows_d(16, [&](auto from) { v = fmax(v, from(v)); });
  return fmax(fmax(ch_lane_d(v, 0), ch_lane_d(v, 16)), fmax(ch_lane_d(v, 32), ch_lane_d(v, 48)));
}
__device__ __forceinline__ double ch_wave_sum_d(double v) {
  ch_rows_d(16, [&](auto from) { v += from(v); });
  return (ch_lane_d(v, 0) + ch_lane_d(v, 16)) + (ch_lane_d(v, 32) + ch_lane_d(v, 48));
}

// The choice in 64 bits: lane j < k gets winner j. The logits are read again: the few tokens that come here shall not cost
// the others registers.
template <typename Z, int PER>
__device__ __forceinline__ int ch_exact(const ChooseArgs& a, const ChooseLane& l, int64_t t, int lane) {
  const int n = l.n, first = l.first, lg = l.lg, group = l.group;
  float z[PER];
  double key[PER];
  const double none = -__builtin_inf();
#pragma unroll
  for (int i = 0; i < PER; ++i) z[i] = i < n ? to_float(((const Z*)a.z)[t * a.E + first + i * lg]) : -__builtin_inff();
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
    sum = ch_wave_sum_d(sum);
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
    const auto join = [&](auto from) {
      const double o1 = from(t1), o2 = from(t2);
      t2 = fmax(fmin(t1, o1), fmax(t2, o2));
      t1 = fmax(t1, o1);
    };
    ch_rows_d(lg, join);
    for (int o = 16; o < lg; o <<= 1) join([&](double v) { return __shfl_xor(v, o, 64); });
    double v = a.E > a.groups ? t1 + t2 : t1;
    if (v != v) v = none;
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const double o = ch_lane_d(v, h * lg);
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
    const int e = ch_min(best == top ? at : 0x7fffffff);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e == first + i * lg && i < n) open &= ~(1u << i);
    mine = lane == j ? e : mine;
  }
  return mine;
}

// How far a score formed in fp32 may be from the real one, of the row's largest score. Sigmoid and sqrt(softplus): expf and
// log1pf by a step or two, the sum, the reciprocal or root: under 4 x 2^-23. Softmax: the exponent rounds by |z - m| 2^-24, which
// times e^(z - m) is under 0.4 x 2^-24 of the largest; expf by a step; the sum of up to 32 values a lane and 64 lanes by 40 2^-24.
__device__ __forceinline__ float ch_unsure(int func) { return func == KEEP_SCORE_SOFTMAX ? 0x1p-18f : 0x1p-21f; }

// Rounds of the selection: a lane's keys are sorted once with their experts, a round is the wave's largest head, whose lane
// pops it. Lane j keeps winner j; scores and biases of the winners are read and formed again by their lanes together, and
// neighbours compared there.
template <typename Z, int PER>
__global__ __launch_bounds__(256) void k_route_experts(ChooseArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (a.load && blockIdx.x == 0)
    for (int e = threadIdx.x; e < a.E; e += 256) a.load[e] = 0;
  if (t >= a.T) return;
  const ChooseLane l(a.E, a.groups, lane);
  const Z* row = (const Z*)a.z + t * a.E;
  const bool biased = a.bias != nullptr, grouped = a.topk_groups < a.groups;
  Z raw[PER];
  float z[PER], b[PER], s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) raw[i] = i < l.n ? row[l.first + i * l.lg] : Z{};
#pragma unroll
  for (int i = 0; i < PER; ++i) b[i] = biased && i < l.n ? a.bias[l.first + i * l.lg] : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) z[i] = i < l.n ? to_float(raw[i]) : -__builtin_inff();
  const ChooseScore score = ch_scores<PER>(z, l.n, a.func, s);
  bool sure = true, in = l.n > 0;
  // how far any two keys' scores may be off together
  float unsure = 0.f;
  if (biased || grouped) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmaxf(m, s[i]);
    unsure = 2.f * ch_unsure(a.func) * rt_wave_reduce(m, true);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] += b[i];  // the keys
  }
  if (grouped) {
    const float none = -__builtin_inff();
    float t1 = none, t2 = none;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float v = i < l.n ? s[i] : none;
      t2 = fmaxf(t2, fminf(t1, v));
      t1 = fmaxf(t1, v);
    }
    ch_lanes(l.lg, [&](auto from) {
      const float o1 = from(t1), o2 = from(t2);
      t2 = fmaxf(fminf(t1, o1), fmaxf(t2, o2));
      t1 = fmaxf(t1, o1);
    });
    const bool pair = a.E > a.groups;
    float v = pair ? t1 + t2 : t1;
    if (v != v) v = none;
    // two values' scores, and the roundings of two keys and their sum in each
    const float err = 2.f * unsure + 0x1p-21f * rt_wave_reduce(l.n > 0 ? fabsf(t1) + (pair ? fabsf(t2) : 0.f) : 0.f, true);
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const float o = ch_lane(v, h * l.lg);
      rank += o > v || (o == v && h < l.group) ? 1 : 0;
    }
    in = in && rank < a.topk_groups;
    // the last group that is in and the first that is not
    const uint64_t ma = __ballot(l.group < a.groups && rank == a.topk_groups - 1);
    const uint64_t mb = __ballot(l.group < a.groups && rank == a.topk_groups);
    sure = ma != 0 && mb != 0 && ch_lane(v, __builtin_ctzll(ma ? ma : 1)) - ch_lane(v, __builtin_ctzll(mb ? mb : 1)) > err;
  }
  // without a bias the logits are the keys
  uint32_t key[PER];
  int at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = in && i < l.n ? rt_sortable(biased ? s[i] : z[i]) : 0u;
    at[i] = l.first + i * l.lg;
  }
#pragma unroll
  for (int p = 0; p < PER; ++p) {  // odd-even transposition sort, descending; equal keys keep their order
#pragma unroll
    for (int i = p & 1; i + 1 < PER; i += 2) {
      const bool swap = key[i + 1] > key[i];
      const uint32_t k0 = key[i], k1 = key[i + 1];
      const int e0 = at[i], e1 = at[i + 1];
      key[i] = swap ? k1 : k0;
      key[i + 1] = swap ? k0 : k1;
      at[i] = swap ? e1 : e0;
      at[i + 1] = swap ? e0 : e1;
    }
  }
  int mine = 0;
  uint32_t mykey = 0u;
  const int rounds = min(biased ? a.k + 1 : a.k, a.topk_groups * (a.E / a.groups));
  for (int j = 0; j < rounds; ++j) {
    const uint32_t best = ch_max(key[0]);
    const uint64_t who = __ballot(key[0] == best);
    int owner = __builtin_ctzll(who);
    if (who & (who - 1)) {  // several lanes: the lowest expert
      const int e = ch_min(key[0] == best ? at[0] : 0x7fffffff);
      owner = __builtin_ctzll(__ballot(key[0] == best && at[0] == e));
    }
    const int e = __builtin_amdgcn_readlane(at[0], owner);
    mine = lane == j ? e : mine;
    mykey = lane == j ? best : mykey;
    const uint32_t pop = lane == owner ? 0xffffffffu : 0u;  // (bitfield selects)
#pragma unroll
    for (int i = 0; i + 1 < PER; ++i) {
      key[i] = (key[i + 1] & pop) | (key[i] & ~pop);
      at[i] = (int)(((uint32_t)at[i + 1] & pop) | ((uint32_t)at[i] & ~pop));
    }
    key[PER - 1] &= ~pop;
  }
  const bool chosen = lane < a.k;
  if (biased) {
    // each winner against the next one (lane k: the first that is not chosen); a key further down may be off as far
    const float kw = mykey ? rt_unsortable(mykey) : -__builtin_inff(), kn = __shfl_down(kw, 1, 64);
    const uint64_t close = __ballot(chosen && !(kw - kn > unsure + 0x1p-23f * (fabsf(kw) + fabsf(kn))));
    if (close) {  // equal logits under equal biases are no cause, nor is the end of the experts
      const bool have = mykey != 0u;
      const float zw = have ? to_float(row[mine]) : 0.f, bw = have ? a.bias[mine] : 0.f;
      const float zn = __shfl_down(zw, 1, 64), bn = __shfl_down(bw, 1, 64);
      const bool next = __shfl_down((int)have, 1, 64) != 0;
      bool same = !(close >> lane & 1) || !next || (zw == zn && bw == bn);
      if (close >> (a.k - 1) & 1) {  // the last winner's equal is left out: so must be all that come as close behind it
        const float kl = ch_lane(kw, a.k - 1), zl = ch_lane(zw, a.k - 1), bl = ch_lane(bw, a.k - 1);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float ki = key[i] ? rt_unsortable(key[i]) : -__builtin_inff();
          if (key[i] && !(kl - ki > unsure + 0x1p-23f * (fabsf(kl) + fabsf(ki))))
            same = same && to_float(row[at[i]]) == zl && a.bias[at[i]] == bl;
        }
      }
      sure = sure && __all(same);
    }
  }
  if (!sure) mine = ch_exact<Z, PER>(a, l, t, lane);
  const float zw = !chosen ? 0.f : biased || !sure ? to_float(row[mine]) : rt_unsortable(mykey);
  const float sw = chosen ? score.of(zw, a.func) : 0.f;
  float w = sw;
  if (a.renorm) {
    float total = 0.f;
    for (int j = 0; j < a.k; ++j) total += ch_lane(sw, j);
    w = sw / (total + 1e-20f);
  }
  if (chosen) {
    a.idx[t * a.k + lane] = mine;
    a.w[t * a.k + lane] = w * a.scale;
  }
}

// The tokens of every expert: a block counts a run of routes in LDS and adds its counts. Counted by the tokens' own waves,
// one global addition a route, 24576 routes took 15 us beside the choice's 9; here 4.
constexpr int LOAD_ROUTES = 8192;
__global__ __launch_bounds__(1024) void k_route_load(const int32_t* idx, int64_t routes, int E, int32_t* load) {
  __shared__ int count[64 * RT_MAX_PER_LANE];
  for (int e = threadIdx.x; e < E; e += 1024) count[e] = 0;
  __syncthreads();
  const int64_t r0 = (int64_t)blockIdx.x * LOAD_ROUTES;
#pragma unroll
  for (int i = 0; i < LOAD_ROUTES / 1024; ++i) {
    const int64_t r = r0 + i * 1024 + threadIdx.x;
    if (r < routes) atomicAdd(&count[idx[r]], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += 1024)
    if (count[e]) atomicAdd(load + e, count[e]);
}

struct ChooseGradArgs {
  const void* z;
  const int32_t* idx;
  const float* dw;
  int T, E, k;
  int func, renorm;
  float scale;
  void* dz;
};

template <typename Z, int PER>
__global__ __launch_bounds__(256) void k_route_experts_grad(ChooseGradArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int n = lane < a.E ? (a.E - lane + 63) / 64 : 0;
  const Z* row = (const Z*)a.z + t * a.E;
  Z raw[PER];
  float z[PER], s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) raw[i] = i < n ? row[lane + 64 * i] : Z{};
  // lane j < k: the j-th choice
  int e = lane < a.k ? a.idx[t * a.k + lane] : -1;
  const bool chosen = e >= 0 && e < a.E;
  const float g = chosen ? a.dw[t * a.k + lane] : 0.f;
  const float ze = chosen ? to_float(row[e]) : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) z[i] = i < n ? to_float(raw[i]) : -__builtin_inff();
  const ChooseScore score = ch_scores<PER>(z, n, a.func, s);
  const float se = chosen ? score.of(ze, a.func) : 0.f;
  float p = a.scale * g;
  if (a.renorm) {
    const float total = rt_wave_reduce(se, false) + 1e-20f;
    p = a.scale / total * (g - rt_wave_reduce(g * se, false) / total);
  }
  float dot = 0.f;
  if (a.func == KEEP_SCORE_SOFTMAX) {
    dot = rt_wave_reduce(chosen ? p * se : 0.f, false);
  } else if (a.func == KEEP_SCORE_SIGMOID) {
    p *= score.of(-ze, KEEP_SCORE_SIGMOID);  // 1 - s with its bits where s rounds to 1 (times the score below)
  } else {
    // sigmoid(z) / (2 s) over s; where both vanish, s^2 -> e^z and the slope is s / 2
    p *= se > 0.f ? 0.5f * score.of(ze, KEEP_SCORE_SIGMOID) / se / se : 0.f;
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
    if (i < n) ((Z*)a.dz)[t * a.E + lane + 64 * i] = from_float<Z>(s[i] * d[i]);
}

template <typename Z>
static void choose_launch(const ChooseArgs& a, int64_t per, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + 3) / 4)), block(256);
  if (per <= 1) hipLaunchKernelGGL((k_route_experts<Z, 1>), grid, block, 0, s, a);
  else if (per <= 2) hipLaunchKernelGGL((k_route_experts<Z, 2>), grid, block, 0, s, a);
  else if (per <= 4) hipLaunchKernelGGL((k_route_experts<Z, 4>), grid, block, 0, s, a);
  else if (per <= 6) hipLaunchKernelGGL((k_route_experts<Z, 6>), grid, block, 0, s, a);
  else if (per <= 8) hipLaunchKernelGGL((k_route_experts<Z, 8>), grid, block, 0, s, a);
  else if (per <= 16) hipLaunchKernelGGL((k_route_experts<Z, 16>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_route_experts<Z, 32>), grid, block, 0, s, a);  // groups a little more than a power of two
}

template <typename Z>
static void choose_grad_launch(const ChooseGradArgs& a, int64_t per, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + 3) / 4)), block(256);
  if (per <= 2) hipLaunchKernelGGL((k_route_experts_grad<Z, 2>), grid, block, 0, s, a);
  else if (per <= 4) hipLaunchKernelGGL((k_route_experts_grad<Z, 4>), grid, block, 0, s, a);
  else if (per <= 6) hipLaunchKernelGGL((k_route_experts_grad<Z, 6>), grid, block, 0, s, a);
  else if (per <= 8) hipLaunchKernelGGL((k_route_experts_grad<Z, 8>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_route_experts_grad<Z, 16>), grid, block, 0, s, a);
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
  ChooseArgs a{logits, bias, (int)T, (int)E, (int)k, (int)groups, (int)topk_groups, score_func, renormalize,
               route_scale, idx, w, load};
  int lg = 1;
  while (lg * 2 * groups <= 64) lg *= 2;
  const int64_t per = (E / groups + lg - 1) / lg;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KEEP_F32) choose_launch<float>(a, per, s);
  else if (dtype == KEEP_F16) choose_launch<_Float16>(a, per, s);
  else choose_launch<bf16s>(a, per, s);
  if (load)
    hipLaunchKernelGGL(k_route_load, dim3((unsigned)((T * k + LOAD_ROUTES - 1) / LOAD_ROUTES)), dim3(1024), 0, s, idx, T * k,
                       (int)E, load);
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
  ChooseGradArgs a{logits, idx, dw, (int)T, (int)E, (int)k, score_func, renormalize, route_scale, dlogits};
  const int64_t per = (E + 63) / 64;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KEEP_F32) choose_grad_launch<float>(a, per, s);
  else if (dtype == KEEP_F16) choose_grad_launch<_Float16>(a, per, s);
  else choose_grad_launch<bf16s>(a, per, s);
  return launch_status("keep_route_experts_grad");
}
