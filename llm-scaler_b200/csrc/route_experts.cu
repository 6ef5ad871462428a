// Which experts a token goes to, and with what weights: the top k of its router logits, by softmax or sigmoid scores, optionally with a bias per
// expert that only the choice sees, and within the best groups of experts.
//
// Choices are exact.  Without a bias an expert's key is its logit, since both scores grow with it; with one, score + bias in 64 bits, as are
// the scores that a group's two best add up to.  So no rounding of the scores decides between two experts, and equal keys go to the lowest index.
// Weights are fp32, of the scores without the bias.
//
// Latency-bound: a warp per token, its logits in registers, k rounds of a warp-wide maximum.
#include "g4.cuh"

namespace b2q {
namespace rex {
constexpr int WARPS = 4;
using Key = unsigned long long;

struct Params {
  const void* logits; int dt; int64_t ldl;
  const void* bias; int bias_dt;
  float* weights; int32_t* ids;
  int T, E, k, groups, size, top_groups, renorm;           // size: experts per group
  float scale;
};

// Larger values have larger keys, equal ones equal keys; -inf and NaN, which are never chosen, have key 0.
__device__ __forceinline__ Key key_of(double v) {
  if (!(v > -INFINITY)) return 0;
  const Key u = (Key)__double_as_longlong(v + 0.0);        // -0 becomes +0
  return (u >> 63) ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ Key warp_max(Key v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (Key)hi << 32 | lo;
}
__device__ __forceinline__ double value_of(Key k) {        // of a key that is not 0
  return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
}

template <int PER, bool SIGMOID, bool BIAS, bool GROUPS, bool TOP2>
__global__ void __launch_bounds__(32 * WARPS) route_experts_kernel(const Params p) {
  const int lane = threadIdx.x & 31, t = blockIdx.x * WARPS + (threadIdx.x >> 5);
  grid_dep_release();
  grid_dep_wait();
  if (t >= p.T) return;
  const int64_t row = (int64_t)t * p.ldl;
  float v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    v[j] = e < p.E ? load_scalar(p.logits, row + e, p.dt) : -INFINITY;
  }
  float mx = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    mx = fmaxf(mx, v[j]);
    bad = bad || !(v[j] < INFINITY);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  bad = __any_sync(0xffffffffu, bad) || mx == -INFINITY;

  constexpr bool SCORES = BIAS || (GROUPS && TOP2);
  double s[SCORES ? PER : 1];
  if constexpr (SCORES) {
    double sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (SIGMOID) s[j] = 1.0 / (1.0 + exp(-(double)v[j]));
      else { s[j] = exp((double)v[j] - (double)mx); sum += s[j]; }
    }
    if (!SIGMOID) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
      for (int j = 0; j < PER; ++j) s[j] /= sum;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = lane + 32 * j;
      if (BIAS && e < p.E) s[j] += (double)load_scalar(p.bias, e, p.bias_dt);
      if (v[j] == -INFINITY) s[j] = -INFINITY;             // an expert that is masked out
    }
  }
  Key key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) key[j] = key_of(BIAS ? s[j] : (double)v[j]);

  if constexpr (GROUPS) {
    Key mine = 0;                                          // lane g: of group g
    for (int g = 0; g < p.groups; ++g) {
      const int lo = g * p.size, hi = lo + p.size;
      Key a = 0, b = 0;                                    // the two largest
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int e = lane + 32 * j;
        Key c = e >= lo && e < hi ? (TOP2 ? key_of(s[j]) : key[j]) : 0;
        b = max(b, min(a, c));
        a = max(a, c);
      }
      Key best = warp_max(a);
      if (TOP2 && p.size > 1) {
        const uint32_t who = __ballot_sync(0xffffffffu, a == best);
        if (lane == __ffs(who) - 1) a = b;
        const Key second = warp_max(a);
        best = best && second ? key_of(value_of(best) + value_of(second)) : 0;
      }
      if (lane == g) mine = best;
    }
    uint32_t keep = 0;
    for (int i = 0; i < p.top_groups; ++i) {
      const Key best = warp_max(mine);
      if (best == 0) break;
      const int g = __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1;
      keep |= 1u << g;
      if (lane == g) mine = 0;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = lane + 32 * j;
      if (e < p.E && !(keep >> (e / p.size) & 1u)) key[j] = 0;
    }
  }

  int id = -1;
  for (int i = 0; i < p.k; ++i) {
    Key best = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) best = max(best, key[j]);
    best = warp_max(best);
    if (best == 0) break;
    uint32_t e = 0xFFFFu;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j)
      if (key[j] == best) e = lane + 32 * j;
    e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j == (int)e) key[j] = 0;
    if (lane == i) id = (int)e;
  }
  if (bad) id = -1;

  // Scores of the chosen.  Renormalised, they are taken relative to the largest where that is below a half, so that logits far below zero do not all
  // become zero.
  const float l = id >= 0 ? load_scalar(p.logits, row + id, p.dt) : -INFINITY;
  float w = 0.f;
  if (SIGMOID) {
    float top = l;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float c = p.renorm ? fminf(top, 0.f) : 0.f;
    if (id >= 0) w = l < 0.f ? expf(l - c) / (1.f + expf(l)) : 1.f / (1.f + expf(-l));
  } else {
    float top = l;
    if (p.renorm) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    } else {
      top = mx;
    }
    if (id >= 0) w = expf(l - top);
  }
  float sum = 1.f;
  if (p.renorm) {
    sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  } else if (!SIGMOID) {
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += expf(v[j] - mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (lane < p.k) {
    p.weights[(int64_t)t * p.k + lane] = id >= 0 ? w / sum * p.scale : 0.f;
    p.ids[(int64_t)t * p.k + lane] = id;
  }
}

template <int PER, bool SIGMOID> static void pick(const Params& p, bool groups, bool top2, cudaStream_t st) {
  auto go = [&](void (*kern)(const Params)) {
    launch_overlapped(kern, dim3((p.T + WARPS - 1) / WARPS), dim3(32 * WARPS), 0, st, tls().overlap_mode > 0, p);
  };
  if (!groups) return p.bias ? go(route_experts_kernel<PER, SIGMOID, true, false, false>) : go(route_experts_kernel<PER, SIGMOID, false, false, false>);
  if (top2) return p.bias ? go(route_experts_kernel<PER, SIGMOID, true, true, true>) : go(route_experts_kernel<PER, SIGMOID, false, true, true>);
  return p.bias ? go(route_experts_kernel<PER, SIGMOID, true, true, false>) : go(route_experts_kernel<PER, SIGMOID, false, true, false>);
}
template <bool SIGMOID> static void by_experts(const Params& p, bool groups, bool top2, cudaStream_t st) {
  if (p.E <= 64) return pick<2, SIGMOID>(p, groups, top2, st);
  if (p.E <= 128) return pick<4, SIGMOID>(p, groups, top2, st);
  if (p.E <= 256) return pick<8, SIGMOID>(p, groups, top2, st);
  if (p.E <= 512) return pick<16, SIGMOID>(p, groups, top2, st);
  pick<32, SIGMOID>(p, groups, top2, st);
}
}  // namespace rex

int route_experts(const RouteExpertsArgs& a, cudaStream_t st) {
  rex::Params p{a.logits, a.dtype, a.ldl, a.bias, a.bias_dtype, a.weights, a.ids, a.T, a.E, a.k, a.groups, a.E / a.groups, a.top_groups, a.renorm, a.scale};
  const bool groups = a.groups > 1 && a.top_groups < a.groups;
  if (a.sigmoid) rex::by_experts<true>(p, groups, a.top2, st);
  else rex::by_experts<false>(p, groups, a.top2, st);
  note_launch("route_experts");
  return launch_status();
}
}  // namespace b2q
