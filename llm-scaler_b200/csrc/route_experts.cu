// Which experts a token goes to, and with what weights: the top k of its router logits, by softmax or sigmoid scores, optionally with a bias per
// expert that only the choice sees, and within the best groups of experts.
//
// Choices are exact.  Without a bias an expert's key is its logit, since both scores grow with it; with one, score + bias in 64 bits, as are
// the scores that a group's two best add up to.  So no rounding of the scores decides between two experts, and equal keys go to the lowest index.
// Weights are fp32, of the scores without the bias.
//
// Held by latencies: for many tokens those of loads, arithmetic and exchanges together (4093 tokens of 256 experts: 1090 instructions a token, 47 % of the issue slots), for a few by one chain of exchanges.  A warp per token,
// its logits in registers.  The need-th largest of the lanes' maxima leaves a dozen experts or so, which are then ranked by counting, a lane each; k rounds of a
// warp-wide maximum over all registers took 13.8 us where this takes 11.1 (16384 tokens of 128 experts: 10.5 and 9.5; one of 256: 4.5 and 3.6).  Groups of 32
// experts are registers, whose two best change hands by halves, and are ranked in the same way.
// Scores are made in fp32 first, good to EPS; where no two that the choice depends on are nearer to each other than their errors, it is the one of 64 bits, and
// only the other tokens are done again in those (in 64 bits throughout: 24 us, when the rest took 14).
#include <cfloat>
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

// fp32 values as keys of 32 bits, in the same order; those of -inf and NaN are 0.
__device__ __forceinline__ uint32_t key32(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value32(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k); }      // of a key that is not 0
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ Key as_key(double v, Key) { return key_of(v); }
__device__ __forceinline__ uint32_t as_key(float v, uint32_t) { return key32(v); }
__device__ __forceinline__ double value(Key k) { return value_of(k); }
__device__ __forceinline__ float value(uint32_t k) { return value32(k); }
// The key of what two add up to.  In fp32 a sum below all finite values is the lowest of those and not -inf, which would be no key; apart() then tells it from nothing near it.
__device__ __forceinline__ Key both(Key a, Key b) { return key_of(value_of(a) + value_of(b)); }
__device__ __forceinline__ uint32_t both(uint32_t a, uint32_t b) { return key32(fmaxf(value32(a) + value32(b), -FLT_MAX)); }

// How far the fp32 keys may be off, relative to the larger of 1 and the key.  __expf is good to 2 + 1.17 |x| units of 2^-23, so that a sigmoid's p (1 - p) |x| of it is below 2^-23, the
// quotient's two units are another 2^-23 at most, and the sums with 1 and with the bias are rounded to 2^-24.  A softmax has 2^-22 of its exponential and as much of those that its
// sum is made of, and that sum's roundings: PER a lane, five over lanes, and a reciprocal.
template <bool SIGMOID, int PER> constexpr float EPS = SIGMOID ? 4.76837158203125e-7f : 4.76837158203125e-7f + (PER + 6) * 5.9604644775390625e-8f;      // 2^-21; 2^-24

// Values of experts lane + 32 j; `beyond` from E on.
template <int PER> __device__ __forceinline__ void load_row(float (&v)[PER], const void* from, int64_t at, int dt, int E, float beyond) {
  const int lane = threadIdx.x & 31;
  if (dt == B2Q_F32) {
    const float* q = reinterpret_cast<const float*>(from) + at;
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = lane + 32 * j < E ? __ldcg(q + lane + 32 * j) : beyond;
  } else {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(from) + at;
    uint32_t raw[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) raw[j] = lane + 32 * j < E ? __ldcg(q + lane + 32 * j) : 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = lane + 32 * j < E ? scalar_from_raw(raw[j], dt) : beyond;
  }
}
// exp and 1 / x of the two precisions; the fp32 ones are good to 2^-22, more or less.
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float exp_of(float x) { return __expf(x); }
__device__ __forceinline__ double inverse(double x) { return 1.0 / x; }
__device__ __forceinline__ float inverse(float x) { return __fdividef(1.f, x); }

// The choice of lane i < k, -1 where there is none, from keys (key: of experts lane + 32 j; gkey: what groups add up, with TOP2).  CHECK_GROUPS, CHECK: returns false where keys
// of groups, of experts, that the choice depends on are too near to each other.
template <int PER, bool SIGMOID, bool GROUPS, bool TOP2, bool CHECK_GROUPS, bool CHECK, typename K>
__device__ __forceinline__ bool choose(K (&key)[PER], const K (&gkey)[TOP2 ? PER : 1], const Params& p, int& id) {
  const int lane = threadIdx.x & 31;
  bool sure = true;
  auto apart = [](K a, K b, float times) {                 // a >= b, both there
    const float x = (float)value(a), y = (float)value(b);
    return x - y > times * EPS<SIGMOID, PER> * fmaxf(1.f, fmaxf(fabsf(x), fabsf(y)));
  };
  if constexpr (GROUPS) {
    K mine = 0;                                            // lane g: of group g
    auto of_group = [&](K a, K b) {                        // the two largest of each lane
      K best = warp_max(a);
      if (TOP2 && p.size > 1) {
        const uint32_t who = __ballot_sync(0xffffffffu, a == best);
        if (lane == __ffs(who) - 1) a = b;
        const K second = warp_max(a);
        if (second) best = both(best, second);      // the only one left counts for itself
      }
      return best;
    };
    if (p.size == 32) {                                    // a register each: halves change hands until a lane has one group, then its lanes agree
      K a[PER], b[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) { a[j] = TOP2 ? gkey[TOP2 ? j : 0] : key[j]; b[j] = 0; }
#pragma unroll
      for (int n = PER / 2, o = 16; o > 0; n /= 2, o /= 2) {
        const bool upper = lane & o;
#pragma unroll
        for (int j = 0; j < (n ? n : 1); ++j) {
          const K c = __shfl_xor_sync(0xffffffffu, n && !upper ? a[j + n] : a[j], o);
          const K own = n && upper ? a[j + n] : a[j];
          if (TOP2) {
            const K d = __shfl_xor_sync(0xffffffffu, n && !upper ? b[j + n] : b[j], o);
            b[j] = max(max(n && upper ? b[j + n] : b[j], d), min(own, c));
          }
          a[j] = max(own, c);
        }
      }
      K best = a[0];
      if (TOP2 && b[0]) best = both(best, b[0]);
      mine = __shfl_sync(0xffffffffu, best, lane * (32 / PER) & 31);
      if (lane >= p.groups) mine = 0;
    } else {
      for (int g = 0; g < p.groups; ++g) {
        const int lo = g * p.size, hi = lo + p.size;
        K a = 0, b = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int e = lane + 32 * j;
          const K c = e >= lo && e < hi ? (TOP2 ? gkey[TOP2 ? j : 0] : key[j]) : 0;
          if (TOP2) b = max(b, min(a, c));
          a = max(a, c);
        }
        const K best = of_group(a, b);
        if (lane == g) mine = best;
      }
    }
    int rank = 0;                                          // among the groups; equal ones by their index
#pragma unroll 8
    for (int g = 0; g < p.groups; ++g) {
      const K other = __shfl_sync(0xffffffffu, mine, g);
      rank += other > mine || (other == mine && g < lane);
    }
    if (lane >= p.groups) rank = 32;
    const uint32_t keep = __ballot_sync(0xffffffffu, mine != 0 && rank < p.top_groups);
    if (CHECK_GROUPS) {
      const K last = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, rank == p.top_groups - 1)) - 1);
      const K next = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, rank == p.top_groups)) - 1);
      if (next) sure = apart(last, next, TOP2 ? 4.f : 2.f);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = lane + 32 * j, g = p.size == 32 ? j : e / p.size;
      if (e < p.E && !(keep >> g & 1u)) key[j] = 0;
    }
  }
  id = -1;
  K mine = 0;                                              // lane i: the key of its choice; lane k: of the best that is left
  const int need = p.k + (CHECK ? 1 : 0);
  // The need-th largest of the lanes' maxima (1, if there are fewer) is no larger than the need-th largest of all: what is below it is out.
  K least = 1, top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, key[j]);
  for (int left = need; left > 0;) {
    const K best = warp_max(top);
    least = max(best, (K)1);
    if (best == 0) break;
    left -= __popc(__ballot_sync(0xffffffffu, top == best));
    if (top == best) top = 0;
  }
  // The others, a lane each in the order of their index, are ranked by counting.
  __shared__ struct { K key[32]; int e[32]; } all[WARPS];
  auto& of = all[threadIdx.x >> 5];
  int n = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const bool in = key[j] >= least;
    const uint32_t who = __ballot_sync(0xffffffffu, in);
    const int at = n + __popc(who & ((1u << lane) - 1));
    if (in && at < 32) { of.key[at] = key[j]; of.e[at] = lane + 32 * j; }
    n += __popc(who);
  }
  __syncwarp();
  if (n <= 32) {
    const K own = lane < n ? of.key[lane] : 0;
    const int e = of.e[lane];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const K other = of.key[i];
      rank += other > own || (other == own && i < lane);
    }
    __syncwarp();
    if (lane < n) { of.key[rank] = own; of.e[rank] = e; }
    __syncwarp();
    if (lane < n && lane < need) mine = of.key[lane];
    if (lane < n && lane < p.k) id = of.e[lane];
  } else {                                                 // equal ones, for the most part
    for (int i = 0; i < need; ++i) {
      K best = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) best = max(best, key[j]);
      best = warp_max(best);
      if (best == 0) break;
      if (CHECK && (lane == i || (i == 32 && lane == 31))) {
        if (i == 32) sure = sure && apart(mine, best, 2.f);
        else mine = best;
      }
      if (i == p.k) break;
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
  }
  if (CHECK) {
    const K next = __shfl_down_sync(0xffffffffu, mine, 1);
    if (lane < 31 && mine && next) sure = sure && apart(mine, next, 2.f);
  }
  return sure;
}

// Scores in F, plus bias, of experts lane + 32 j.
template <int PER, bool SIGMOID, bool BIAS, typename F> __device__ __forceinline__ void scores(F (&s)[PER], const float (&v)[PER], float mx, const Params& p) {
  F sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (SIGMOID) s[j] = inverse((F)1 + exp_of(-(F)v[j]));
    else { s[j] = exp_of((F)v[j] - (F)mx); sum += s[j]; }
  }
  if (!SIGMOID) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const F inv = (F)1 / sum;
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] *= inv;
  }
  if (BIAS) {
    float b[PER];
    load_row<PER>(b, p.bias, 0, p.bias_dt, p.E, 0.f);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] += (F)b[j];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (v[j] == -INFINITY) s[j] = -INFINITY;               // an expert that is masked out
}
template <int PER, bool SIGMOID, bool BIAS, bool GROUPS, bool TOP2, bool CHECK, typename F, typename K>
__device__ __forceinline__ bool choose_by_scores(const float (&v)[PER], float mx, const Params& p, int& id) {
  F s[PER];
  scores<PER, SIGMOID, BIAS, F>(s, v, mx, p);
  K key[PER], gkey[TOP2 ? PER : 1];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const K of_score = as_key(s[j], K{});
    if (TOP2) gkey[TOP2 ? j : 0] = of_score;
    key[j] = BIAS ? of_score : as_key((F)v[j], K{});
  }
  // without a bias the keys are the logits themselves, which are exact; 16-bit ones are often equal (4093 tokens of 256 experts, a group's two best: 14.5 us when that was checked, 9.3 now; one token 7.1 and 3.5)
  return choose<PER, SIGMOID, GROUPS, TOP2, CHECK, CHECK && BIAS, K>(key, gkey, p, id);
}
template <int PER, bool SIGMOID, bool BIAS, bool GROUPS, bool TOP2> __device__ __noinline__ int choose_exactly(const float (&v)[PER], float mx, const Params& p) {
  int id;
  choose_by_scores<PER, SIGMOID, BIAS, GROUPS, TOP2, false, double, Key>(v, mx, p, id);
  return id;
}

template <int PER, bool SIGMOID, bool BIAS, bool GROUPS, bool TOP2>
__global__ void __launch_bounds__(32 * WARPS) route_experts_kernel(const Params p) {
  const int lane = threadIdx.x & 31, t = blockIdx.x * WARPS + (threadIdx.x >> 5);
  grid_dep_release();
  grid_dep_wait();
  if (t >= p.T) return;
  const int64_t row = (int64_t)t * p.ldl;
  float v[PER];
  load_row<PER>(v, p.logits, row, p.dt, p.E, -INFINITY);
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

  int id = -1;
  if constexpr (BIAS || (GROUPS && TOP2)) {
    if (!bad) {
      const bool sure = choose_by_scores<PER, SIGMOID, BIAS, GROUPS, TOP2, true, float, uint32_t>(v, mx, p, id);
      if (!__all_sync(0xffffffffu, sure)) id = choose_exactly<PER, SIGMOID, BIAS, GROUPS, TOP2>(v, mx, p);
    }
  } else if (!bad) {
    uint32_t key[PER];
    const uint32_t none[1] = {0};
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = key32(v[j]);
    choose<PER, SIGMOID, GROUPS, false, false, false, uint32_t>(key, none, p, id);
  }

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
