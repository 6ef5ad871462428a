// Top-k of a token's router logits by one warp, for the int8 expert layers: the k largest logits, the lowest index first among equals; their
// softmax over all experts, or over the chosen.  A token whose logits hold a NaN, or have no finite maximum, goes to no expert.
#pragma once
#include "common.cuh"

namespace b2q {
namespace i8r {

// Larger logits have larger keys, equal ones equal keys, none has key 0.
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);             // -0 becomes +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A lane's logits, of experts lane, lane + 32, ...; -inf beyond E.  All are requested before any is looked at.
template <int PER> __device__ __forceinline__ void load_logits(const void* logits, int dt, int E, int tok, float (&v)[PER]) {
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)tok * E;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    v[j] = -INFINITY;
    if (e < E)
      v[j] = dt == B2Q_F32 ? __ldcg(reinterpret_cast<const float*>(logits) + at + e)
                           : scalar_from_raw(__ldcg(reinterpret_cast<const unsigned short*>(logits) + at + e), dt);
  }
}

// Lane s < k: the s-th choice (-1: none) and its weight.
template <int PER> __device__ __forceinline__ void top_k(const float (&v)[PER], int E, int k, bool renorm, int& id, float& weight) {
  const int lane = threadIdx.x & 31;
  uint32_t key[PER];
  float mx = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    mx = fmaxf(mx, v[j]);
    nan = nan || v[j] != v[j];
    key[j] = lane + 32 * j < E ? logit_key(v[j]) : 0u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const bool none = __any_sync(0xffffffffu, nan) || !(fabsf(mx) < INFINITY);
  float sum = 0.f;
  if (!renorm) {
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += expf(v[j] - mx);  // absent experts: exp(-inf) = 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  float mine = 0.f, chosen = 0.f;
  id = -1;
  for (int s = 0; s < k; ++s) {
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    uint32_t e = 0xFFFFu;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j)
      if (key[j] == best) e = lane + 32 * j;
    e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j == (int)e) key[j] = 0;
    const float l = __uint_as_float((best & 0x80000000u) ? best & 0x7FFFFFFFu : ~best), w = expf(l - mx);
    chosen += w;
    if (lane == s) { mine = w; id = (int)e; }
  }
  if (none) id = -1;
  weight = none ? 0.f : mine / (renorm ? chosen : sum);
}

}  // namespace i8r
}  // namespace b2q
