// What expert routing and the layers of 4-bit group-quantised weights share: their host interface.
#pragma once
#include "common.cuh"

namespace b2q {

int sm_count();                                            // of the current device; 148 where there is none

struct RouteExpertsArgs {
  const void* logits; int dtype; int64_t ldl;
  const void* bias; int bias_dtype;                        // [E] or null
  float* weights; int32_t* ids;                            // [T, k]
  int T, E, k, groups, top_groups;
  bool sigmoid, top2, renorm;
  float scale;
};
int route_experts(const RouteExpertsArgs& a, cudaStream_t st);

// w[n, k] = (q[n, k] - z[k / G, n]) s[k / G, n]; q two to a byte, even k in the low half.  x, s, bias and out are of one 16-bit type.
struct G4LinearArgs {
  const void* x; int64_t ldx; bool bf16;
  const uint8_t* w; const void* scale; const uint8_t* zero;      // zero: null for 8 everywhere
  const void* bias; void* out; int64_t ldo;
  int M, N, K, G;
};
bool g4_stream_fits(int M, int N, int K, int G);           // up to sixteen tokens whose shares fit shared memory
size_t g4_stream_bytes(int M, int N, int K, int G);
int g4_stream_linear(const G4LinearArgs& a, void* scratch, cudaStream_t st);
int g4_tile_linear(const G4LinearArgs& a, cudaStream_t st);

struct G4MoeArgs {
  const void* x; bool bf16;
  const float* weights; const int32_t* ids;                // [T, k]
  const uint8_t* w13; const void* s13; const uint8_t* z13;
  const uint8_t* w2; const void* s2; const uint8_t* z2;
  void* out;
  int T, E, k, H, I, G13, G2;
};
size_t g4_tile_moe_bytes(const G4MoeArgs& a);
int g4_tile_moe(const G4MoeArgs& a, void* scratch, cudaStream_t st);

}  // namespace b2q
