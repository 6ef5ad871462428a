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
bool g4_stream_preferred(int M, int N, int K, int G);           // sixteen tokens at most
size_t g4_stream_bytes(int M, int N, int K, int G);
int g4_stream_linear(const G4LinearArgs& a, void* scratch, cudaStream_t st);

// Many tokens, on tcgen05.  out_w: grouped, what every row of the output is multiplied by.
struct G4GroupedArgs {
  const void* x; bool bf16;                                // rows sorted by expert, k permuted in eights (g4_position)
  const uint8_t* w; const void* scale; const uint8_t* zero;      // [E, N (gated: 2 N), K / 2], [E, K / G, N (2 N)]
  const int32_t* offsets; const int32_t* tiles; int tile, tile_cap, E;      // tile list of this height (g4_grouped_tile)
  const float* out_w; void* out; int rows, N, K, G; bool gated;      // gated: out is silu(gate) * up, its columns permuted in eights
};
size_t umma_g4_bytes(const void* x, int64_t ldx, int M, int N, int K, int G);      // x null: the most that any x takes
int umma_g4_linear(const G4LinearArgs& a, void* scratch, cudaStream_t st);
int g4_grouped_tile(int64_t rows, int E);
int umma_g4_grouped(const G4GroupedArgs& a, cudaStream_t st);
// Where value k of eight is kept for the grouped kernel: its masks take the codes of a word in the order 0, 4, 1, 5, 2, 6, 3, 7.
__host__ __device__ constexpr int g4_position(int k) { return (k & ~7) | (k & 3) << 1 | (k >> 2 & 1); }

struct G4MoeArgs {
  const void* x; bool bf16;
  const float* weights; const int32_t* ids;                // [T, k]
  const uint8_t* w13; const void* s13; const uint8_t* z13;
  const uint8_t* w2; const void* s2; const uint8_t* z2;
  void* out;
  int T, E, k, H, I, G13, G2;
};
bool moe_g4_few_preferred(const G4MoeArgs& a);
size_t moe_g4_few_bytes(const G4MoeArgs& a);               // 0 where it serves with no groups
int moe_g4_few(const G4MoeArgs& a, void* scratch, cudaStream_t st);
bool moe_g4_many_fits(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I);      // its tiles can be counted
size_t moe_g4_many_bytes(const G4MoeArgs& a);
int moe_g4_many(const G4MoeArgs& a, void* scratch, cudaStream_t st);

}  // namespace b2q
