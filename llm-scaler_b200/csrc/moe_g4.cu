// The 4-bit expert layer of many tokens for given routes: the pairs (token, expert) sorted by expert, the tokens' rows copied into that order, a grouped GEMM with SiLU * mul
// in its epilogue, a grouped GEMM whose outputs are multiplied by the routes' weights, the sum of each token's rows.
//
// h and the weighted outputs have 16 bits in between: h because it is the second product's operand; the outputs, one rounding each before the sum of top_k of them,
// because they are read and written once (67 M values for 4096 tokens, top-8, H = 2048).  An expert's rows come in any order, which changes no bits: a row's sums depend on the
// expert and the output alone, not on the tile that it is in.
//
// Each kernel lets the next begin only when all before itself are done, so that the GEMMs read the tile list, weights and scales before the tokens are there (311 tokens of 64 experts
// 127.8 -> 121.1 us, 118.1 now; 4096 of 128 422 -> 387).
#include "i8.cuh"
#include "g4.cuh"

namespace b2q {
namespace g4m {
struct Copies {
  const int32_t *ids, *place, *base; const float* weights;
  int32_t* rows; float* row_w;                             // of pairs; of rows
  int k, E, run;
};

// A CTA per token: its row to the row of each of its pairs, the values of every eight in the order that the grouped kernel wants.
__global__ void __launch_bounds__(256) g4_copies_kernel(const uint4* x, uint4* to, int per, const Copies c) {
  __shared__ int rows[32];
  grid_dep_wait();
  grid_dep_release();                                      // in this order: the next kernel may then read the tile list and weights at once
  const int t = blockIdx.x;
  if (threadIdx.x < c.k) {
    const int64_t pair = (int64_t)t * c.k + threadIdx.x;
    const int id = __ldcg(c.ids + pair);
    int row = -1;
    if ((uint32_t)id < (uint32_t)c.E) {
      row = __ldcg(c.base + (int64_t)(t / c.run) * c.E + id) + __ldcg(c.place + pair);
      c.row_w[row] = __ldcg(c.weights + pair);
    }
    c.rows[pair] = row;
    rows[threadIdx.x] = row;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < per; i += 256) {
    const uint4 v = ld_vec(x + (int64_t)t * per + i);
    const uint4 o = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
    for (int s = 0; s < c.k; ++s)
      if (rows[s] >= 0) to[(int64_t)rows[s] * per + i] = o;
  }
}

struct Outputs {                                           // what the outputs are made of: h by row, the experts' matrices, the pairs' experts and weights
  const uint16_t* h; const uint8_t* w; const uint16_t* s; const uint8_t* z; const int32_t* ids; const float* weights; int I, G;
};
template <bool BF16> __device__ __forceinline__ float half_f(uint32_t raw) { return scalar_from_raw(raw, BF16 ? B2Q_BF16 : B2Q_F16); }
// Expert e's output n of row r of h, in fp32.
template <bool BF16> __device__ __forceinline__ float output(const Outputs& of, int64_t r, int64_t e, int H, int n) {
  const uint16_t* h = of.h + r * of.I;
  const uint8_t* w = of.w + (e * H + n) * (of.I / 2);
  const int groups = of.I / of.G;
  float sum = 0.f;
#pragma unroll 1
  for (int g = 0; g < groups; ++g) {
    const int64_t at = (e * groups + g) * H + n;
    const float zero = of.z ? (float)of.z[at] : 8.f;
    float d = 0.f;
#pragma unroll 1
    for (int k = g * of.G; k < (g + 1) * of.G; k += 8) {
      const uint4 v = ld_vec(h + k);
      const uint32_t q = *reinterpret_cast<const uint32_t*>(w + k / 2), x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {                        // h has them as g4_position says
        d = fmaf(half_f<BF16>(x[j] & 0xFFFFu), (float)(q >> 4 * j & 15u) - zero, d);
        d = fmaf(half_f<BF16>(x[j] >> 16), (float)(q >> (4 * j + 16) & 15u) - zero, d);
      }
    }
    sum = fmaf(half_f<BF16>(of.s[at]), d, sum);
  }
  return sum;
}
// Eight columns n of token t once more, with every weighted output that is infinite in y made anew.
template <bool BF16> __device__ __forceinline__ void sum_again(const uint16_t* y, const int32_t* rows, const Outputs& of, uint16_t* out, int64_t t, int n, int H, int k) {
#pragma unroll 1
  for (int j = n; j < n + 8; ++j) {
    float acc = 0.f;
#pragma unroll 1
    for (int s = 0; s < k; ++s) {
      const int64_t pair = t * k + s, r = __ldcg(rows + pair);
      if (r < 0) continue;
      float f = half_f<BF16>(__ldcg(reinterpret_cast<const unsigned short*>(y) + r * H + j));
      if (fabsf(f) == INFINITY) f = __ldcg(of.weights + pair) * output<BF16>(of, r, __ldcg(of.ids + pair), H, j);
      acc += f;
    }
    out[t * H + j] = (uint16_t)pack2<BF16>(acc, 0.f);
  }
}

// A weighted output that its 16 bits cannot hold (fp16 beyond 65504) would make a sum infinite that is not, and is not so for few tokens, whose outputs stay in fp32: where a thread's
// sums are not finite, it adds them up again and takes such outputs from h.
template <bool BF16> __global__ void __launch_bounds__(256) g4_sum_kernel(const uint4* y, const int32_t* rows, uint4* out, int per, int k, const Outputs of) {
  constexpr int AT_ONCE = 8;
  grid_dep_enter();
  const int64_t t = blockIdx.x;
  float none = 0.f;                                        // NaN once a sum of this thread's was not finite
  for (int c = threadIdx.x; c < per; c += 256) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < k; s0 += AT_ONCE) {
      uint4 v[AT_ONCE];
      int32_t r[AT_ONCE];
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) r[s] = s0 + s < k ? __ldcg(rows + t * k + s0 + s) : -1;
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) v[s] = r[s] >= 0 ? __ldcg(y + (int64_t)r[s] * per + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) {
        const uint32_t e[4] = {v[s].x, v[s].y, v[s].z, v[s].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a, b;
          unpack2<BF16>(e[j], a, b);
          acc[2 * j] += a;
          acc[2 * j + 1] += b;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) none = fmaf(acc[j], 0.f, none);
    out[t * per + c] = make_uint4(pack2<BF16>(acc[0], acc[1]), pack2<BF16>(acc[2], acc[3]), pack2<BF16>(acc[4], acc[5]), pack2<BF16>(acc[6], acc[7]));
  }
  if (none != 0.f) {
#pragma unroll 1
    for (int c = threadIdx.x; c < per; c += 256) sum_again<BF16>(reinterpret_cast<const uint16_t*>(y), rows, of, reinterpret_cast<uint16_t*>(out), t, 8 * c, 8 * per, k);
  }
}

struct Parts { uint8_t *place, *rows, *row_w, *base, *offsets, *count, *tiles, *x, *h, *y; size_t total; };
static Parts parts_of(void* ws, const G4MoeArgs& a) {
  Parts p{};
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  size_t at = 0;
  auto take = [&](size_t bytes) { uint8_t* q = base + at; at += (bytes + 255) / 256 * 256; return q; };
  const size_t rows = (size_t)a.T * a.k;
  p.place = take(rows * 4); p.rows = take(rows * 4); p.row_w = take(rows * 4);
  p.base = take((size_t)moe_i8_route_ctas(a.T) * a.E * 4); p.offsets = take((size_t)(a.E + 1) * 4); p.count = take(8);
  p.tiles = take(16 + 8 * (rows / 32 + 1 + a.E));
  p.x = take(rows * a.H * 2); p.h = take(rows * a.I * 2); p.y = take(rows * a.H * 2);
  p.total = at;
  return p;
}
}  // namespace g4m

bool moe_g4_many_fits(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I) {
  const int64_t tile = g4_grouped_tile(T * k, (int)E), tiles = (T * k + tile - 1) / tile + E;
  return tiles * ((I + 127) / 128) <= INT32_MAX / 2 && tiles * ((H + 255) / 256) <= INT32_MAX / 2;
}

size_t moe_g4_many_bytes(const G4MoeArgs& a) { return g4m::parts_of(nullptr, a).total; }

int moe_g4_many(const G4MoeArgs& a, void* scratch, cudaStream_t st) {
  using namespace g4m;
  const Parts p = parts_of(scratch, a);
  const int64_t rows = (int64_t)a.T * a.k;
  const int tile = g4_grouped_tile(rows, a.E), ctas = moe_i8_route_ctas(a.T);
  const bool overlap = tls().overlap_mode > 0;
  int32_t *off = reinterpret_cast<int32_t*>(p.offsets), *tiles = reinterpret_cast<int32_t*>(p.tiles), *out_rows = reinterpret_cast<int32_t*>(p.rows);
  int rc = moe_route_given(a.ids, a.T, a.E, a.k, tile, reinterpret_cast<int32_t*>(p.place), reinterpret_cast<int32_t*>(p.base), off, tiles, p.count, st);
  if (rc) return rc;
  Copies c{};
  c.ids = a.ids; c.place = reinterpret_cast<int32_t*>(p.place); c.base = reinterpret_cast<int32_t*>(p.base); c.weights = a.weights;
  c.rows = out_rows; c.row_w = reinterpret_cast<float*>(p.row_w); c.k = a.k; c.E = a.E; c.run = (a.T + ctas - 1) / ctas;
  launch_overlapped(g4_copies_kernel, dim3(a.T), dim3(256), 0, st, overlap, reinterpret_cast<const uint4*>(a.x), reinterpret_cast<uint4*>(p.x), a.H / 8, c);
  note_launch("g4_copies");
  G4GroupedArgs g{};
  g.x = p.x; g.bf16 = a.bf16; g.w = a.w13; g.scale = a.s13; g.zero = a.z13; g.offsets = off; g.tiles = tiles; g.tile = tile; g.tile_cap = (int)((rows + tile - 1) / tile + a.E); g.E = a.E;
  g.out = p.h; g.rows = (int)rows; g.N = a.I; g.K = a.H; g.G = a.G13; g.gated = true;
  rc = umma_g4_grouped(g, st);
  g.x = p.h; g.w = a.w2; g.scale = a.s2; g.zero = a.z2; g.out_w = c.row_w; g.out = p.y; g.N = a.H; g.K = a.I; g.G = a.G2; g.gated = false;
  if (!rc) rc = umma_g4_grouped(g, st);
  if (rc) return rc;
  const Outputs of{reinterpret_cast<const uint16_t*>(p.h), a.w2, reinterpret_cast<const uint16_t*>(a.s2), a.z2, a.ids, a.weights, a.I, a.G2};
  launch_overlapped(a.bf16 ? g4_sum_kernel<true> : g4_sum_kernel<false>, dim3(a.T), dim3(256), 0, st, overlap, reinterpret_cast<const uint4*>(p.y),
                    (const int32_t*)out_rows, reinterpret_cast<uint4*>(a.out), a.H / 8, a.k, of);
  note_launch("g4_sum");
  return launch_status();
}
}  // namespace b2q
