// What the int8 expert layer of many tokens has around its grouped GEMMs: the routing in one launch, and the weighted sum.
//
// Routing.  A CTA routes a run of tokens, a warp each in turn, and counts its pairs per expert in shared memory; the place a pair is counted at
// is its place among the CTA's pairs of that expert.  The last CTA to finish (arrivals.cuh) turns the counts into where each CTA's pairs of an
// expert begin in the sorted order, and lists the tiles.  Where a pair's row is then follows from its expert, its CTA and its place.  Which
// of a CTA's pairs comes first is a matter of chance, and no result depends on it: a row of the sorted order does not see the others.
// 4096 tokens, 128 experts, top-8: five launches of 27 us before (top-k, a stable sort in three, tiles).
//
// Weighted sum.  Memory-bound; a thread has eight columns of a token and requests eight experts' rows at a time, or four in fp32.  An expert's output
// that its 16 bits cannot hold (fp16 beyond 65504) would make a sum infinite that is not: where a thread's sums are not finite, it adds
// them up again and takes such outputs from the codes of h.
#include "arrivals.cuh"
#include "i8.cuh"
#include "i8_route.cuh"

namespace b2q {

namespace i8m {
constexpr int THREADS = 512, WARPS = THREADS / 32, MAX_E = 1024;
constexpr int CHUNKS = 4, SPANS = WARPS / CHUNKS, MAX_CTAS = 64, SPAN = MAX_CTAS / SPANS;      // of the last CTA's work: 128 experts at a time

struct Params {
  const void* logits; int dt;
  int T, E, k, renorm, per_cta, tile;
  float* weights; int32_t *ids, *place;                    // [T * k]
  int32_t *base, *offsets, *tiles;                         // [CTAs, E], [E + 1], {n, pad, (expert, first row) ...}
  Arrivals* count; Arrivals tag; const Arrivals* epoch;
};

template <int PER>
__global__ void __launch_bounds__(THREADS) moe_i8_route_kernel(const Params p) {
  __shared__ int counts[MAX_E];
  __shared__ int part[SPANS][CHUNKS][32];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < p.E; e += THREADS) counts[e] = 0;
  __syncthreads();
  grid_dep_enter();
  const bool alone = gridDim.x == 1;                       // its counts need not leave the SM (16 tokens: 8.2 us otherwise, by itself)
  if (threadIdx.x == 0 && !alone) arrivals_open(p.count, p.tag, p.epoch);
  const int t0 = blockIdx.x * p.per_cta, t1 = min(p.T, t0 + p.per_cta);
  float v[PER];
  if (t0 + warp < t1) i8r::load_logits<PER>(p.logits, p.dt, p.E, t0 + warp, v);
  for (int t = t0 + warp; t < t1; t += WARPS) {
    float now[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) now[j] = v[j];
    if (t + WARPS < t1) i8r::load_logits<PER>(p.logits, p.dt, p.E, t + WARPS, v);
    int id;
    float w;
    i8r::top_k<PER>(now, p.E, p.k, p.renorm != 0, id, w);
    if (lane < p.k) {
      const int64_t pair = (int64_t)t * p.k + lane;
      p.weights[pair] = w;
      p.ids[pair] = id;
      p.place[pair] = id >= 0 ? atomicAdd(&counts[id], 1) : 0;
    }
  }
  __syncthreads();
  if (!alone) {
    for (int e = threadIdx.x; e < p.E; e += THREADS) p.base[(int64_t)blockIdx.x * p.E + e] = counts[e];
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      last = arrivals_last(p.count, gridDim.x - 1);
      __threadfence();
    }
    __syncthreads();
    if (!last) return;
  }

  // ---- the last CTA: where every expert and every CTA's part of it begins.  A warp has 32 experts and a span of CTAs ----
  const int chunk = warp % CHUNKS, span = warp / CHUNKS, ctas = gridDim.x;
  int before = 0, tiles_before = 0;                        // rows and tiles of the experts so far
  int2* list = reinterpret_cast<int2*>(p.tiles + 4);
  for (int e0 = 0; e0 < p.E; e0 += 32 * CHUNKS) {
    const int e = e0 + 32 * chunk + lane;
    int32_t* mine = p.base + (int64_t)span * SPAN * p.E + e;
    int n[SPAN], sum = 0;
#pragma unroll
    for (int i = 0; i < SPAN; ++i) n[i] = e < p.E && span * SPAN + i < ctas ? (alone ? counts[e] : __ldcg(mine + (int64_t)i * p.E)) : 0;
#pragma unroll
    for (int i = 0; i < SPAN; ++i) sum += n[i];
    part[span][chunk][lane] = sum;
    __syncthreads();
    int front = 0, all = 0, begin = before, first_tile = tiles_before;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      int of = 0;                                          // rows of this lane's expert of chunk c
#pragma unroll
      for (int s = 0; s < SPANS; ++s) {
        const int v = part[s][c][lane];
        of += v;
        if (c == chunk && s < span) front += v;
      }
      const int nt = (of + p.tile - 1) / p.tile;
      if (c == chunk) {
        all = of;
        int rows_upto = of, tiles_upto = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, rows_upto, o), y = __shfl_up_sync(0xffffffffu, tiles_upto, o);
          if (lane >= o) { rows_upto += x; tiles_upto += y; }
        }
        begin = before + rows_upto - of;
        first_tile = tiles_before + tiles_upto - nt;
      }
      before += __reduce_add_sync(0xffffffffu, of);
      tiles_before += __reduce_add_sync(0xffffffffu, nt);
    }
    if (e < p.E) {
      if (span == 0) p.offsets[e] = begin;
      for (int i = span; i < (all + p.tile - 1) / p.tile; i += SPANS) list[first_tile + i] = make_int2(e, i * p.tile);
      int at = begin + front;
#pragma unroll
      for (int i = 0; i < SPAN; ++i) {
        if (span * SPAN + i < ctas) mine[(int64_t)i * p.E] = at;
        at += n[i];
      }
    }
    __syncthreads();                                       // part is used again
  }
  if (threadIdx.x == 0) { p.offsets[p.E] = before; p.tiles[0] = tiles_before; }
}

// Eight columns c of token t once more, with every output that is infinite in y made anew.
template <bool BF16> __device__ __forceinline__ void sum_again(const void* y, const float* weights, const int32_t* rows, const I8Outputs& of, int64_t t, int64_t c, int64_t H, int k, uint16_t* out) {
#pragma unroll 1
  for (int j = 0; j < 8; ++j) {
    float acc = 0.f;
#pragma unroll 1
    for (int s = 0; s < k; ++s) {
      const int64_t pair = t * k + s;
      const int32_t r = __ldcg(rows + pair);
      if (r < 0) continue;
      float f = scalar_from_raw(__ldcg(reinterpret_cast<const unsigned short*>(y) + r * H + c + j), BF16 ? B2Q_BF16 : B2Q_F16);
      if (fabsf(f) == INFINITY) {
        const int64_t column = (int64_t)__ldcg(of.ids + pair) * H + c + j;
        const int8_t *q = of.q + (int64_t)r * of.I, *m = of.w + column * of.I;
        int sum = 0;
#pragma unroll 1
        for (int i = 0; i < of.I; i += 16) {
          const uint4 a = ld_vec(q + i), b = ld_vec(m + i);
          sum = __dp4a((int)a.w, (int)b.w, __dp4a((int)a.z, (int)b.z, __dp4a((int)a.y, (int)b.y, __dp4a((int)a.x, (int)b.x, sum))));
        }
        f = i8_scaled(sum, ld_f32(of.s + r), load_scalar(of.ws, column, of.ws_dt));
      }
      acc = fmaf(__ldcg(weights + pair), f, acc);
    }
    out[t * H + c + j] = (uint16_t)pack2<BF16>(acc, 0.f);
  }
}

// F32: y is
template <bool BF16, bool F32>
__global__ void __launch_bounds__(256) moe_i8_sum_kernel(const void* y, const float* weights, const int32_t* rows, uint16_t* out, int64_t total, int H8, int k, const I8Outputs of) {
  constexpr int AT_ONCE = F32 ? 4 : 8;                     // experts whose rows are on their way together
  grid_dep_enter();
  const int64_t H = (int64_t)H8 * 8;
  float none = 0.f;                                        // NaN once a sum of this thread's was not finite (as their largest it cost 4 us of 282)
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t t = i / H8, c = (i - t * H8) * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < k; s0 += AT_ONCE) {
      uint4 v[AT_ONCE][F32 ? 2 : 1];
      float w[AT_ONCE];
      int32_t r[AT_ONCE];
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) r[s] = s0 + s < k ? __ldcg(rows + t * k + s0 + s) : -1;
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) {
        const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(y) + (r[s] * H + c) * (F32 ? 4 : 2));
#pragma unroll
        for (int h = 0; h < (F32 ? 2 : 1); ++h) v[s][h] = r[s] >= 0 ? __ldcg(from + h) : make_uint4(0, 0, 0, 0);
        w[s] = r[s] >= 0 ? __ldcg(weights + t * k + s0 + s) : 0.f;
      }
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) {
        if (r[s] < 0) continue;
        float f[8];
        if constexpr (F32) {
          const uint4 a = v[s][0], b = v[s][1];
          const uint32_t e[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(e[j]);
        } else {
          const uint32_t e[4] = {v[s][0].x, v[s][0].y, v[s][0].z, v[s][0].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) unpack2<BF16>(e[j], f[2 * j], f[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = fmaf(w[s], f[j], acc[j]);
      }
    }
    if constexpr (!F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) none = fmaf(acc[j], 0.f, none);
    }
    *reinterpret_cast<uint4*>(out + t * H + c) =
        make_uint4(pack2<BF16>(acc[0], acc[1]), pack2<BF16>(acc[2], acc[3]), pack2<BF16>(acc[4], acc[5]), pack2<BF16>(acc[6], acc[7]));
  }
  if constexpr (!F32) {
    if (none != 0.f) {
#pragma unroll 1
      for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) sum_again<BF16>(y, weights, rows, of, i / H8, i % H8 * 8, H, k, out);
    }
  }
}
}  // namespace i8m

int moe_i8_route_ctas(int64_t T) {
  const int64_t n = (T + 15) / 16;
  return (int)(n < i8m::MAX_CTAS ? n : i8m::MAX_CTAS);
}

int moe_i8_route(const void* logits, int dt, int64_t T, int E, int k, bool renorm, int tile, float* weights, int32_t* ids, int32_t* place, int32_t* base,
                 int32_t* offsets, int32_t* tiles, void* count, cudaStream_t st) {
  using namespace i8m;
  Params p{};
  p.logits = logits; p.dt = dt; p.T = (int)T; p.E = E; p.k = k; p.renorm = renorm; p.tile = tile;
  p.weights = weights; p.ids = ids; p.place = place; p.base = base; p.offsets = offsets; p.tiles = tiles;
  p.count = reinterpret_cast<Arrivals*>(count); p.tag = arrivals_tag(); p.epoch = arrivals_epoch();
  if (!p.epoch) return B2Q_ERR_CUDA;
  const int ctas = moe_i8_route_ctas(T);
  p.per_cta = (int)((T + ctas - 1) / ctas);
  auto go = [&](void (*kern)(const Params)) { launch_overlapped(kern, dim3(ctas), dim3(THREADS), 0, st, tls().overlap_mode > 0, p); };
  if (E <= 128) go(moe_i8_route_kernel<4>);
  else if (E <= 256) go(moe_i8_route_kernel<8>);
  else go(moe_i8_route_kernel<32>);
  note_launch("moe_i8_route");
  return launch_status();
}

int moe_i8_sum(const void* y, bool y_f32, const float* weights, const int32_t* rows, const I8Outputs& of, void* out, bool bf16, int64_t T, int k, int H, cudaStream_t st) {
  const int64_t total = T * (H / 8);
  const int64_t g = (total + 255) / 256;
  const dim3 grid((unsigned)(g < 148 * 8 ? g : 148 * 8));
  auto go = [&](auto kern) { launch_overlapped(kern, grid, dim3(256), 0, st, tls().overlap_mode > 0, y, weights, rows, reinterpret_cast<uint16_t*>(out), total, H / 8, k, of); };
  if (y_f32) { if (bf16) go(i8m::moe_i8_sum_kernel<true, true>); else go(i8m::moe_i8_sum_kernel<false, true>); }
  else { if (bf16) go(i8m::moe_i8_sum_kernel<true, false>); else go(i8m::moe_i8_sum_kernel<false, false>); }
  note_launch("moe_i8_sum");
  return launch_status();
}

}  // namespace b2q
