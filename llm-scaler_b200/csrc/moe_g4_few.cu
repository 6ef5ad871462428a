// The 4-bit expert layer of a few tokens for given routes: two kernels that stream the chosen experts' weights (g4_stream.cuh has the mathematics and the layout), and a sum where
// tokens are more than a handful.
//
// A chain of latencies for one token (128 experts of 2048 x 768, top-8: 18.1 us in a graph, 3.0 of bytes), and no unit's limit for a batch (16 tokens: 70 us, 3.0 TB/s,
// where the linear with the same loop reaches 4.4): three warps to a scheduler, not four, and 1.3 to 1.6 of the 7 cycles between a warp's instructions at barriers (the linear: 0.6), while routes are sorted, tiles found, tokens
// prepared and sums added up and no weight is multiplied; 45 and 41 % of the issue slots are used.  64-bit divisions ahead of the
// first load cost a microsecond a layer, so there are none.  Every CTA sorts the routes by itself, in shared memory: the pairs (token, slot) of an expert form groups of
// up to eight, whose tokens are the columns of one MMA.  A tile is 32 weight rows of one group; CTAs have equal runs of the tiles of all groups, and their
// warps equal runs of the tiles' steps of 128 k, as in the linear.
//  * up: a tile has sixteen gate rows and the sixteen up rows of the same outputs; h = silu(gate) * up goes out in 16 bits, with its largest magnitude per tile, from which the
//    second kernel takes the power of two that it scales a row of h by.  16 bits because h is what a layer of separate linears would hand on, and what the form of many tokens has as its operand.
//  * down: weighted outputs of each pair in fp32, which a third kernel adds up in the order of the slots.  Its weights are on their way before the first kernel is done.
#include <algorithm>
#include "i8.cuh"
#include "g4_stream.cuh"

namespace b2q {
namespace g4f {
using namespace g4s;
// Twelve warps: sixteen were as fast, and leave less room for the columns.
constexpr int WARPS = 12, THREADS = 32 * WARPS, MAX_PAIRS = THREADS, MAX_E = 1024, PER = (MAX_E + THREADS - 1) / THREADS, TOK = 8;
constexpr int MAX_TILES = 64;                              // that are summed up at a time
constexpr int SMEM = 214 * 1024;                           // beside the routes'

struct Params {
  const uint16_t* x; const int32_t* ids; const float* weights;      // x: tokens, or h by pair
  Matrix w; int64_t w_rows, s_expert;                      // rows, scales of an expert
  uint16_t* h; uint32_t* h_max;                            // [pairs, I], [pairs, I / 16]
  float* y; uint16_t* out;                                 // [pairs, N], [T, N]
  int T, E, k, N, K, steps;                                // N: outputs (I, H)
  int columns, groups, cap;                                // columns, groups and tiles that there is room for
  int early;
};

struct Group { int16_t expert, first, count; };            // first, count: of the sorted pairs

struct alignas(16) Shared {
  int ids[MAX_PAIRS];
  int count[MAX_E];                                        // pairs of an expert, then where they begin
  int16_t pairs[MAX_PAIRS];                                // sorted by expert
  Group groups[MAX_PAIRS];
  int warp_sum[WARPS][2];
  int n_groups;
  uint32_t max[MAX_PAIRS];                                 // of a staged column's row
  struct { int16_t group, strip, first, last; } tiles[MAX_TILES];      // of a batch; warps that have units of it
};

// The routes' pairs sorted by expert, those of an expert by their number: all CTAs of both kernels have to agree on which group a pair is in.
__device__ __forceinline__ void sort_routes(Shared& sh, const Params& p) {
  const int n = p.T * p.k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (n <= 32) {                                           // one warp, by counting (1 token, top-8: the layer 19.1 us in a graph, 20.8 with what is below)
    if (warp == 0) {
      int id = lane < n ? __ldcg(p.ids + lane) : -1;
      if ((uint32_t)id >= (uint32_t)p.E) id = -1;
      int at = 0, same = 0, all = 0;                       // pairs in front of this one; of its expert: in front, and in all
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const int other = __shfl_sync(0xffffffffu, id, j);
        all += other == id;
        same += other == id && j < lane;
        at += other >= 0 && other < id;
      }
      at += same;
      const bool first = id >= 0 && same % TOK == 0;
      const uint32_t groups = __reduce_or_sync(0xffffffffu, first ? 1u << at : 0u);
      if (first) sh.groups[__popc(groups & ((1u << at) - 1))] = Group{(int16_t)id, (int16_t)at, (int16_t)min(TOK, all - same)};
      if (id >= 0) sh.pairs[at] = (int16_t)lane;
      if (lane == 0) sh.n_groups = __popc(groups);
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < p.E; e += THREADS) sh.count[e] = 0;
  __syncthreads();
  int id = -1, at = 0;
  if (threadIdx.x < n) {
    id = __ldcg(p.ids + threadIdx.x);
    if ((uint32_t)id >= (uint32_t)p.E) id = -1;
    if (id >= 0) atomicAdd(&sh.count[id], 1);
  }
  sh.ids[threadIdx.x] = id;
  __syncthreads();
  if (id >= 0) {
    for (int j = 0; j < (int)threadIdx.x; j += 4) {
      const int4 v = *reinterpret_cast<const int4*>(sh.ids + j);
      at += (v.x == id) + (v.y == id && j + 1 < (int)threadIdx.x) + (v.z == id && j + 2 < (int)threadIdx.x) + (v.w == id && j + 3 < (int)threadIdx.x);
    }
  }
  // a thread has PER experts
  const int e0 = PER * threadIdx.x;
  int c[PER], pairs = 0, groups = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = e0 + i < p.E ? sh.count[e0 + i] : 0;
    pairs += c[i];
    groups += (c[i] + TOK - 1) / TOK;
  }
  const int own_pairs = pairs, own_groups = groups;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, pairs, o), b = __shfl_up_sync(0xffffffffu, groups, o);
    if (lane >= o) { pairs += a; groups += b; }
  }
  if (lane == 31) { sh.warp_sum[warp][0] = pairs; sh.warp_sum[warp][1] = groups; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { pairs += sh.warp_sum[w][0]; groups += sh.warp_sum[w][1]; }
  if (threadIdx.x == THREADS - 1) sh.n_groups = groups;
  int first = pairs - own_pairs, to_group = groups - own_groups;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (e0 + i < p.E) sh.count[e0 + i] = first;
    for (int j = 0; j < c[i]; j += TOK) sh.groups[to_group++] = Group{(int16_t)(e0 + i), (int16_t)(first + j), (int16_t)min(TOK, c[i] - j)};
    first += c[i];
  }
  __syncthreads();
  if (threadIdx.x < n) {
    if (id >= 0) sh.pairs[sh.count[id] + at] = (int16_t)threadIdx.x;
  }
  __syncthreads();
}

template <int VEC, bool BF16, bool UP, bool PART>
__global__ void __launch_bounds__(THREADS, 1) g4_experts_kernel(const Params p) {
  constexpr int G = 32 * VEC, GS = STEP / G;               // groups of k in a step
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int steps = p.steps, group_xg = steps * GS * TOK;  // group sums of a group's columns: [steps * GS][8]
  uint8_t* xs = smem + WARPS * WARP_BYTES;                 // [columns][steps][256], then [groups][group_xg]
  float* xg = reinterpret_cast<float*>(xs + (size_t)p.columns * steps * 256);
  float* slots = xg + p.groups * group_xg;                 // [cap + WARPS][ROWS][TOK]

  // up lets the next kernel begin only when it has itself seen that all before it is done: that one may then read the routes, and its weights, while up runs
  bool waited = UP || !p.early;
  if (waited) grid_dep_wait();
  grid_dep_release();
  sort_routes(sh, p);

  // this CTA's tiles: strip by strip of every group in turn
  constexpr int STRIP = UP ? 16 : 32;                      // outputs of a tile
  const int strips = (p.N + STRIP - 1) / STRIP, all = sh.n_groups * strips;
  const int share = all / (int)gridDim.x, more = all - share * (int)gridDim.x, begin = (int)blockIdx.x * share + min((int)blockIdx.x, more), end = begin + share + ((int)blockIdx.x < more);
  int cap = end - begin;
  if (cap > p.cap) { const int batches = (cap + p.cap - 1) / p.cap; cap = (cap + batches - 1) / batches; }
  const uint32_t ring = smem_addr(smem) + warp * WARP_BYTES;

  for (int b0 = begin; b0 < end;) {
    // a batch: tiles whose groups' columns and sums fit
    const int ga = b0 / strips;
    int gb = ga + 1, columns = sh.groups[ga].count;
    int b1 = min(min(end, gb * strips), b0 + cap);
    while (b1 == gb * strips && b1 < end && b1 - b0 < cap && columns + sh.groups[gb].count <= p.columns && gb - ga < p.groups) {
      columns += sh.groups[gb].count;
      ++gb;
      b1 = min(min(end, gb * strips), b0 + cap);
    }
    const int pair0 = sh.groups[ga].first;                 // columns are the sorted pairs from here on
    const int tiles = b1 - b0, units = tiles * steps, even = (units + WARPS - 1) / WARPS, run = even > 6 ? (even + 1) / 2 * 2 : even, u0 = min(units, warp * run), u1 = min(units, u0 + run);

    if (threadIdx.x < tiles) {
      const int id = b0 + threadIdx.x, gi = id / strips;
      sh.tiles[threadIdx.x] = {(int16_t)gi, (int16_t)(id - gi * strips), (int16_t)(threadIdx.x * steps / run), (int16_t)(((threadIdx.x + 1) * steps - 1) / run)};
    }
    __syncthreads();
    struct Tiles {
      const Shared& sh; const Params& p; int ga, pair0, group_xg; uint32_t xs, xg;
      __device__ __forceinline__ int rows(int tile, int64_t (&row)[4], uint32_t (&off)[4], int64_t& base) const {
        const int e = sh.groups[sh.tiles[tile].group].expert, r = STRIP * sh.tiles[tile].strip, g = (threadIdx.x & 31) >> 2, left = p.N - r;
        const int64_t first = (int64_t)e * p.w_rows;
        base = e * p.s_expert;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // up: rows 0 to 15 of the tile are gate rows, 16 to 31 up rows, which lie N behind them
          off[i] = UP ? r + g + 8 * (i & 1) + (i >> 1) * p.N : r + min(g + 8 * i, left - 1);
          row[i] = first + off[i];
        }
        return UP || left > 16 ? 2 : 1;
      }
      __device__ __forceinline__ void columns(int tile, uint32_t (&at)[1], uint32_t& x) const {
        const int gi = sh.tiles[tile].group, lane = threadIdx.x & 31;
        const Group gr = sh.groups[gi];
        at[0] = xs + (gr.first - pair0 + min(lane >> 2, gr.count - 1)) * (p.steps * 256);      // columns beyond the group's repeat its last: nobody looks at them
        x = xg + (gi - ga) * group_xg * 4 + 8 * (lane & 3);
      }
    } of{sh, p, ga, pair0, group_xg, smem_addr(xs), smem_addr(xg)};
    Stream<VEC, 1, BF16, PART, Tiles> stream(p.w, of, p.K, steps, 0, u0, u1, ring);
    stream.load(ring);
    if (!waited) { grid_dep_wait(); waited = true; }

    // ---- columns ----
    auto source = [&](int c) {
      const int pair = sh.pairs[pair0 + c];
      return p.x + (int64_t)(UP ? pair / p.k : pair) * p.K;
    };
    const int per = steps * (STEP / 8), total = columns * per;
    const uint32_t inv = 0xFFFFFFFFu / (uint32_t)per + 1;  // i / per = i * inv >> 32 for i < 2^17, 1 < per < 2^14
    constexpr int V = 4;
    uint4 v[V];
    auto fetch_x = [&](int base) {
#pragma unroll
      for (int a = 0; a < V; ++a) {
        const int i = base + a * THREADS + threadIdx.x, c = (int)__umulhi((uint32_t)i, inv), at = 8 * (i - c * per);
        v[a] = i < total && at < p.K ? ld_eight(source(c) + at, true) : make_uint4(0, 0, 0, 0);
      }
    };
    if (UP) {
      for (int c = threadIdx.x; c < columns; c += THREADS) sh.max[c] = 0;
      __syncthreads();
      for (int base = 0; base < total; base += V * THREADS) {
        fetch_x(base);
#pragma unroll
        for (int a = 0; a < V; ++a) {
          const int i = base + a * THREADS + threadIdx.x, c = (int)__umulhi((uint32_t)i, inv);
          if ((i & ~31) >= total) break;                   // whole warps
          uint32_t mx = max_bits(v[a]);                    // a half warp has one column, since `per` is a multiple of 16
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          if (i < total && (lane & 15) == 0) atomicMax(sh.max + c, mx);
        }
      }
    } else {
      const int n = p.K / 16;
      for (int c = warp; c < columns; c += WARPS) {
        const uint32_t* from = p.h_max + (int64_t)sh.pairs[pair0 + c] * n;
        uint32_t mx = 0;
        for (int i = lane; i < n; i += 32) mx = max(mx, __ldcg(from + i));
        mx = __reduce_max_sync(0xffffffffu, mx);
        if (lane == 0) sh.max[c] = mx;
      }
      if (total <= V * THREADS) fetch_x(0);
    }
    __syncthreads();
    for (int base = 0; base < total; base += V * THREADS) {
      if (total > V * THREADS) fetch_x(base);
#pragma unroll
      for (int a = 0; a < V; ++a) {
        const int i = base + a * THREADS + threadIdx.x, c = (int)__umulhi((uint32_t)i, inv), at = i - c * per;
        if ((i & ~31) >= total) break;
        float sum = 0.f;
        int local = 0, gi = ga;                            // the column's place in its group
        if (i < total) {
          while (gi + 1 < gb && pair0 + c >= sh.groups[gi + 1].first) ++gi;
          local = pair0 + c - sh.groups[gi].first;
          *reinterpret_cast<uint4*>(xs + ((size_t)c * steps + (at >> 4)) * 256 + eight_at(at & 15, local)) = scaled_eight<BF16>(v[a], pow2(row_shift<BF16>(sh.max[c])), sum);
        }
#pragma unroll
        for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (i < total && at % (G / 8) == 0) xg[(gi - ga) * group_xg + at / (G / 8) * TOK + local] = sum * 5.9604644775390625e-8f;      // 2^-24
      }
    }
    __syncthreads();

    // ---- products ----
    stream.run(256, GS * TOK * 4, slots, warp);
    __syncthreads();

    // ---- sums of warps in their order ----
    auto total_of = [&](int tl, int r, int c) {            // row r of tile tl, column c of its group
      const float* from = slots + (tl * ROWS + r) * TOK + c;
      float f = 0.f;
      for (int w = sh.tiles[tl].first; w <= sh.tiles[tl].last; ++w) f += from[w * ROWS * TOK];
      return f;
    };
    if constexpr (UP) {
      // sixteen lanes a column: its outputs in this tile
      for (int i = threadIdx.x; i < tiles * 128; i += THREADS) {
        const int tl = i >> 7, c = (i >> 4) & 7, r = i & 15;
        const Group gr = sh.groups[sh.tiles[tl].group];
        if (c >= gr.count) continue;                       // whole half warps
        const int pair = sh.pairs[gr.first + c], shift = row_shift<BF16>(sh.max[gr.first - pair0 + c]), st = sh.tiles[tl].strip;
        const float gate = unshift(total_of(tl, r, c), shift), up = unshift(total_of(tl, r + 16, c), shift);
        const uint16_t bits = to_half<BF16>(gate / (1.f + expf(-gate)) * up);
        uint32_t mx = bits & 0x7FFFu;
        const uint32_t half = 0xFFFFu << (lane & 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(half, mx, o));
        p.h[(int64_t)pair * p.N + 16 * st + r] = bits;
        if (r == 0) p.h_max[(int64_t)pair * (p.N / 16) + st] = mx;
      }
    } else {
      for (int i = threadIdx.x; i < tiles * 256; i += THREADS) {
        const int tl = i >> 8, c = (i >> 5) & 7, r = i & 31, n = 32 * sh.tiles[tl].strip + r;
        const Group gr = sh.groups[sh.tiles[tl].group];
        if (c >= gr.count || n >= p.N) continue;
        const int pair = sh.pairs[gr.first + c];
        p.y[(int64_t)pair * p.N + n] = __ldcg(p.weights + pair) * unshift(total_of(tl, r, c), row_shift<BF16>(sh.max[gr.first - pair0 + c]));
      }
    }
    __syncthreads();                                       // slots and columns are used again
    b0 = b1;
  }
  if (!waited) grid_dep_wait();                            // the kernel behind waits for this one, and so for all before it
}

template <bool BF16> __global__ void __launch_bounds__(256) g4_pairs_sum_kernel(const float* y, const int32_t* ids, uint16_t* out, int N, int k, int E) {
  grid_dep_release();
  grid_dep_wait();
  const int64_t t = blockIdx.y;
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n < N) {
    float f = 0.f;
    for (int s0 = 0; s0 < k; s0 += 8) {                    // requested together
      float v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) v[s] = s0 + s < k && (uint32_t)__ldcg(ids + t * k + s0 + s) < (uint32_t)E ? __ldcg(y + (t * k + s0 + s) * N + n) : 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) f += v[s];
    }
    out[t * N + n] = to_half<BF16>(f);
  }
}

// ---- host ----
// What shared memory has room for: tiles first, as many as a CTA is likely to have, as long as one group's columns fit beside them; then columns, with a group for two of them
// and one more.
struct Room { int columns, groups, cap, smem; };
static int groups_of(int columns) { return columns / 2 + 1; }
static int bytes_of(int columns, int K, int G) { const int steps = (K + STEP - 1) / STEP; return columns * steps * 256 + groups_of(columns) * steps * (STEP / G) * TOK * 4; }
static Room room_for(int pairs, int E, int strips, int K, int G) {
  const int least = std::min(pairs, TOK), groups = std::min(pairs, E + pairs / TOK);
  Room r{};
  r.cap = std::max(8, std::min(MAX_TILES, (int)((int64_t)groups * strips / sm_count()) + 1));
  auto fixed = [](int cap) { return WARPS * WARP_BYTES + (cap + WARPS) * ROWS * TOK * 4; };
  while (r.cap > 8 && fixed(r.cap) + bytes_of(least, K, G) > SMEM) --r.cap;
  for (r.columns = pairs; r.columns > 0 && fixed(r.cap) + bytes_of(r.columns, K, G) > SMEM;) --r.columns;
  if (r.columns < least) r.columns = 0;
  r.groups = groups_of(r.columns);
  r.smem = fixed(r.cap) + bytes_of(r.columns, K, G);
  return r;
}
struct Plan { Room up, down; bool fits; };
static Plan plan(const G4MoeArgs& a) {
  Plan q{};
  const int pairs = a.T * a.k;                             // few_pairs()
  q.up = room_for(pairs, a.E, a.I / 16, a.H, a.G13);
  q.down = room_for(pairs, a.E, (a.H + ROWS - 1) / ROWS, a.I, a.G2);
  q.fits = q.up.columns > 0 && q.down.columns > 0;
  return q;
}
template <int VEC, bool BF16, bool UP, bool PART> static int launch(Params& p, const Room& r, cudaStream_t st) {
  p.columns = r.columns; p.groups = r.groups; p.cap = r.cap;
  auto kern = g4_experts_kernel<VEC, BF16, UP, PART>;
  static thread_local bool configured[16] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return B2Q_ERR_CUDA;
    if (dev < 16) configured[dev] = true;
  }
  launch_overlapped(kern, dim3(sm_count()), dim3(THREADS), r.smem, st, tls().overlap_mode > 0, p);
  note_launch(UP ? "g4_experts_up" : "g4_experts_down");
  return launch_status();
}
template <bool UP> static int by_type(Params& p, bool bf16, int G, const Room& r, cudaStream_t st) {
  const bool part = p.K % STEP != 0;                       // groups of 128 leave no part of a step
  if (G == 128) return bf16 ? launch<4, true, UP, false>(p, r, st) : launch<4, false, UP, false>(p, r, st);
  if (G == 64) {
    if (part) return bf16 ? launch<2, true, UP, true>(p, r, st) : launch<2, false, UP, true>(p, r, st);
    return bf16 ? launch<2, true, UP, false>(p, r, st) : launch<2, false, UP, false>(p, r, st);
  }
  if (part) return bf16 ? launch<1, true, UP, true>(p, r, st) : launch<1, false, UP, true>(p, r, st);
  return bf16 ? launch<1, true, UP, false>(p, r, st) : launch<1, false, UP, false>(p, r, st);
}
static size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
}  // namespace g4f

// Up to five rows per expert (few / many, us; rows per expert in brackets): 128 experts of 2048 x 768, top-8, 16 tokens [1] 67 / 89, 48 [3] 102 / 119; 8 of 4096 x 4096, top-2, 16 [4]
// 70 / 90, 32 [8] 97 / 91; 64 of 2048 x 1408 in groups of 32, top-6, 32 [3] 123 / 124, 60 [5.6] 141 / 127; 16 of 2048 x 2048, top-4, 16 [4] 45 / 59, 32 [8] 57 / 60.
static bool few_pairs(const G4MoeArgs& a) { const int64_t pairs = (int64_t)a.T * a.k; return pairs <= g4f::MAX_PAIRS && pairs <= 5 * (int64_t)a.E; }
bool moe_g4_few_preferred(const G4MoeArgs& a) { return few_pairs(a) && g4f::plan(a).fits; }

size_t moe_g4_few_bytes(const G4MoeArgs& a) {
  if (!few_pairs(a)) return 0;                             // I / 4 bytes more for each pair than the form of many tokens takes
  const size_t pairs = (size_t)a.T * a.k;
  return g4f::align_up(pairs * a.I * 2) + g4f::align_up(pairs * (a.I / 16) * 4) + g4f::align_up(pairs * a.H * 4);
}

int moe_g4_few(const G4MoeArgs& a, void* scratch, cudaStream_t st) {
  using namespace g4f;
  const Plan q = plan(a);
  const size_t pairs = (size_t)a.T * a.k;
  uint8_t* at = reinterpret_cast<uint8_t*>(scratch);
  Params p{};
  p.ids = a.ids; p.weights = a.weights; p.T = a.T; p.E = a.E; p.k = a.k;
  p.h = reinterpret_cast<uint16_t*>(at); at += align_up(pairs * a.I * 2);
  p.h_max = reinterpret_cast<uint32_t*>(at); at += align_up(pairs * (a.I / 16) * 4);
  p.y = reinterpret_cast<float*>(at);
  p.out = reinterpret_cast<uint16_t*>(a.out);
  p.x = reinterpret_cast<const uint16_t*>(a.x);
  p.w = Matrix{a.w13, reinterpret_cast<const uint16_t*>(a.s13), a.z13, a.H / 2, 2 * (int64_t)a.I};
  p.w_rows = 2 * (int64_t)a.I; p.s_expert = (int64_t)(a.H / a.G13) * 2 * a.I;
  p.N = a.I; p.K = a.H; p.steps = (a.H + STEP - 1) / STEP; 
  int rc = by_type<true>(p, a.bf16, a.G13, q.up, st);
  if (rc) return rc;
  p.x = p.h;
  p.w = Matrix{a.w2, reinterpret_cast<const uint16_t*>(a.s2), a.z2, a.I / 2, a.H};
  p.w_rows = a.H; p.s_expert = (int64_t)(a.I / a.G2) * a.H;
  p.N = a.H; p.K = a.I; p.steps = (a.I + STEP - 1) / STEP; 
  p.early = tls().overlap_mode == 2;
  rc = by_type<false>(p, a.bf16, a.G2, q.down, st);
  if (rc) return rc;
  launch_overlapped(a.bf16 ? g4_pairs_sum_kernel<true> : g4_pairs_sum_kernel<false>, dim3((a.H + 255) / 256, a.T), dim3(256), 0, st, tls().overlap_mode > 0, (const float*)p.y, a.ids, p.out, a.H, a.k, a.E);
  note_launch("g4_pairs_sum");
  return launch_status();
}
}  // namespace b2q
