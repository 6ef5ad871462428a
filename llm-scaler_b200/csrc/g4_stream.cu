// Linear of a few tokens on 4-bit group-quantised weights: out[m, n] = sum_g s[g, n] (sum_k x[m, k] q[n, k] - z[g, n] X[m, g]) (+ bias[n]).
//
// The weights are read once, and there is little time to convert them (g4_stream.cuh has the mathematics, the layout and what holds the loop).  A CTA per SM has rows of its own, dealt
// out evenly.  Its units (32 rows of 128 k each) go to its warps in equal runs; a warp's next units are on their way while one is multiplied, and
// nothing in the loop waits for another warp.  A warp leaves its sums of a tile of rows in a slot of shared memory; at the end they are added up in the
// order of warps, so that results are the same every time.  In graphs: 1 x 28672 x 8192 28.1 us (4.4 TB/s), 1 x 2048 x 2048 3.9, 7 x 5120 x 13824 in groups of 64 18.1.  Tiles of sixteen
// rows or fewer count as whole ones: dealt out as halves they made the first 30.3.
//
// The tokens are scaled and permuted by each CTA for itself where that is one round of loads, else by a kernel in front, whose image of shared memory the CTAs
// then fetch with one bulk copy, under the first weights.  Where the image does not fit, a cluster of two or four CTAs has rows together and a share of k each; their sums
// meet in distributed shared memory.
#include <algorithm>
#include "sm100.cuh"
#include "g4_stream.cuh"
#include "umma_gemm.cuh"

namespace b2q {
namespace g4s {
constexpr int MOST_WARPS = 16, THREADS = 32 * MOST_WARPS;      // sixteen warps, or twelve where that many tokens leave no room for more
constexpr int SELF = 4;                                    // eights that a thread prepares at most where a CTA prepares the tokens itself
enum { ST_IMAGE = 961 };

struct Params {
  const uint16_t* x; int64_t ldx; int vec;
  const uint8_t* image; const int* shifts;                 // of the kernel in front, or null
  Matrix w; const uint16_t* bias; uint16_t* out; int64_t ldo;
  int M, N, K, steps;                                      // steps: of all K
  int early;
  int* status;
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// One CTA per token: its row's image and shift.
template <int G, int TT, bool BF16>
__global__ void __launch_bounds__(256) g4_prep_kernel(const uint16_t* x, int64_t ldx, int vec, uint8_t* image, int* shifts, int M, int K, int steps) {
  __shared__ uint32_t warp_max[8];
  grid_dep_release();
  grid_dep_wait();
  constexpr int V = 8;
  const int m = blockIdx.x, n = steps * (STEP / 8);
  const uint16_t* row = x + m * ldx;
  uint4 v[V];
  uint32_t mx = 0;
  for (int base = 0; base < n; base += V * 256) {
#pragma unroll
    for (int a = 0; a < V; ++a) {
      const int c = base + a * 256 + threadIdx.x;
      v[a] = 8 * c < K ? ld_eight(row + 8 * c, vec) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int a = 0; a < V; ++a) mx = max(mx, max_bits(v[a]));
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) mx = max(mx, warp_max[w]);
  const int shift = row_shift<BF16>(mx);
  const float f = pow2(shift);
  if (threadIdx.x == 0) shifts[m] = shift;
  for (int base = 0; base < n; base += V * 256) {
    if (n > V * 256) {
#pragma unroll
      for (int a = 0; a < V; ++a) {
        const int c = base + a * 256 + threadIdx.x;
        v[a] = 8 * c < K ? ld_eight(row + 8 * c, vec) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int a = 0; a < V; ++a) {
      const int c = base + a * 256 + threadIdx.x;
      if ((c & ~31) >= n) break;                           // whole warps
      put_eight<G, TT, BF16>(image, M, m, c, v[a], f, c < n);
    }
  }
}

template <int VEC, int TT, bool BF16, bool PART>
__global__ void __launch_bounds__(THREADS, 1) g4_stream_kernel(const Params p) {
  constexpr int G = 32 * VEC, GS = STEP / G, TOK = 8 * TT;      // GS: groups in a step
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t row_max[TOK];
  __shared__ int shifts[TOK];
  __shared__ __align__(8) unsigned long long bar;
  __shared__ int abort_flag;
  uint32_t C;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  const int rank = (int)sm100::cluster_ctarank();
  const int log_c = (int)C >> 1, cluster = blockIdx.x >> log_c, clusters = gridDim.x >> log_c;      // of 1, 2, 4
  const int s0 = rank * p.steps >> log_c, s1 = (rank + 1) * p.steps >> log_c, steps = s1 - s0;
  const int sb = step_bytes(p.M, G, TT);
  uint8_t* xs = smem + blockDim.x / 32 * WARP_BYTES;       // [steps][step_bytes]
  float* slots = reinterpret_cast<float*>(xs + ((p.steps + (int)C - 1) >> log_c) * sb);      // [tiles + WARPS][ROWS][TOK]

  const int WARPS = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int share = p.N / clusters, more = p.N - share * clusters, r0 = cluster * share + min(cluster, more), rows = share + (cluster < more);
  const int tiles = (rows + ROWS - 1) / ROWS, units = tiles * steps;
  const int run = (units + WARPS - 1) / WARPS, u0 = min(units, warp * run), u1 = min(units, u0 + run);

  grid_dep_release();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    sm100::mbar_init(smem_addr(&bar), 1);
    sm100::fence_barrier_init();
  }
  if (threadIdx.x < TOK) row_max[threadIdx.x] = 0;
  if (!p.early) grid_dep_wait();
  struct Tiles {
    int r0, nrows, g, t, M; uint32_t xs;
    __device__ __forceinline__ int rows(int tile, int64_t (&row)[4], uint32_t (&off)[4], int64_t& base) const {
      base = r0;
#pragma unroll
      for (int i = 0; i < 4; ++i) { off[i] = min(ROWS * tile + g + 8 * i, nrows - 1); row[i] = r0 + off[i]; }
      return nrows - ROWS * tile > 16 ? 2 : 1;
    }
    __device__ __forceinline__ void columns(int, uint32_t (&at)[TT], uint32_t& xg) const {
#pragma unroll
      for (int n = 0; n < TT; ++n) at[n] = xs + min(8 * n + g, M - 1) * STEP * 2;      // columns beyond M repeat the last: nobody looks at them
      xg = xs + M * STEP * 2 + 8 * t;
    }
  } of{r0, rows, g, t, p.M, smem_addr(xs)};
  const uint32_t ring = smem_addr(smem) + warp * WARP_BYTES;
  Stream<VEC, TT, BF16, PART, Tiles> stream(p.w, of, p.K, steps, s0, u0, u1, ring);
  stream.load(ring);
  if (p.early) grid_dep_wait();
  __syncthreads();                                         // the barrier and the maxima
  bool ok = true;
  if (p.image) {
    const uint32_t at = smem_addr(&bar);
    if (threadIdx.x == 0) {
      sm100::mbar_expect_tx(at, steps * sb);
      for (int i = 0; i < steps * sb; i += 32768) sm100::bulk_load(smem_addr(xs) + i, p.image + (int64_t)s0 * sb + i, min(32768, steps * sb - i), at);
    }
    if (threadIdx.x < p.M) shifts[threadIdx.x] = __ldcg(p.shifts + threadIdx.x);
    ok = sm100::mbar_wait_warp(at, 0, &abort_flag, p.status, ST_IMAGE);
    if (!ok && threadIdx.x == 0) sm100::drain_issued(at, 1, 1);
  } else {
    const int per = steps * (STEP / 8), total = p.M * per;
    const uint32_t inv = 0xFFFFFFFFu / (uint32_t)per + 1;  // i / per = i * inv >> 32 for i < 2^17, 1 < per < 2^14
    uint4 v[SELF];
    for (int i = threadIdx.x; i < steps * GS * TOK; i += blockDim.x) reinterpret_cast<float*>(xs + i / (GS * TOK) * sb + p.M * STEP * 2)[i % (GS * TOK)] = 0.f;
#pragma unroll
    for (int a = 0; a < SELF; ++a) {
      const int i = a * blockDim.x + threadIdx.x, m = (int)__umulhi((uint32_t)i, inv), k = 8 * (i - m * per);
      v[a] = i < total && k < p.K ? ld_eight(p.x + m * p.ldx + k, p.vec) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int a = 0; a < SELF; ++a) {
      const int i = a * blockDim.x + threadIdx.x, m = (int)__umulhi((uint32_t)i, inv);
      if ((i & ~31) >= total) break;                       // whole warps
      uint32_t mx = max_bits(v[a]);                        // a half warp has one token, since `per` is a multiple of 16
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (i < total && (lane & 15) == 0) atomicMax(row_max + m, mx);
    }
    __syncthreads();
    if (threadIdx.x < p.M) shifts[threadIdx.x] = row_shift<BF16>(row_max[threadIdx.x]);
#pragma unroll
    for (int a = 0; a < SELF; ++a) {
      const int i = a * blockDim.x + threadIdx.x, m = (int)__umulhi((uint32_t)i, inv);
      if ((i & ~31) >= total) break;
      put_eight<G, TT, BF16>(xs, p.M, m, i - m * per, v[a], pow2(row_shift<BF16>(row_max[i < total ? m : 0])), i < total);
    }
  }
  __syncthreads();

  if (ok) stream.run(sb, sb, slots, warp);
  copy_wait<0>();
  __syncthreads();

  // this CTA's sums, tile by tile, of warps in their order; sixteen lanes have consecutive rows
  auto put = [&](int m, int r, float v) {
    if (p.bias) v += half_f<BF16>(p.bias[r0 + r]);
    p.out[m * p.ldo + r0 + r] = to_half<BF16>(v);
  };
  float* part = reinterpret_cast<float*>(smem);            // [M][rows], where the rings and the tokens were
  const bool alone = C == 1;
  for (int h = warp; h < tiles * 2; h += WARPS) {          // sixteens of rows
    const int tl = h / 2, first = tl * steps / run, last = ((tl + 1) * steps - 1) / run, r = 16 * h + (lane & 15);      // warps that have units of it
    for (int m = lane >> 4; m < p.M; m += 2) {
      const float* from = slots + (tl * ROWS + r - ROWS * tl) * TOK + m;
      float v = 0.f;
      for (int w = first; w <= last; ++w) v += from[w * ROWS * TOK];
      v = unshift(v, shifts[m]);
      if (r < rows) {
        if (alone) put(m, r, v);
        else part[m * rows + r] = v;
      }
    }
  }
  if (!alone) {
    sm100::cluster_sync_all();
    const uint32_t from = smem_addr(part);
    for (int r = rank * 32 + lane; r < rows; r += C * 32) {
      for (int m = warp; m < p.M; m += WARPS) {
        float v = 0.f;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c)
          if (c < C) v += ld_cluster_f32(sm100::map_to_cta(from + (m * rows + r) * 4, c));
        put(m, r, v);
      }
    }
    sm100::cluster_sync_all();                             // nobody leaves while its sums may be read
  }
}

// ---- host ----
constexpr int SMEM = 220 * 1024;
struct Plan { int C, clusters, cap, smem, tt, steps, warps; bool self; };
// Clusters of four that the SMs hold at a time: not all of them can be in one.
static int resident(int C) { return C == 4 ? sm_count() * 7 / 32 : sm_count() / C; }
static Plan plan(int M, int N, int K, int G) {
  Plan q{};
  q.steps = (K + STEP - 1) / STEP;
  q.tt = M <= 8 ? 1 : 2;
  for (q.C = 1; q.C <= 4; q.C *= 2) {
    if (q.C > q.steps) break;
    q.clusters = resident(q.C);
    if (q.clusters > (N + 7) / 8) q.clusters = (N + 7) / 8;
    const int rows = (N + q.clusters - 1) / q.clusters, most = (q.steps + q.C - 1) / q.C;
    q.cap = (rows + ROWS - 1) / ROWS;
    // (fewer where there is little for each to do: 1 x 2048 x 2048 4.6 us with sixteen, 4.15 with twelve; 1 x 28672 x 8192 28.1 and 30.4)
    for (q.warps = (int64_t)q.cap * most >= 4 * MOST_WARPS ? MOST_WARPS : 12; q.warps >= 12; q.warps -= 4) {
      const int64_t front = (int64_t)q.warps * WARP_BYTES + (int64_t)most * step_bytes(M, G, q.tt);
      const int64_t smem = front + (int64_t)(q.cap + q.warps) * ROWS * 8 * q.tt * 4;
      q.self = M * q.steps * (STEP / 8) <= SELF * 32 * q.warps;
      if (q.self && q.C > 1) break;
      if (smem <= SMEM && (q.C == 1 || (int64_t)M * rows * 4 <= front)) { q.smem = (int)smem; return q; }
    }
  }
  return q;
}

template <int VEC, int TT, bool BF16, bool PART> static int launch(Params& p, const Plan& q, cudaStream_t st) {
  const bool overlap = tls().overlap_mode > 0;
  if (p.image) {
    launch_overlapped(g4_prep_kernel<32 * VEC, TT, BF16>, dim3(p.M), dim3(256), 0, st, overlap, p.x, p.ldx, p.vec, const_cast<uint8_t*>(p.image), const_cast<int*>(p.shifts), p.M, p.K, p.steps);
    note_launch("g4_prep");
  }
  auto kern = g4_stream_kernel<VEC, TT, BF16, PART>;
  static thread_local bool configured[16] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return B2Q_ERR_CUDA;
    if (dev < 16) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(q.clusters * q.C); cfg.blockDim = dim3(32 * q.warps); cfg.dynamicSmemBytes = q.smem; cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (q.C > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = q.C; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (overlap) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at; cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kern, p);                       // launch_status() reports
  note_launch("g4_stream");
  return launch_status();
}
template <int VEC, bool BF16, bool PART> static int by_size(Params& p, const Plan& q, cudaStream_t st) {
  return q.tt == 1 ? launch<VEC, 1, BF16, PART>(p, q, st) : launch<VEC, 2, BF16, PART>(p, q, st);
}
template <int VEC, bool PART> static int by_type(Params& p, bool bf16, const Plan& q, cudaStream_t st) {
  return bf16 ? by_size<VEC, true, PART>(p, q, st) : by_size<VEC, false, PART>(p, q, st);
}
}  // namespace g4s

// Up to eight tokens, and up to sixteen of small layers (here / on tcgen05, us: 16 x 2048 x 2048 7.2 / 8.2, 16 x 1024 x 8192 9.1 / 11.2, 16 x 4096 x 4096 10.8 / 10.3, 12 x 28672 x
// 2048 16.7 / 14.7, 16 x 17408 x 5120 24.0 / 18.8; 8 x 4096 x 4096 7.8 / 10.0).  Eight tokens of a K above some 25000 have no room in shared memory and go to tcgen05, for want of another form: 8 x 4096 x 24576
// 22.6 / 28.4, 7 x 4096 x 28672 25.7 / 32.3, 8 x 4096 x 28672 - / 32.2.
bool g4_stream_preferred(int M, int N, int K, int G) { return M <= (N * (int64_t)K <= 12 << 20 ? 16 : 8) && g4s::plan(M, N, K, G).smem > 0; }

size_t g4_stream_bytes(int M, int N, int K, int G) {
  const g4s::Plan q = g4s::plan(M, N, K, G);
  return q.self ? 0 : (size_t)q.steps * g4s::step_bytes(M, G, q.tt) + 16 * sizeof(int);
}

int g4_stream_linear(const G4LinearArgs& a, void* scratch, cudaStream_t st) {
  using namespace g4s;
  const Plan q = plan(a.M, a.N, a.K, a.G);
  if (!q.smem) return B2Q_ERR_LIMIT;
  Params p{};
  p.x = reinterpret_cast<const uint16_t*>(a.x); p.ldx = a.ldx; p.vec = ((reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(2 * a.ldx)) & 15u) == 0;
  p.w = Matrix{a.w, reinterpret_cast<const uint16_t*>(a.scale), a.zero, a.K / 2, a.N};
  p.bias = reinterpret_cast<const uint16_t*>(a.bias); p.out = reinterpret_cast<uint16_t*>(a.out); p.ldo = a.ldo;
  p.M = a.M; p.N = a.N; p.K = a.K; p.steps = q.steps; p.early = tls().overlap_mode == 2;
  p.status = umma_status_ptr();
  if (!p.status) return B2Q_ERR_CUDA;
  if (!q.self) {
    p.image = reinterpret_cast<const uint8_t*>(scratch);
    p.shifts = reinterpret_cast<const int*>(p.image + (size_t)q.steps * step_bytes(a.M, a.G, q.tt));
  }
  const bool part = a.K % STEP != 0;                       // groups of 128 leave no part of a step
  if (a.G == 128) return by_type<4, false>(p, a.bf16, q, st);
  if (a.G == 64) return part ? by_type<2, true>(p, a.bf16, q, st) : by_type<2, false>(p, a.bf16, q, st);
  return part ? by_type<1, true>(p, a.bf16, q, st) : by_type<1, false>(p, a.bf16, q, st);
}
}  // namespace b2q
