// A whole int8 expert layer of up to sixteen tokens in two kernels:
//   ids, w = top-k of the logits;  h = silu(x W_gate) * (x W_up) per (token, expert) pair;  out = sum of w * (h W_down),
// where x and h meet the int8 weights as int8 codes with one scale per row.
//
// HBM-bound: the chosen experts' matrices, once.  One thread fetches them, eight or sixteen rows at a time, into a ring that fills the SM's
// shared memory: rows that are taken whole are one contiguous run and one untiled bulk copy of exactly the rows that are wanted; pieces of
// longer rows are TMA boxes.  Eight warps feed them to mma.sync m16n8k32 (the up to sixteen pairs of an expert are the MMA's rows, with k permuted
// alike on both sides so that a lane reads sixteen bytes of a row at a time).  A stage is one warp's, whose sums are added up in shared
// memory, in integers, so that no division of the work changes a bit.
//
// Up kernel.  Every CTA routes all tokens and makes all their codes by itself, which costs less than a launch.  The columns j of all chosen
// experts, one expert behind the other, are dealt out evenly to the column; eight columns are eight gate rows and eight up rows.  h is
// written in fp32.  An expert's rows of h become codes as soon as its last CTA has delivered (arrivals.cuh): that one CTA does it.
// Down kernel.  A CTA owns output columns and runs through all chosen experts, so no sum crosses CTAs: the pairs' products add up in the
// order of the slots.  It routes the tokens again rather than wait for the up kernel to tell, and has its first weights on their way
// before that has finished; nothing it reads there is written by a kernel that may still run (the up kernel lets it start only
// behind its own wait).
//
// Every mbarrier wait is bounded; a warp that gives up still goes to the barriers where the others expect it.
#include "arrivals.cuh"
#include "i8.cuh"
#include "sm100.cuh"
#include "umma_gemm.cuh"

namespace b2q {

using namespace sm100;

namespace mi8 {
enum { ST_UP_EMPTY = 901, ST_UP_FULL = 902, ST_DOWN_EMPTY = 903, ST_DOWN_FULL = 904, ST_DOWN_XEMPTY = 905 };
constexpr int WARPS = 8, WORKERS = 32 * WARPS;              // the warps that multiply
constexpr int UP_THREADS = WORKERS + 32, DOWN_THREADS = WORKERS + 64;      // and those that fetch: weights; codes
constexpr int MAX_TOK = I8_STREAM_MAX_TOK, MAX_K = 32, MAX_PAIRS = MAX_TOK * MAX_K, MAX_E = 1024;
constexpr int CODES_MAX = 68 * 1024;                       // bytes of the tokens' codes in the up kernel's shared memory
constexpr int PASS = 16;                                   // groups of eight columns whose sums are held at a time
constexpr int TABLE_MAX = 24 * 1024;                       // bytes of sums in the down kernel's, and of scales
constexpr int PIECE = 2048;                                // longest k of a stage: 256 elements of eight bytes in a TMA box
constexpr int MAX_STAGES = 4 * WARPS, BAR_BYTES = 16 * MAX_STAGES + 16;
constexpr int SMEM_MAX = 232448 - 1024;                    // of a CTA, static part included

struct Params {
  const uint16_t* x; const void* logits; int ldt;
  const int8_t* w13; const void* s13; int s13_dt;
  const int8_t* w2; const void* s2; int s2_dt;
  uint16_t* out;
  int T, E, k, H, I, renorm;
  float* h; int8_t* hq; float* hs;                         // [pairs, I], [pairs, I], [pairs]
  Arrivals* counts; Arrivals tag; const Arrivals* epoch;
  int pitch, row_cap;
  // the ring: k and weight rows of a stage; a multiple of WARPS of them, so that a stage always comes back to the same warp (a parity wait
  // cannot tell the phase it waits for from the one two before)
  int piece, stage_rows, stages, stage_bytes;
  int* status;
};

// Who goes where.  Slots are the chosen experts in the order in which the pairs (token, choice) first name them, the same in every CTA.
struct Route {
  int first[MAX_E];                                        // the first pair that names an expert, then the expert's slot
  int count[MAX_E];
  int16_t expert[MAX_PAIRS];                               // of a pair; -1: none
  int16_t place[MAX_PAIRS];                                // of a pair among its expert's
  float weight[MAX_PAIRS];
  int16_t slot_expert[MAX_PAIRS];
  int16_t slot_first[MAX_PAIRS + 1];                       // into list
  int16_t list[MAX_PAIRS];                                 // pairs by slot
  int slots;
};

// Larger logits have larger keys, equal ones equal keys, none has key 0.
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);             // -0 becomes +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// One warp: the k largest of E logits, the lowest index first among equals; softmax over all or over the chosen.  A token whose logits
// hold a NaN, or have no finite maximum, goes to no expert.
template <int PER> __device__ __forceinline__ void route_token(const Params& p, int tok, Route& r) {
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)tok * p.E;
  float v[PER];
  uint32_t key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    v[j] = -INFINITY;
    if (e < p.E)
      v[j] = p.ldt == B2Q_F32 ? __ldcg(reinterpret_cast<const float*>(p.logits) + at + e)
                              : scalar_from_raw(__ldcg(reinterpret_cast<const unsigned short*>(p.logits) + at + e), p.ldt);
  }
  float mx = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    mx = fmaxf(mx, v[j]);
    nan = nan || v[j] != v[j];
    key[j] = lane + 32 * j < p.E ? logit_key(v[j]) : 0u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const bool none = __any_sync(0xffffffffu, nan) || !(fabsf(mx) < INFINITY);
  float sum = 0.f;
  if (!p.renorm) {
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += expf(v[j] - mx);  // absent experts: exp(-inf) = 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  float mine = 0.f, chosen = 0.f;
  int id = -1;
  for (int s = 0; s < p.k; ++s) {
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
  if (lane < p.k) {
    const int pair = tok * p.k + lane;
    r.expert[pair] = none ? -1 : (int16_t)id;
    r.weight[pair] = none ? 0.f : mine / (p.renorm ? chosen : sum);
    if (!none) {
      atomicMin(&r.first[id], pair);
      r.place[pair] = (int16_t)atomicAdd(&r.count[id], 1);
    }
  }
}

// The whole CTA; barriers inside.  Which place a pair gets among its expert's is a matter of chance and changes no result.
template <int PER> __device__ __forceinline__ void route(const Params& p, Route& r) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pairs = p.T * p.k;
  for (int i = threadIdx.x; i < p.E; i += blockDim.x) { r.first[i] = pairs; r.count[i] = 0; }
  __syncthreads();
  for (int t = warp; t < p.T; t += blockDim.x / 32) route_token<PER>(p, t, r);
  __syncthreads();
  if (warp == 0) {
    int slots = 0, before = 0;
    for (int b = 0; b < pairs; b += 32) {
      const int e = b + lane < pairs ? r.expert[b + lane] : -1;
      const bool names = e >= 0 && r.first[e] == b + lane;
      const unsigned some = __ballot_sync(0xffffffffu, names);
      const int c = names ? r.count[e] : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (names) {
        const int s = slots + __popc(some & ((1u << lane) - 1u));
        r.slot_expert[s] = (int16_t)e;
        r.slot_first[s] = (int16_t)(before + upto - c);
        r.first[e] = s;                                    // a slot is no larger than the pair that named it: nobody looks at it as one again
      }
      slots += __popc(some);
      before += __shfl_sync(0xffffffffu, upto, 31);
      __syncwarp();
    }
    if (lane == 0) { r.slots = slots; r.slot_first[slots] = (int16_t)before; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += blockDim.x)
    if (r.expert[i] >= 0) r.list[r.slot_first[r.first[r.expert[i]]] + r.place[i]] = (int16_t)i;
  __syncthreads();
}

// The CTA that has column c when n columns are dealt out to G CTAs, [b n / G, (b + 1) n / G) to CTA b.
__device__ __forceinline__ int owner(int64_t c, int64_t n, int64_t G) {
  int64_t b = c * G / n;
  while ((b + 1) * n / G <= c) ++b;
  while (b * n / G > c) --b;
  return (int)b;
}

__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory"); }      // the eight warps

// Codes of an expert's rows of h, by the eight warps.  Rows of up to 8192 stay in registers between the maximum and the codes.
__device__ __forceinline__ void quantize_rows(const Params& p, const Route& r, int slot, uint32_t* red) {
  constexpr int V = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n4 = p.I >> 2;
  const bool once = n4 <= V * WORKERS;
  for (int i = r.slot_first[slot]; i < r.slot_first[slot + 1]; ++i) {
    const int pair = r.list[i];
    const float4* h = reinterpret_cast<const float4*>(p.h + (int64_t)pair * p.I);
    float4 v[V];
    auto fetch = [&](int base) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = base + j * WORKERS + threadIdx.x;
        v[j] = c < n4 ? __ldcg(h + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    uint32_t mx = 0;
    for (int base = 0; base < n4; base += V * WORKERS) {
      fetch(base);
#pragma unroll
      for (int j = 0; j < V; ++j)
        mx = max(max(mx, __float_as_uint(v[j].x) & 0x7FFFFFFFu), max(__float_as_uint(v[j].y) & 0x7FFFFFFFu, max(__float_as_uint(v[j].z) & 0x7FFFFFFFu, __float_as_uint(v[j].w) & 0x7FFFFFFFu)));
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) red[warp] = mx;
    __syncwarp();
    meet();
    mx = __reduce_max_sync(0xffffffffu, red[lane & (WARPS - 1)]);
    const bool finite = mx < 0x7F800000u;
    const float a = fmaxf(__uint_as_float(mx), I8_MIN_AMAX), s = 127.f / a;
    if (threadIdx.x == 0) p.hs[pair] = finite ? a / 127.f : __uint_as_float(0x7FC00000u);
    uint32_t* q = reinterpret_cast<uint32_t*>(p.hq + (int64_t)pair * p.I);
    for (int base = 0; base < n4; base += V * WORKERS) {
      if (!once) fetch(base);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = base + j * WORKERS + threadIdx.x;
        const float f[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        if (c < n4) q[c] = finite ? i8_codes4_computed(f, s) : 0u;
      }
    }
    __syncwarp();
    meet();                                                // red is used again
  }
}

__device__ __forceinline__ uint4 lds(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// Eight weight rows at w against up to sixteen rows of codes at xa (rows g) and xb (rows g + 8), len of their k; addresses are the lane's.
__device__ __forceinline__ void multiply(int (&acc)[4], uint32_t w, uint32_t xa, uint32_t xb, bool has_a, bool has_b, int len) {
  const int t16 = 16 * (threadIdx.x & 3);
  int more[4] = {0, 0, 0, 0};                              // two chains, as an MMA takes long to deliver
  auto step = [&](int k, bool in) {
    uint4 a = make_uint4(0, 0, 0, 0), b = a, v = a;
    if (in) v = lds(w + k);
    if (in && has_a) a = lds(xa + k);
    if (in && has_b) b = lds(xb + k);
    mma_s8(acc, a.x, b.x, a.y, b.y, v.x, v.y);
    mma_s8(more, a.z, b.z, a.w, b.w, v.z, v.w);
  };
  const int whole = len & ~63;
#pragma unroll 4
  for (int k = 0; k < whole; k += 64) step(k, true);
  if (whole < len) step(whole, whole + t16 < len);         // the last 64 bytes of a row may be fewer
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] += more[c];
}

template <bool BF16, int PER>
__global__ void __launch_bounds__(UP_THREADS, 1) moe_i8_up_kernel(const __grid_constant__ CUtensorMap tm_w, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Route rt;
  __shared__ I8Tokens tok;
  __shared__ uint32_t red[WARPS];
  __shared__ int last;
  // [ring: eight gate or up rows x piece] [codes: T x pitch] [sums of two passes: 2 x PASS x T x 16] [barriers]
  const uint32_t ring = smem_u32(smem);
  uint8_t* codes = smem + p.stages * p.stage_bytes;
  int* sums = reinterpret_cast<int*>(codes + p.T * p.pitch);
  const uint32_t full = smem_u32(sums + 2 * PASS * p.T * 16), empty = full + 8 * MAX_STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(sums + 2 * PASS * p.T * 16) + 16 * MAX_STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < MAX_TOK) tok.max[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < 2 * PASS * p.T * 16; i += UP_THREADS) sums[i] = 0;
  grid_dep_wait();
  grid_dep_release();                                      // not before the wait: see the down kernel
  route<PER>(p, rt);
  const int64_t n = (int64_t)rt.slots * p.I;               // columns of all slots
  const int64_t G = min((int64_t)gridDim.x, n);            // no CTA without a column
  if (blockIdx.x >= G) return;                             // the whole CTA
  const int64_t c0 = blockIdx.x * n / G, c1 = (blockIdx.x + 1) * n / G;
  const int slot0 = (int)(c0 / p.I), slot1 = (int)((c1 - 1) / p.I);

  // groups of eight columns: those of the first slot's part, then of whole slots; the last slot's part may end early
  const int j0 = (int)(c0 - (int64_t)slot0 * p.I), per_slot = (p.I + 7) / 8;
  const int len0 = (int)min((int64_t)p.I - j0, c1 - c0), groups0 = (len0 + 7) / 8;
  const int end1 = (int)(c1 - (int64_t)slot1 * p.I);       // columns of the last slot end here
  const int groups = slot0 == slot1 ? groups0 : groups0 + (slot1 - slot0 - 1) * per_slot + (end1 + 7) / 8;
  struct Group { int slot, j, n; };                        // n: valid columns
  auto group_at = [&](int i) {
    Group q;
    if (i < groups0) {
      q.slot = slot0; q.j = j0 + 8 * i; q.n = min(8, j0 + len0 - q.j);
    } else {
      const int b = (i - groups0) / per_slot;
      q.slot = slot0 + 1 + b; q.j = 8 * (i - groups0 - b * per_slot);
      q.n = min(8, (q.slot == slot1 ? end1 : p.I) - q.j);
    }
    return q;
  };
  const int pieces = (p.H + p.piece - 1) / p.piece, per_group = 2 * pieces;      // stages of a group: its gate rows' pieces, its up rows'

  if (warp == WARPS) {
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      for (int i = 0; ok && i < groups; ++i) {
        const Group q = group_at(i);
        for (int h = 0; ok && h < 2; ++h) {
          const int64_t row = (int64_t)(2 * rt.slot_expert[q.slot] + h) * p.I + q.j;
          for (int k = 0; k < p.H; k += p.piece) {
            ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_UP_EMPTY);
            if (!ok) break;
            const int len = min(p.piece, p.H - k);
            const uint32_t dst = ring + s * p.stage_bytes, bar = full + 8 * s;
            const int8_t* src = p.w13 + row * p.H + k;
            if (pieces == 1) {                             // whole rows: they follow one another
              mbar_expect_tx(bar, q.n * len);
              bulk_load(dst, src, q.n * len, bar);
            } else if (q.n == 8) {                         // a box, zeros beyond H
              mbar_expect_tx(bar, 8 * p.piece);
              tma_load_2d(dst, &tm_w, k / 8, (int)row, bar);
            } else {
              mbar_expect_tx(bar, q.n * len);
              for (int r = 0; r < q.n; ++r) bulk_load(dst + r * p.piece, src + (int64_t)r * p.H, len, bar);
            }
            ++issued;
            if (++s == p.stages) { s = 0; par ^= 1u; }
          }
        }
      }
      if (!ok) drain_issued(full, p.stages, issued);
    }
    return;
  }

  for (int s = slot0 + threadIdx.x; s <= slot1; s += WORKERS) arrivals_open(p.counts + s, p.tag, p.epoch);
  i8_quantize_tokens<BF16, WORKERS>(p.x, p.H, p.T, p.H, codes, p.pitch, tok, meet);
  const uint32_t codes_at = smem_u32(codes) + 16 * t;
  int item = warp;                                         // stages are dealt out to the warps in turn
  bool ok = true;
  for (int pass = 0, b = 0; pass < groups; pass += PASS, b ^= 1) {
    const int here = min(PASS, groups - pass);
    int* mine = sums + b * PASS * p.T * 16;
    // the scales of the columns that this warp will finish, fetched under the stream: groups warp and warp + 8 of the pass
    float sg[PASS / WARPS], su[PASS / WARPS];
#pragma unroll
    for (int i = 0; i < PASS / WARPS; ++i) {
      sg[i] = su[i] = 0.f;
      if (warp + i * WARPS < here) {
        const Group q = group_at(pass + warp + i * WARPS);
        const int64_t at = (int64_t)rt.slot_expert[q.slot] * 2 * p.I + q.j + (lane & 7);
        if ((lane & 7) < q.n) { sg[i] = load_scalar(p.s13, at, p.s13_dt); su[i] = load_scalar(p.s13, at + p.I, p.s13_dt); }
      }
    }
    for (; item < (pass + here) * per_group; item += WARPS) {
      const int gi = item / per_group, sub = item - gi * per_group, h = sub >= pieces, k0 = (sub - h * pieces) * p.piece;
      const int slot = group_at(gi).slot, first = rt.slot_first[slot], rows = rt.slot_first[slot + 1] - first;
      const uint32_t xa = codes_at + (g < rows ? rt.list[first + g] / p.k : 0) * p.pitch + k0;
      const uint32_t xb = codes_at + (g + 8 < rows ? rt.list[first + g + 8] / p.k : 0) * p.pitch + k0;
      const int s = item % p.stages;
      ok = ok && mbar_wait_warp(full + 8 * s, (item / p.stages) & 1, abort_flag, p.status, ST_UP_FULL);
      if (!ok) continue;
      int acc[4] = {0, 0, 0, 0};
      multiply(acc, ring + s * p.stage_bytes + g * p.piece + 16 * t, xa, xb, g < rows, g + 8 < rows, min(p.piece, p.H - k0));
      mbar_arrive_read(empty + 8 * s);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = g + (c & 2) * 4;
        if (row < rows) add_shared(mine + ((gi - pass) * p.T + row) * 16 + 8 * h + 2 * t + (c & 1), acc[c]);
      }
    }
    __syncwarp();
    meet();                                                // the pass's sums are complete, and those before it have been read
#pragma unroll
    for (int i = 0; i < PASS / WARPS; ++i) {
      if (warp + i * WARPS >= here) break;
      const Group q = group_at(pass + warp + i * WARPS);
      const int first = rt.slot_first[q.slot], rows = rt.slot_first[q.slot + 1] - first, col = lane & 7;
      for (int row = lane >> 3; row < rows; row += 4) {
        const int pair = rt.list[first + row];
        int* v = mine + ((warp + i * WARPS) * p.T + row) * 16 + col;
        const float xs = tok.scale[pair / p.k];
        if (col < q.n) p.h[(int64_t)pair * p.I + q.j + col] = silu_mul_f(i8_scaled(v[0], xs, sg[i]), i8_scaled(v[8], xs, su[i]));
        v[0] = v[8] = 0;
      }
    }
  }
  // deliver: whoever is the last of a slot makes its rows' codes
  __threadfence();
  __syncwarp();
  meet();
  for (int i = slot0; i <= slot1; ++i) {
    if (threadIdx.x == 0) {
      const int others = owner((int64_t)(i + 1) * p.I - 1, n, G) - owner((int64_t)i * p.I, n, G);
      last = arrivals_last(p.counts + i, others);
      __threadfence();
    }
    __syncwarp();
    meet();
    const bool mine = last != 0;
    meet();
    if (mine) quantize_rows(p, rt, i, red);
  }
}

template <bool BF16, int PER>
__global__ void __launch_bounds__(DOWN_THREADS, 1) moe_i8_down_kernel(const __grid_constant__ CUtensorMap tm_w, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Route rt;
  __shared__ float code_scale[MAX_PAIRS];
  // [ring: weight rows and T rows of codes x piece] [sums: pairs x row_cap] [scales: the same] [barriers]
  const int pairs = p.T * p.k;
  const uint32_t ring = smem_u32(smem);
  int* sums = reinterpret_cast<int*>(smem + p.stages * p.stage_bytes);
  float* scales = reinterpret_cast<float*>(sums + pairs * p.row_cap);
  const uint32_t full = smem_u32(scales + pairs * p.row_cap), empty = full + 8 * MAX_STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(scales + pairs * p.row_cap) + 16 * MAX_STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int r0 = (int)((int64_t)blockIdx.x * p.H / gridDim.x), rows = (int)((int64_t)(blockIdx.x + 1) * p.H / gridDim.x) - r0;

  grid_dep_release();
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) { mbar_init(full + 8 * i, 2); mbar_init(empty + 8 * i, 1); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  for (int i = threadIdx.x; i < pairs * p.row_cap; i += DOWN_THREADS) sums[i] = 0;
  route<PER>(p, rt);
  const int sr = p.stage_rows, nrg = (rows + sr - 1) / sr, pieces = (p.I + p.piece - 1) / p.piece;

  if (warp == WARPS) {
    // ---- weights: before the up kernel has finished ----
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      for (int slot = 0; ok && slot < rt.slots; ++slot) {
        const int64_t row0 = (int64_t)rt.slot_expert[slot] * p.H + r0;
        for (int rg = 0; ok && rg < nrg; ++rg) {
          const int nr = min(sr, rows - sr * rg);
          const int8_t* src = p.w2 + (row0 + sr * rg) * p.I;
          for (int k = 0; k < p.I; k += p.piece) {
            ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_DOWN_EMPTY);
            if (!ok) break;
            const int len = min(p.piece, p.I - k);
            const uint32_t dst = ring + s * p.stage_bytes, bar = full + 8 * s;
            if (pieces == 1) {
              mbar_expect_tx(bar, nr * len);
              bulk_load(dst, src, nr * len, bar);
            } else if (nr == 8) {
              mbar_expect_tx(bar, 8 * p.piece);
              tma_load_2d(dst, &tm_w, k / 8, (int)row0 + sr * rg, bar);
            } else {
              mbar_expect_tx(bar, nr * len);
              for (int r = 0; r < nr; ++r) bulk_load(dst + r * p.piece, src + (int64_t)r * p.I + k, len, bar);
            }
            ++issued;
            if (++s == p.stages) { s = 0; par ^= 1u; }
          }
        }
      }
      if (!ok) drain_issued(full, p.stages, issued);
    }
    return;
  }
  if (warp == WARPS + 1) {
    // ---- the pairs' codes of the same k, which the up kernel makes ----
    if (elect_one()) {
      grid_dep_wait();
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      for (int slot = 0; ok && slot < rt.slots; ++slot) {
        const int first = rt.slot_first[slot], nx = rt.slot_first[slot + 1] - first;
        for (int rg = 0; ok && rg < nrg; ++rg) {
          for (int k = 0; k < p.I; k += p.piece) {
            ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_DOWN_XEMPTY);
            if (!ok) break;
            const int len = min(p.piece, p.I - k);
            const uint32_t dst = ring + s * p.stage_bytes + sr * p.piece, bar = full + 8 * s;
            mbar_expect_tx(bar, nx * len);
            for (int r = 0; r < nx; ++r) bulk_load(dst + r * p.piece, p.hq + (int64_t)rt.list[first + r] * p.I + k, len, bar);
            ++issued;
            if (++s == p.stages) { s = 0; par ^= 1u; }
          }
        }
      }
      if (!ok) drain_issued(full, p.stages, issued);
    }
    return;
  }

  for (int i = threadIdx.x; i < pairs * rows; i += WORKERS) {
    const int pair = i / rows, r = i - pair * rows, e = rt.expert[pair];
    scales[pair * p.row_cap + r] = e >= 0 ? load_scalar(p.s2, (int64_t)e * p.H + r0 + r, p.s2_dt) : 0.f;
  }
  bool ok = true;
  const int per_slot = nrg * pieces, items = rt.slots * per_slot;
  for (int item = warp; ok && item < items; item += WARPS) {
    const int slot = item / per_slot, sub = item - slot * per_slot, rg = sub / pieces, k0 = (sub - rg * pieces) * p.piece;
    const int first = rt.slot_first[slot], nx = rt.slot_first[slot + 1] - first, s = item % p.stages;
    ok = mbar_wait_warp(full + 8 * s, (item / p.stages) & 1, abort_flag, p.status, ST_DOWN_FULL);
    if (!ok) break;
    const uint32_t w = ring + s * p.stage_bytes + g * p.piece + 16 * t, x = w + sr * p.piece;
    const int len = min(p.piece, p.I - k0), left = rows - sr * rg;
    int acc[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    multiply(acc[0], w, x, x + 8 * p.piece, g < nx, g + 8 < nx, len);
    if (sr > 8 && left > 8) multiply(acc[1], w + 8 * p.piece, x, x + 8 * p.piece, g < nx, g + 8 < nx, len);
    mbar_arrive_read(empty + 8 * s);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int row = g + (c & 2) * 4, r = sr * rg + (c & 4) * 2 + 2 * t + (c & 1);
      if (row < nx && (c & 4) * 2 + 2 * t + (c & 1) < sr && r < rows) add_shared(sums + rt.list[first + row] * p.row_cap + r, acc[c >> 2][c & 3]);
    }
  }
  grid_dep_wait();                                         // over by now; the scales of the codes are the up kernel's
  for (int i = threadIdx.x; i < pairs; i += WORKERS) code_scale[i] = rt.expert[i] >= 0 ? ld_f32(p.hs + i) : 0.f;
  __syncwarp();
  meet();
  for (int i = threadIdx.x; i < p.T * rows; i += WORKERS) {
    const int tok = i / rows, r = i - tok * rows;
    float v = 0.f;
    for (int q = 0; q < p.k; ++q) {
      const int pair = tok * p.k + q;
      if (rt.expert[pair] >= 0) v = fmaf(rt.weight[pair], i8_scaled(sums[pair * p.row_cap + r], code_scale[pair], scales[pair * p.row_cap + r]), v);
    }
    p.out[(int64_t)tok * p.H + r0 + r] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
static int sm_count() {
  static thread_local int sms[16] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16) return 148;
  if (!sms[dev]) {
    cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
    if (sms[dev] <= 0) sms[dev] = 148;
  }
  return sms[dev];
}
static size_t align256(size_t v) { return (v + 255) / 256 * 256; }
static int down_grid(int64_t H) { return (int)(sm_count() < H ? sm_count() : H); }
static int up_fixed(int T, int pitch) { return T * pitch + 2 * PASS * T * 16 * 4 + BAR_BYTES; }
static int down_fixed(int pairs, int cap) { return 2 * pairs * cap * 4 + BAR_BYTES; }

static int room(int fixed) { return SMEM_MAX - (int)sizeof(Route) - 4 * MAX_PAIRS - 512 - fixed; }

static int launch(void (*kern)(const CUtensorMap, const Params), const char* name, int grid, int threads, int fixed, const int8_t* w, int64_t rows, int K, Params& p,
                  int* configured, cudaStream_t st) {
  p.stages = room(fixed) / p.stage_bytes / WARPS * WARPS;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  const int smem = p.stages * p.stage_bytes + fixed;
  CUtensorMap tm{};
  if (p.piece < K) {
    const int rc = make_tmap_2d(&tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 8, w, rows, K / 8, (uint64_t)K, 8, p.piece / 8, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc) return rc;
  }
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || configured[dev] < smem) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return B2Q_ERR_CUDA;
    if (dev < 16) configured[dev] = smem;
  }
  launch_overlapped(kern, dim3(grid), dim3(threads), smem, st, tls().overlap_mode > 0, tm, p);
  note_launch(name);
  return launch_status();
}

// k of a stage: the whole row where a stage of that for every warp fits, else what fits (a TMA box has 2048 bytes of a row at most)
static int piece_of(int K, int bytes_per_k, int fixed) {
  const int fits = room(fixed) / WARPS / bytes_per_k;
  if (K <= fits && K <= PIECE) return K;
  const int v = fits < PIECE ? fits : PIECE;
  return v / 64 * 64;
}

template <bool BF16, int PER> static int run(Params& p, cudaStream_t st) {
  static thread_local int configured[2][16] = {{0}};
  p.pitch = i8_code_pitch(p.H);
  int fixed = up_fixed(p.T, p.pitch);
  p.stage_rows = 8;
  p.piece = piece_of(p.H, 8, fixed);
  p.stage_bytes = 8 * p.piece;
  int rc = launch(moe_i8_up_kernel<BF16, PER>, "moe_i8_up", sm_count(), UP_THREADS, fixed, p.w13, (int64_t)p.E * 2 * p.I, p.H, p, configured[0], st);
  if (rc) return rc;
  const int grid = down_grid(p.H);
  p.row_cap = (p.H + grid - 1) / grid;
  fixed = down_fixed(p.T * p.k, p.row_cap);
  // sixteen rows that are one run of memory, if there are that many and they fit; else eight
  p.stage_rows = p.row_cap > 8 && piece_of(p.I, 16 + p.T, fixed) == p.I ? 16 : 8;
  p.piece = piece_of(p.I, p.stage_rows + p.T, fixed);
  p.stage_bytes = (p.stage_rows + p.T) * p.piece;
  return launch(moe_i8_down_kernel<BF16, PER>, "moe_i8_down", grid, DOWN_THREADS, fixed, p.w2, (int64_t)p.E * p.H, p.I, p, configured[1], st);
}
}  // namespace mi8

bool moe_i8_few_supported(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I) {
  using namespace mi8;
  if (T > MAX_TOK || E > MAX_E || k > MAX_K || H > INT32_MAX / 64 || I > INT32_MAX / 64) return false;
  const int64_t cap = (H + down_grid(H) - 1) / down_grid(H);
  return T * i8_code_pitch((int)H) <= CODES_MAX && T * k * cap * 4 <= TABLE_MAX;
}

size_t moe_i8_few_bytes(int64_t T, int64_t k, int64_t I) {
  const size_t pairs = (size_t)T * k;
  return mi8::align256(pairs * I * 4) + mi8::align256(pairs * I) + mi8::align256(pairs * 4) + mi8::align256(pairs * 8);
}

int moe_i8_few(const I8FewArgs& a, cudaStream_t st) {
  using namespace mi8;
  Params p{};
  p.x = reinterpret_cast<const uint16_t*>(a.x); p.logits = a.logits; p.ldt = a.logits_dtype;
  p.w13 = a.w13; p.s13 = a.s13; p.s13_dt = a.s13_dtype; p.w2 = a.w2; p.s2 = a.s2; p.s2_dt = a.s2_dtype;
  p.out = reinterpret_cast<uint16_t*>(a.out);
  p.T = a.T; p.E = a.E; p.k = a.k; p.H = a.H; p.I = a.I; p.renorm = a.renorm;
  const size_t pairs = (size_t)a.T * a.k;
  uint8_t* at = reinterpret_cast<uint8_t*>(a.scratch);
  p.h = reinterpret_cast<float*>(at); at += align256(pairs * a.I * 4);
  p.hq = reinterpret_cast<int8_t*>(at); at += align256(pairs * a.I);
  p.hs = reinterpret_cast<float*>(at); at += align256(pairs * 4);
  p.counts = reinterpret_cast<Arrivals*>(at);
  p.tag = arrivals_tag();
  p.epoch = arrivals_epoch();
  p.status = umma_status_ptr();
  if (!p.epoch || !p.status) return B2Q_ERR_CUDA;
  if (a.bf16) return a.E <= 128 ? run<true, 4>(p, st) : (a.E <= 256 ? run<true, 8>(p, st) : run<true, 32>(p, st));
  return a.E <= 128 ? run<false, 4>(p, st) : (a.E <= 256 ? run<false, 8>(p, st) : run<false, 32>(p, st));
}

}  // namespace b2q
