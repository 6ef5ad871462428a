// A whole int8 expert layer of a few tokens (up to sixteen; moe_i8_few_preferred has the line) in one kernel:
//   ids, w = top-k of the logits;  h = silu(x W_gate) * (x W_up) per (token, expert) pair;  out = sum of w * (h W_down),
// where x and h meet the int8 weights as int8 codes with one scale per row.
//
// HBM-bound: the chosen experts' matrices, once.  One CTA per SM; one thread fetches weights, eight or up to sixteen rows at a time, into a
// ring that fills the SM's shared memory, first of the up and gate matrices, then, without a pause, of the down matrices: rows that are
// taken whole are one contiguous run and one untiled bulk copy of exactly the rows that are wanted; pieces of longer rows are TMA boxes.
// Eight warps feed them to mma.sync m16n8k32 (the up to sixteen pairs of an expert are the MMA's rows, with k permuted alike on both sides so
// that a lane reads sixteen bytes of a row at a time).  A stage is one warp's, whose sums are added up in shared memory, in integers, so
// that no division of the work changes a bit.
//
// Up.  Every CTA routes all tokens and makes all their codes by itself, which costs less than a launch.  The columns j of all chosen experts,
// one expert behind the other, are dealt out evenly to the column; eight columns are eight gate rows and eight up rows.  h is written in
// fp32.  An expert's rows of h become codes as soon as its last CTA has delivered (arrivals.cuh): that one CTA makes them and
// raises the expert's flag.
// Down.  A CTA owns output columns and runs through all chosen experts, so no sum crosses CTAs: the pairs' products add up in the order of
// the slots.  The codes of h that go with a stage of weights are fetched by the warp that owns the stage, as soon as it has done with it,
// behind the expert's flag (one thread for all stages took 580 ns per stage).
//
// CTAs wait for one another's flags, so the launch is cooperative.  One token, 128 experts of 2048 x 768, top-8: 19.3 us, 5.8 of them the weights'; the
// rest is a chain: launch, routing and codes, the ring's first weights, the codes of h behind the last column, the down part behind those.  As two
// kernels, each with its own routing and an empty ring to begin with, 23.4.
//
// Every wait is bounded; a warp that gives up still goes to the barriers where the others expect it.
#include "arrivals.cuh"
#include "i8.cuh"
#include "i8_route.cuh"
#include "moe_i8_sizes.h"
#include "sm100.cuh"
#include "umma_gemm.cuh"

namespace b2q {

using namespace sm100;

namespace mi8 {
enum { ST_EMPTY = 901, ST_UP_FULL = 902, ST_DOWN_FULL = 903, ST_FLAG = 904 };
constexpr int THREADS = 512, W_WARP = 15;                  // the warp that fetches weights, beside those that multiply; all sixteen route
constexpr int HELPERS = 32 * W_WARP;                       // threads that make the tokens' codes, fill tables and store
static_assert(MAX_TOK == I8_STREAM_MAX_TOK, "");
static_assert(I8_FEW_LOAD + MAX_TOK * 192 <= 68 * 1024, "the tokens' codes leave the ring its shared memory");

struct Params {
  const uint16_t* x; const void* logits; int ldt;
  const int8_t* w13; const void* s13; int s13_dt;
  const int8_t* w2; const void* s2; int s2_dt;
  uint16_t* out;
  int T, E, k, H, I, renorm;
  float* h; int8_t* hq;                                    // [pairs, I]; [pairs, I + 16]: codes, then their scale
  Arrivals *counts, *flags, *left;                         // of slots; of slots; CTAs that have seen all flags
  Arrivals tag; const Arrivals* epoch;
  int pitch, row_cap, front;                               // front: bytes of the codes, or of the tables that take their place
  // The ring.  Stage s is always warp s % WARPS's (a parity wait cannot tell the phase it waits for from the one two before, so nobody may
  // come to a stage that another has not finished).
  int stages, stage_bytes;
  int up_piece, down_piece, down_rows;                     // k of a stage; weight rows of a down stage
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
  int16_t chunk_slot[MAX_PAIRS], chunk_first[MAX_PAIRS];   // up to XR pairs of a slot each; where in list
  int slots, chunks;
  __device__ __forceinline__ int chunk_pairs(int c) const { return min(XR, slot_first[chunk_slot[c] + 1] - chunk_first[c]); }
};
static_assert(sizeof(Route) + sizeof(I8Tokens) + 4 * (WORKERS + MAX_PAIRS) <= STATIC_BYTES, "");

template <int PER> __device__ __forceinline__ void route_token(const Params& p, int tok, const float (&v)[PER], Route& r) {
  int id;
  float weight;
  i8r::top_k<PER>(v, p.E, p.k, p.renorm != 0, id, weight);
  if ((threadIdx.x & 31) < p.k) {
    const int pair = tok * p.k + (threadIdx.x & 31);
    r.expert[pair] = (int16_t)id;
    r.weight[pair] = weight;
    if (id >= 0) {
      atomicMin(&r.first[id], pair);
      r.place[pair] = (int16_t)atomicAdd(&r.count[id], 1);
    }
  }
}

// The whole CTA.  Which place a pair gets among its expert's is a matter of chance and changes no result.  between(0) runs behind the barrier
// that has all tokens' choices, in every warp but the first, which finds the slots; between(1) behind the one that has the slots.
// r.first is p.T * p.k and r.count zero before, for everybody.
template <int PER, class Between> __device__ __forceinline__ void route(const Params& p, Route& r, const float (&logits)[PER], Between between) {
  static_assert(THREADS / 32 >= MAX_TOK, "a warp per token");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pairs = p.T * p.k;
  if (warp < p.T) route_token<PER>(p, warp, logits, r);
  __syncthreads();
  if (warp == 0) {
    int slots = 0, before = 0;
    for (int b = 0; b < pairs; b += 32) {
      const int e = b + lane < pairs ? r.expert[b + lane] : -1;
      const bool names = e >= 0 && r.first[e] == b + lane;
      const unsigned some = __ballot_sync(0xffffffffu, names);
      const int c = names ? r.count[e] : 0, n = (c + XR - 1) / XR;
      int upto = c | n << 16;                              // pairs and chunks up to here
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (names) {
        const int s = slots + __popc(some & ((1u << lane) - 1u)), first = (before + upto & 0xFFFF) - c;
        int chunk = (before + upto >> 16) - n;
        r.slot_expert[s] = (int16_t)e;
        r.slot_first[s] = (int16_t)first;
        for (int i = 0; i < c; i += XR, ++chunk) { r.chunk_slot[chunk] = (int16_t)s; r.chunk_first[chunk] = (int16_t)(first + i); }
        r.first[e] = s;                                    // a slot is no larger than the pair that named it: nobody looks at it as one again
      }
      slots += __popc(some);
      before += __shfl_sync(0xffffffffu, upto, 31);
      __syncwarp();
    }
    if (lane == 0) { r.slots = slots; r.slot_first[slots] = (int16_t)(before & 0xFFFF); r.chunks = before >> 16; }
    __syncwarp();
  }
  between(0);
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += THREADS)
    if (r.expert[i] >= 0) r.list[r.slot_first[r.first[r.expert[i]]] + r.place[i]] = (int16_t)i;
  between(1);
  __syncthreads();
}

// n things dealt out to G CTAs in turn: the first n % G have one more.
struct Share {
  int each, more;
  __device__ __forceinline__ Share(int n, int G) : each(n / G), more(n - n / G * G) {}
  __device__ __forceinline__ int begin(int b) const { return b * each + min(b, more); }
  __device__ __forceinline__ int owner(int c) const {      // each > 0
    const int big = more * (each + 1);
    return c < big ? c / (each + 1) : more + (c - big) / each;
  }
};

__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory"); }      // the eight warps

// Codes of one row of h, by one warp.  Up to 1024 values stay in registers between the maximum and the codes.
__device__ __forceinline__ void quantize_row(const Params& p, int pair) {
  constexpr int V = 8;
  const int lane = threadIdx.x & 31, n4 = p.I >> 2;
  const float4* h = reinterpret_cast<const float4*>(p.h + (int64_t)pair * p.I);
  float4 v[V];
  auto fetch = [&](int base) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = base + j * 32 + lane;
      v[j] = c < n4 ? __ldcg(h + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  uint32_t mx = 0;
  for (int base = 0; base < n4; base += V * 32) {
    fetch(base);
#pragma unroll
    for (int j = 0; j < V; ++j)
      mx = max(max(mx, __float_as_uint(v[j].x) & 0x7FFFFFFFu), max(__float_as_uint(v[j].y) & 0x7FFFFFFFu, max(__float_as_uint(v[j].z) & 0x7FFFFFFFu, __float_as_uint(v[j].w) & 0x7FFFFFFFu)));
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  const bool finite = mx < 0x7F800000u;
  const float a = fmaxf(__uint_as_float(mx), I8_MIN_AMAX), s = 127.f / a;
  uint32_t* q = reinterpret_cast<uint32_t*>(p.hq + (int64_t)pair * (p.I + 16));
  if (lane == 0) q[n4] = __float_as_uint(finite ? a / 127.f : __uint_as_float(0x7FC00000u));
  for (int base = 0; base < n4; base += V * 32) {
    if (n4 > V * 32) fetch(base);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = base + j * 32 + lane;
      const float f[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
      if (c < n4) q[c] = finite ? i8_codes4_computed(f, s) : 0u;
    }
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

// Nine to sixteen weight rows, at u and, where second says that the lane has one there, at v, against up to eight rows of codes at x.
__device__ __forceinline__ void multiply16(int (&acc)[2][4], uint32_t u, uint32_t v, uint32_t x, bool has, bool second, int len) {
  const int t16 = 16 * (threadIdx.x & 3);
  int more[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  auto step = [&](int k, bool in) {
    uint4 a = make_uint4(0, 0, 0, 0), b = a, c = a;
    if (in) b = lds(u + k);
    if (in && second) c = lds(v + k);                      // a stage ends behind its own rows
    if (in && has) a = lds(x + k);
    mma_s8(acc[0], a.x, 0u, a.y, 0u, b.x, b.y);
    mma_s8(acc[1], a.x, 0u, a.y, 0u, c.x, c.y);
    mma_s8(more[0], a.z, 0u, a.w, 0u, b.z, b.w);
    mma_s8(more[1], a.z, 0u, a.w, 0u, c.z, c.w);
  };
  const int whole = len & ~63;
#pragma unroll 4
  for (int k = 0; k < whole; k += 64) step(k, true);
  if (whole < len) step(whole, whole + t16 < len);
#pragma unroll
  for (int c = 0; c < 4; ++c) { acc[0][c] += more[0][c]; acc[1][c] += more[1][c]; }
}

// The whole warp: how many of the slots from `from` on, up to 32, have their flags raised without a gap.  At least one, or 0 after two seconds.
__device__ __forceinline__ int wait_flags(const Arrivals* flags, int from, int slots, Arrivals mark, volatile int* abort_flag, int* status) {
  const int slot = from + (threadIdx.x & 31);
  const long long t0 = clock64();
  for (;;) {
    Arrivals v = 0;
    if (slot < slots) asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(flags + slot) : "memory");
    const unsigned down = ~__ballot_sync(0xffffffffu, slot < slots && v == mark);
    if (!(down & 1u)) {
      __syncwarp();                                        // the lane that copies is behind what the others have acquired
      asm volatile("fence.proxy.async;" ::: "memory");     // what the flags stand for was written by ordinary stores and is read by bulk copies
      return down ? __ffs(down) - 1 : 32;
    }
    if (__any_sync(0xffffffffu, *abort_flag || clock64() - t0 > WAIT_LIMIT_TICKS)) break;
  }
  if ((threadIdx.x & 31) == 0 && !*abort_flag) {
    *abort_flag = 1;
    atomicCAS(status, 0, (int)ST_FLAG);
  }
  __syncwarp();
  return 0;
}

template <bool BF16, int PER>
__global__ void __launch_bounds__(THREADS, 1) moe_i8_kernel(const __grid_constant__ CUtensorMap tm_up, const __grid_constant__ CUtensorMap tm_down, const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Route rt;
  __shared__ I8Tokens tok;
  __shared__ int done[WORKERS];                            // slots of this CTA that it is the last to deliver
  __shared__ float code_scale[MAX_PAIRS];
  // [ring] [codes: T x pitch; later sums: pairs x row_cap, scales: the same] [sums of two passes: 2 x PASS x T x 16] [barriers]
  const int pairs = p.T * p.k;
  const uint32_t ring = smem_u32(smem);
  uint8_t* codes = smem + p.stages * p.stage_bytes;
  int* down_sums = reinterpret_cast<int*>(codes);
  float* down_scales = reinterpret_cast<float*>(down_sums + pairs * p.row_cap);
  int* sums = reinterpret_cast<int*>(codes + p.front);
  const uint32_t full = smem_u32(sums + 2 * PASS * p.T * 16), empty = full + 8 * MAX_STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(sums + 2 * PASS * p.T * 16) + 16 * MAX_STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  if (threadIdx.x == 0) {
    // full: the weights and, of a down stage, the codes
    for (int i = 0; i < p.stages; ++i) { mbar_init(full + 8 * i, 2); mbar_init(empty + 8 * i, 1); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < MAX_TOK) tok.max[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < 2 * PASS * p.T * 16; i += THREADS) sums[i] = 0;
  for (int i = threadIdx.x; i < p.E; i += THREADS) { rt.first[i] = pairs; rt.count[i] = 0; }
  float logits[PER];
  if (warp < p.T) i8r::load_logits<PER>(p.logits, p.ldt, p.E, warp, logits);
  // One or two tokens' codes are made alongside the routing; of more, only those that this CTA's columns need, behind it.
  const bool soon = p.T <= 2;
  I8TokenCodes<BF16, HELPERS, 6> tc(p.x, p.H, p.T, p.H);
  if (soon && warp < W_WARP) tc.fetch();
  __syncthreads();
  route<PER>(p, rt, logits, [&](int step) {
    if (soon && warp < W_WARP) { if (step == 0) tc.maximum(tok); else tc.rows(tok); }
  });
  grid_dep_release();

  // ---- this CTA's share of the up part: columns [c0, c1) of all slots' columns, as groups of eight: those of the first slot's part, then of
  // whole slots; the last slot's part may end early ----
  const int n = rt.slots * p.I;                            // at most 512 * 131071
  const int G = min((int)gridDim.x, n);                    // CTAs that have a column
  const bool any = (int)blockIdx.x < G;
  const Share share(n, max(G, 1));
  const int c0 = any ? share.begin(blockIdx.x) : 0, c1 = any ? share.begin(blockIdx.x + 1) : 0;
  const int slot0 = c0 / p.I, slot1 = any ? (c1 - 1) / p.I : -1;
  const int j0 = c0 - slot0 * p.I, per_slot = (p.I + 7) / 8;
  const int len0 = min(p.I - j0, c1 - c0), groups0 = (len0 + 7) / 8;
  const int end1 = c1 - slot1 * p.I;                       // columns of the last slot end here
  const int groups = !any ? 0 : (slot0 == slot1 ? groups0 : groups0 + (slot1 - slot0 - 1) * per_slot + (end1 + 7) / 8);
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
  const int up_pieces = (p.H + p.up_piece - 1) / p.up_piece, per_group = 2 * up_pieces;      // stages of a group: its gate rows' pieces, its up rows'
  const int up_items = groups * per_group;
  // ---- and of the down part: rows [r0, r0 + rows) of every slot's matrix ----
  const Share row_share(p.H, gridDim.x);
  const int r0 = row_share.begin(blockIdx.x), rows = row_share.begin(blockIdx.x + 1) - r0;
  const int sr = p.down_rows, nrg = (rows + sr - 1) / sr, down_pieces = (p.I + p.down_piece - 1) / p.down_piece;
  const int per_chunk = nrg * down_pieces, items = up_items + rt.chunks * per_chunk;
  const Arrivals mark = p.tag ^ *reinterpret_cast<const volatile Arrivals*>(p.epoch) << ARRIVALS_BITS;

  if (warp == W_WARP) {
    // ---------------- weights ----------------
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      // n rows of K bytes, len of them from k on: whole rows follow one another; eight pieces are a box, zeros beyond K
      auto put = [&](const int8_t* base, const CUtensorMap* map, int64_t row, int n, int K, int k, int piece, int pieces) {
        const int len = min(piece, K - k);
        const uint32_t dst = ring + s * p.stage_bytes, bar = full + 8 * s;
        const int8_t* src = base + row * K + k;
        if (pieces == 1) {
          mbar_expect_tx(bar, n * len);
          bulk_load(dst, src, n * len, bar);
        } else if (n == 8) {
          mbar_expect_tx(bar, 8 * piece);
          tma_load_2d(dst, map, k / 8, (int)row, bar);
        } else {
          mbar_expect_tx(bar, n * len);
          for (int r = 0; r < n; ++r) bulk_load(dst + r * piece, src + (int64_t)r * K, len, bar);
        }
        ++issued;
      };
      for (int i = 0; ok && i < groups; ++i) {
        const Group q = group_at(i);
        for (int h = 0; ok && h < 2; ++h) {
          const int64_t row = (int64_t)(2 * rt.slot_expert[q.slot] + h) * p.I + q.j;
          for (int k = 0; k < p.H; k += p.up_piece) {
            ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_EMPTY);
            if (!ok) break;
            put(p.w13, &tm_up, row, q.n, p.H, k, p.up_piece, up_pieces);
            mbar_arrive(full + 8 * s);                     // no codes come with it
            if (++s == p.stages) { s = 0; par ^= 1u; }
          }
        }
      }
      for (int c = 0; ok && c < rt.chunks; ++c) {
        const int64_t row = (int64_t)rt.slot_expert[rt.chunk_slot[c]] * p.H + r0;
        for (int rg = 0; ok && rg < nrg; ++rg) {
          for (int k = 0; k < p.I; k += p.down_piece) {
            ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_EMPTY);
            if (!ok) break;
            put(p.w2, &tm_down, row + sr * rg, min(sr, rows - sr * rg), p.I, k, p.down_piece, down_pieces);
            if (++s == p.stages) { s = 0; par ^= 1u; }
          }
        }
      }
      if (!ok) drain_issued(full, p.stages, issued);
    }
    return;
  }
  if (!soon) {
    if (warp == 0) {
      uint32_t mask = 0;
      if (any)
        for (int i = rt.slot_first[slot0] + lane; i < rt.slot_first[slot1 + 1]; i += 32) mask |= 1u << (rt.list[i] / p.k);
      mask = __reduce_or_sync(0xffffffffu, mask);
      if (lane == 0) tok.count = __popc(mask);
      if (mask >> lane & 1) tok.list[__popc(mask & ((1u << lane) - 1u))] = (int16_t)lane;
      __syncwarp();
    }
    asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");
    tc.only(tok);
    tc.fetch();
    tc.maximum(tok);
    asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");
    tc.rows(tok);
    asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");
  }
  tc.codes(tok, codes, p.pitch);
  __syncwarp();
  asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");

  // ---------------- up: eight warps ----------------
  // a warp's items are those of its stages: stage, then the round of the ring
  int stage = warp, item = warp;
  uint32_t par = 0u;
  bool ok = true;
  if (warp >= p.stages || warp >= WARPS) item = items;     // none
  auto next = [&] {
    stage += WARPS; item += WARPS;
    if (stage >= p.stages) { item += p.stages - stage + warp; stage = warp; par ^= 1u; }
  };
  if (warp < WARPS) {
    if (threadIdx.x == 0) arrivals_open(p.left, p.tag, p.epoch);
    for (int s = slot0 + threadIdx.x; s <= slot1; s += WORKERS) arrivals_open(p.counts + s, p.tag, p.epoch);
    const uint32_t codes_at = smem_u32(codes) + 16 * t;
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
      for (; item < (pass + here) * per_group; next()) {
        const int gi = item / per_group, sub = item - gi * per_group, h = sub >= up_pieces, k0 = (sub - h * up_pieces) * p.up_piece;
        const int slot = group_at(gi).slot, first = rt.slot_first[slot], nrows = rt.slot_first[slot + 1] - first;
        const uint32_t xa = codes_at + (g < nrows ? rt.list[first + g] / p.k : 0) * p.pitch + k0;
        const uint32_t xb = codes_at + (g + 8 < nrows ? rt.list[first + g + 8] / p.k : 0) * p.pitch + k0;
        ok = ok && mbar_wait_warp(full + 8 * stage, par, abort_flag, p.status, ST_UP_FULL);
        if (!ok) continue;
        int acc[4] = {0, 0, 0, 0};
        multiply(acc, ring + stage * p.stage_bytes + g * p.up_piece + 16 * t, xa, xb, g < nrows, g + 8 < nrows, min(p.up_piece, p.H - k0));
        mbar_arrive_read(empty + 8 * stage);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = g + (c & 2) * 4;
          if (row < nrows) add_shared(mine + ((gi - pass) * p.T + row) * 16 + 8 * h + 2 * t + (c & 1), acc[c]);
        }
      }
      __syncwarp();
      meet();                                              // the pass's sums are complete, and those before it have been read
#pragma unroll
      for (int i = 0; i < PASS / WARPS; ++i) {
        if (warp + i * WARPS >= here) break;
        const Group q = group_at(pass + warp + i * WARPS);
        const int first = rt.slot_first[q.slot], nrows = rt.slot_first[q.slot + 1] - first, col = lane & 7;
        for (int row = lane >> 3; row < nrows; row += 4) {
          const int pair = rt.list[first + row];
          int* v = mine + ((warp + i * WARPS) * p.T + row) * 16 + col;
          const float xs = tok.scale[pair / p.k];
          if (col < q.n) p.h[(int64_t)pair * p.I + q.j + col] = silu_mul_f(i8_scaled(v[0], xs, sg[i]), i8_scaled(v[8], xs, su[i]));
          v[0] = v[8] = 0;
        }
      }
    }
    // deliver: whoever is the last of a slot makes its rows' codes, a warp each, and raises its flag
    __threadfence();
    __syncwarp();
    meet();
    for (int base = slot0; base <= slot1; base += WORKERS) {
      const int slot = base + threadIdx.x;
      int last = 0;
      if (slot <= slot1) {
        last = arrivals_last(p.counts + slot, share.owner((slot + 1) * p.I - 1) - share.owner(slot * p.I));
        __threadfence();
      }
      done[threadIdx.x] = last;
      __syncwarp();
      meet();
      int at = 0;
      for (int i = base; i <= min(slot1, base + WORKERS - 1); ++i) {
        if (!done[i - base]) continue;
        for (int r = rt.slot_first[i]; r < rt.slot_first[i + 1]; ++r, ++at)
          if ((at & (WARPS - 1)) == warp) quantize_row(p, rt.list[r]);
      }
      __threadfence();
      __syncwarp();
      meet();
      if (last && ok) asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(p.flags + slot), "l"(mark) : "memory");
      __syncwarp();
    }
  }
  __syncwarp();
  asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");      // the tokens' codes are done with: the tables take their place

  // ---------------- down ----------------
  for (int i = threadIdx.x; i < pairs * p.row_cap; i += HELPERS) {
    const int pair = i / p.row_cap, r = i - pair * p.row_cap, e = rt.expert[pair];
    down_sums[i] = 0;
    down_scales[i] = e >= 0 && r < rows ? load_scalar(p.s2, (int64_t)e * p.H + r0 + r, p.s2_dt) : 0.f;
  }
  __syncwarp();
  asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");
  int raised = 0;                                          // slots whose flags this warp has seen
  // the codes of an item of this warp's, to the stage that it goes through
  auto fetch = [&](int it, int at) {
    const int chunk = (it - up_items) / per_chunk, k0 = (it - up_items - chunk * per_chunk) % down_pieces * p.down_piece;
    while (ok && rt.chunk_slot[chunk] >= raised) {
      const int more = wait_flags(p.flags, raised, rt.slots, mark, abort_flag, p.status);
      ok = more > 0;
      raised += more;
    }
    if (!ok) return;
    const int first = rt.chunk_first[chunk], nx = rt.chunk_pairs(chunk);
    const int len = min(p.down_piece, p.I - k0) + (k0 + p.down_piece >= p.I ? 16 : 0);      // the scale comes with the last piece
    const uint32_t dst = ring + at * p.stage_bytes + sr * p.down_piece, bar = full + 8 * at;
    if (elect_one()) {
      mbar_expect_tx(bar, nx * len);
      for (int r = 0; r < nx; ++r) bulk_load(dst + r * (p.down_piece + 16), p.hq + (int64_t)rt.list[first + r] * (p.I + 16) + k0, len, bar);
    }
    __syncwarp();
  };
  // the first down items of this warp's stages; later ones when the stage comes free
  for (int s = warp; warp < WARPS && s < p.stages; s += WARPS) {
    const int it = up_items + (s - up_items % p.stages + p.stages) % p.stages;
    if (it < items) fetch(it, s);
  }
  for (; ok && item < items; next()) {
    const int chunk = (item - up_items) / per_chunk, sub = item - up_items - chunk * per_chunk, rg = sub / down_pieces, k0 = (sub - rg * down_pieces) * p.down_piece;
    const int first = rt.chunk_first[chunk], nx = rt.chunk_pairs(chunk);
    ok = mbar_wait_warp(full + 8 * stage, par, abort_flag, p.status, ST_DOWN_FULL);
    if (!ok) break;
    const uint32_t w = ring + stage * p.stage_bytes + g * p.down_piece + 16 * t, x = ring + stage * p.stage_bytes + sr * p.down_piece + g * (p.down_piece + 16) + 16 * t;
    const int len = min(p.down_piece, p.I - k0), left = rows - sr * rg;
    int acc[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (sr > 8 && left > 8) multiply16(acc, w, w + 8 * p.down_piece, x, g < nx, g + 8 < min(sr, left), len);
    else multiply(acc[0], w, x, 0, g < nx, false, len);
    if (k0 + len == p.I && rg == 0 && t == 0 && g < nx) {
      uint32_t v;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(x + len) : "memory");
      code_scale[rt.list[first + g]] = __uint_as_float(v);
    }
    mbar_arrive_read(empty + 8 * stage);
    if (item + p.stages < items) fetch(item + p.stages, stage);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int r = 8 * (c >> 1) + 2 * t + (c & 1);
      if (g < nx && r < sr && sr * rg + r < rows) add_shared(down_sums + rt.list[first + g] * p.row_cap + sr * rg + r, acc[c >> 1][c & 1]);
    }
  }
  if (!ok && lane == 0) drain_issued(full, p.stages, item + p.stages);      // the copies of this item, and of this warp's other stages
  __syncwarp();
  asm volatile("bar.sync 2, %0;" ::"n"(HELPERS) : "memory");
  // The last CTA that has seen all flags lowers them: a graph's replays have the same mark.  (What a CTA that gave up leaves raised, the
  // reset of the status words makes another launch's.)
  if (threadIdx.x == 32 * WARPS && !*abort_flag && arrivals_last(p.left, gridDim.x - 1))
    for (int i = 0; i < rt.slots; ++i) p.flags[i] = 0;
  for (int i = threadIdx.x; i < p.T * rows; i += HELPERS) {
    const int token = i / rows, r = i - token * rows;
    float v = 0.f;
    for (int q = 0; q < p.k; ++q) {
      const int pair = token * p.k + q;
      if (rt.expert[pair] >= 0) v = fmaf(rt.weight[pair], i8_scaled(down_sums[pair * p.row_cap + r], code_scale[pair], down_scales[pair * p.row_cap + r]), v);
    }
    p.out[(int64_t)token * p.H + r0 + r] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
static size_t align256(size_t v) { return (v + 255) / 256 * 256; }
static int grid_of(int64_t H) { return (int)(sm_count() < H ? sm_count() : H); }

template <bool BF16, int PER> static int run(Params& p, cudaStream_t st) {
  const Sizes s = sizes_of(p.T, p.k, p.H, p.I, i8_code_pitch(p.H), sm_count());
  const int grid = s.grid, smem = s.smem;
  p.pitch = s.pitch; p.row_cap = s.row_cap; p.front = s.front;
  p.up_piece = s.up_piece; p.down_piece = s.down_piece; p.down_rows = s.down_rows;
  p.stages = s.stages; p.stage_bytes = s.stage_bytes;
  CUtensorMap tu{}, td{};
  int rc = B2Q_OK;
  if (p.up_piece < p.H)
    rc = make_tmap_2d(&tu, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 8, p.w13, (uint64_t)p.E * 2 * p.I, p.H / 8, p.H, 8, p.up_piece / 8, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!rc && p.down_piece < p.I)
    rc = make_tmap_2d(&td, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 8, p.w2, (uint64_t)p.E * p.H, p.I / 8, p.I, 8, p.down_piece / 8, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc) return rc;
  auto kern = moe_i8_kernel<BF16, PER>;
  static thread_local int configured[16] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || configured[dev] < smem) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return B2Q_ERR_CUDA;
    if (dev < 16) configured[dev] = smem;
  }
  // No early start: CTAs that wait for one another are launched together or not at all.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, tu, td, p);               // launch_status() reports
  note_launch("moe_i8");
  return launch_status();
}
}  // namespace mi8

// Every CTA makes all tokens' codes and fetches all pairs' codes of h, which grows with the tokens while the weights' bytes do not; the grouped GEMMs
// pay six launches instead, four of them under the weights that a GEMM fetches in advance.  Over 18 layers of 3 to 1395 MB with 1 to 16 tokens the line
// below took 1.003 times as long as the better of the two (always one kernel 1.18, never 1.013).  One kernel / grouped, us: 128 experts of 2048 x 768, top-8,
// 1 / 2 / 4 / 16 tokens 19.3 / 21.7, 29.5 / 29.9, 43.2 / 40.8, 97.9 / 83.3; 16 of 4096 x 1024, top-1, 1 / 8: 16.0 / 19.6, 30.8 / 30.5; 8 of 4096 x 14336, top-2, 1 / 16:
// 87.6 / 76.2, 416 / 229; 8 of 1024 x 512, top-2, 1 / 16: 15.6 / 16.3, 20.8 / 18.3; 8 of 2048 x 2048, top-8, 16: 91.3 / 36.6.  The second condition is room: a CTA's
// sums of all pairs, and as many scales, take the place of the tokens' codes.
bool moe_i8_few_preferred(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I) {
  using namespace mi8;
  if (T > MAX_TOK || E > MAX_E || k > MAX_K || H > INT32_MAX / 64 || I > INT32_MAX / 64) return false;
  const int64_t cap = (H + grid_of(H) - 1) / grid_of(H);
  return T * (4 * k * I + H) <= I8_FEW_LOAD && T * k * cap * 4 <= TABLE_MAX;
}

size_t moe_i8_few_bytes(int64_t T, int64_t k, int64_t I) {
  const size_t pairs = (size_t)T * k;
  return mi8::align256(pairs * I * 4) + mi8::align256(pairs * (I + 16)) + 2 * mi8::align256(pairs * 8) + 256;
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
  p.hq = reinterpret_cast<int8_t*>(at); at += align256(pairs * (a.I + 16));
  p.counts = reinterpret_cast<Arrivals*>(at); at += align256(pairs * 8);
  p.flags = reinterpret_cast<Arrivals*>(at); at += align256(pairs * 8);
  p.left = reinterpret_cast<Arrivals*>(at);
  p.tag = arrivals_tag();
  p.epoch = arrivals_epoch();
  p.status = umma_status_ptr();
  if (!p.epoch || !p.status) return B2Q_ERR_CUDA;
  if (a.bf16) return a.E <= 128 ? run<true, 4>(p, st) : (a.E <= 256 ? run<true, 8>(p, st) : run<true, 32>(p, st));
  return a.E <= 128 ? run<false, 4>(p, st) : (a.E <= 256 ? run<false, 8>(p, st) : run<false, 32>(p, st));
}

}  // namespace b2q
