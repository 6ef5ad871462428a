// Int8 GEMM on tcgen05: out[m, n] = scale[m] wscale[n] sum_k codes[m, k] w[n, k] (+ bias[n]), dense where i8_stream.cu does not serve, and
// grouped by expert.
//
// Both operands go from TMA (128-byte-swizzled boxes of 128 k) straight into tcgen05.mma kind::i8; sums are exact 32-bit integers in
// tensor memory, and scales, bias and rounding happen once per output.  The 128 tokens of a tile are the MMA's rows, up to 256 weight rows
// its columns: a thread of the epilogue then has consecutive outputs of one token.  With the weights as columns a tile can have any
// multiple of sixteen of them, so that the weight rows of a layer are dealt out evenly to the SMs, whatever their number.
//
// Three forms of one kernel, persistent but for the second:
//  * one CTA per tile; two accumulators, so that a tile is drained and stored while the next one is multiplied;
//  * SPLIT: a cluster of two or four CTAs per tile, each with a share of k.  The partial sums meet in distributed shared memory; being
//    integers, they add up to the same whatever the division.  For layers of few rows, whose tiles would leave SMs idle;
//  * PAIR: two CTAs share a tile of 256 tokens and up to 256 weight rows (cta_group::2), each loading half of either.  A CTA then pulls 64 bytes
//    per cycle of MMA through L2 where a tile of its own would take 96.
// GATED (grouped, expert up projection): half of a tile's columns are gate rows, half the up rows of the same outputs, and the epilogue
// stores silu(gate) * up.
//
// Bound by the MMA in prompts: 4001 x 17408 x 5120 226 us in runs too short for the power cap, 3.15 PFLOP/s of int8, and 251 back to back for seconds, 2.84; 2048 x
// 8192 x 28672 291 and 340.  By HBM with few tokens (27 x 17408 x 5120 16.6 us, 5.4 TB/s), where a split of k or half tiles keep all SMs loading.
//
// No multicast load; every mbarrier wait is bounded, as in the other tcgen05 kernels.
#include "umma_gemm.cuh"
#include "sm100.cuh"
#include "i8.cuh"

namespace b2q {

using namespace sm100;

namespace ui8 {
enum { ST_EMPTY = 801, ST_FULL = 802, ST_ACCEMPTY = 803, ST_ACCFULL = 804, ST_XEMPTY = 805 };
constexpr int EPI = 8, FIRST_EPI = 4, THREADS = 32 * (FIRST_EPI + EPI);      // warps: weights, MMA, tokens, (none), epilogue
constexpr int MAX_STAGES = 16, TABLE = 256;
constexpr int STG_BYTES = EPI * 2048;                      // 32 rows x 64 bytes for every epilogue warp
constexpr int TAIL = STG_BYTES + 2 * 2 * TABLE * 4 + 512;  // staging, scale and bias tables of two tiles, barriers
constexpr int SMEM_MAX = 232448;
constexpr int OVERREAD = 16384;                            // an MMA reads 128 token rows, however few are loaded

struct Params {
  const float* xs; const void* ws; int ws_dtype; const void* bias;
  uint16_t* out; int64_t ldo; int out_bf16, vec_out;
  int out_f32;                                             // grouped, not gated
  int M, N;
  int nks;                                                 // stages that K takes
  int h;                                                   // weight rows (MMA columns) per tile
  int n_strips, m_tiles, m_group, total;                   // total: tiles of a dense launch
  int tok_rows, tok_box;                                   // tokens per tile; rows of the token box
  int stages, a_bytes, stage_bytes, split;
  const int32_t* tiles; const int32_t* offsets;            // grouped
  int early;                                               // dense: weights may be read before the kernels in front are done
  int* status;
};

struct Tile { int tok0, rows, n0, cols, w0, w1; };         // cols: valid outputs; w0: first weight row in memory, w1: of the up half

template <bool GROUPED, bool GATED> __device__ __forceinline__ Tile tile_at(const Params& p, int id) {
  Tile t;
  if constexpr (GROUPED) {
    const int ti = id / p.n_strips, st = id - ti * p.n_strips;
    const int e = __ldcg(p.tiles + 4 + 2 * ti), r0 = __ldcg(p.tiles + 4 + 2 * ti + 1);      // from L2: they may be read early
    const int width = GATED ? p.h / 2 : p.h;
    t.tok0 = __ldcg(p.offsets + e) + r0;
    t.rows = min(p.tok_rows, __ldcg(p.offsets + e + 1) - t.tok0);
    t.n0 = st * width;
    t.cols = min(width, p.N - t.n0);
    t.w0 = (GATED ? 2 : 1) * e * p.N + t.n0;
    t.w1 = t.w0 + p.N;
  } else {
    // m_group token tiles against all strips before the next group: what runs at one time shares both operands in L2
    const int per = p.m_group * p.n_strips, gi = id / per, left = id - gi * per, m0 = gi * p.m_group;
    const int gm = min(p.m_group, p.m_tiles - m0), st = left / gm, mt = m0 + left - st * gm;
    t.tok0 = mt * p.tok_rows;
    t.rows = min(p.tok_rows, p.M - t.tok0);
    t.n0 = st * p.h;
    t.cols = min(p.h, p.N - t.n0);
    t.w0 = t.n0;
    t.w1 = 0;
  }
  return t;
}

__device__ __forceinline__ uint4 ld_cluster(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128v(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_out(float a, float b, int bf16) { return bf16 ? pack2<true>(a, b) : pack2<false>(a, b); }
// A warp's 32 rows of 64 bytes through shared memory, so that four lanes store a row's 64 bytes together; 16-byte pieces are permuted
// against bank conflicts.
__device__ __forceinline__ void stage_rows(uint32_t stg, int lane, const uint32_t (&o)[16]) {
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) sts128(stg + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4), o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
  __syncwarp();
}
__device__ __forceinline__ void store_rows(uint32_t stg, int lane, int rows, int bytes, uint8_t* out, int64_t pitch) {      // bytes: of a row, of 64
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = i * 8 + (lane >> 2), q = lane & 3;
    const uint4 v = lds128v(stg + rr * 64 + ((q ^ ((rr >> 1) & 3)) << 4));
    if (rr < rows && 16 * q < bytes) *reinterpret_cast<uint4*>(out + rr * pitch + q * 16) = v;
  }
}
}  // namespace ui8

template <int KPS, bool PAIR, bool SPLIT, bool GROUPED, bool GATED>      // KPS: 128-k boxes of each operand in a stage
__global__ void __launch_bounds__(ui8::THREADS, 1)
umma_i8_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const ui8::Params p) {
  using namespace ui8;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  // [stages of (token box, weight box)] [room for the MMA's reads beyond a low token box] [staging] [tables] [barriers]
  const uint32_t stg_off = p.stages * p.stage_bytes + (p.tok_box < 128 ? OVERREAD : 0);
  const uint32_t tab_off = stg_off + STG_BYTES, bar = base + tab_off + 4 * TABLE * 4;
  float* tab = reinterpret_cast<float*>(gen + tab_off);    // [2 tiles][scales, biases][TABLE]
  const uint32_t full = bar, empty = bar + 8 * MAX_STAGES, acc_full = bar + 16 * MAX_STAGES, acc_empty = acc_full + 16;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + (acc_empty + 16 - base));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + (acc_empty + 24 - base));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR || SPLIT ? cluster_ctarank() : 0;
  const int group = PAIR ? 2 : (SPLIT ? p.split : 1);      // CTAs that work on one tile
  const int first = (int)blockIdx.x / group, step = (int)gridDim.x / group;
  const int ks0 = SPLIT ? (int)rank * p.nks / p.split : 0, ks1 = SPLIT ? ((int)rank + 1) * p.nks / p.split : p.nks;

  grid_dep_release();
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) { mbar_init(full + 8 * i, 2); mbar_init(empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, PAIR ? 2 * EPI : EPI); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) { tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512); tmem_relinquish_pair(); }
    else { tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();                  // both CTAs' barriers exist before anything is signalled across
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // A dense launch knows its tiles.  A grouped one has their list, and its weights, as soon as it begins: that is when the tokens' codes are being made at
  // the earliest, and the kernel that makes them lets it begin only once it has itself seen the routing, and so all that came before, done (COPIES in
  // i8_quant.cu).  16 tokens, 8 experts of 4096 x 2048, top-2: 55 -> 50 us.
  const int total = GROUPED ? __ldcg(p.tiles) * p.n_strips : p.total;

  if (warp == 0) {
    // ---- weights; boxes that begin beyond K read as zero ----
    if (elect_one()) {
      tma_prefetch_desc(&tm_w);
      const int box = PAIR || GATED ? p.h / 2 : p.h;
      const uint32_t bytes = (uint32_t)(p.stage_bytes - p.a_bytes) * (PAIR ? 2u : 1u);
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      if (!GROUPED && !p.early) grid_dep_wait();
      for (int id = first; ok && id < total; id += step) {
        const Tile t = tile_at<GROUPED, GATED>(p, id);
        for (int ks = ks0; ks < ks1; ++ks) {
          ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_EMPTY);
          if (!ok) break;
          const uint32_t dst = base + s * p.stage_bytes + p.a_bytes;
          if (rank == 0 || !PAIR) mbar_expect_tx(full + 8 * s, bytes);
#pragma unroll
          for (int i = 0; i < KPS; ++i) {
            const int k = (ks * KPS + i) * 128;
            if constexpr (PAIR) {
              tma_load_2d_pair(dst + i * box * 128, &tm_w, k, t.w0 + (int)rank * box, map_to_cta(full + 8 * s, 0));
            } else {
              tma_load_2d(dst + i * p.h * 128, &tm_w, k, t.w0, full + 8 * s);
              if constexpr (GATED) tma_load_2d(dst + i * p.h * 128 + box * 128, &tm_w, k, t.w1, full + 8 * s);
            }
          }
          ++issued;
          if (++s == p.stages) { s = 0; par ^= 1u; }
        }
      }
      // gave up: the copies issued land before the CTA leaves (a pair's are counted on the leader's barriers, and the peer stays with it)
      if (!ok && (rank == 0 || !PAIR)) drain_issued(full, p.stages, issued);
    }
  } else if (warp == 2) {
    // ---- tokens ----
    if (elect_one()) {
      tma_prefetch_desc(&tm_x);
      const uint32_t bytes = (uint32_t)p.a_bytes * (PAIR ? 2u : 1u);
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      grid_dep_wait();
      for (int id = first; ok && id < total; id += step) {
        const Tile t = tile_at<GROUPED, GATED>(p, id);
        for (int ks = ks0; ks < ks1; ++ks) {
          ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_XEMPTY);
          if (!ok) break;
          const uint32_t dst = base + s * p.stage_bytes;
          if (rank == 0 || !PAIR) mbar_expect_tx(full + 8 * s, bytes);
#pragma unroll
          for (int i = 0; i < KPS; ++i) {
            const int k = (ks * KPS + i) * 128;
            if constexpr (PAIR) tma_load_2d_pair(dst + i * 16384, &tm_x, k, t.tok0 + (int)rank * 128, map_to_cta(full + 8 * s, 0));
            else tma_load_2d(dst + i * p.tok_box * 128, &tm_x, k, t.tok0, full + 8 * s);
          }
          ++issued;
          if (++s == p.stages) { s = 0; par ^= 1u; }
        }
      }
      if (!ok && (rank == 0 || !PAIR)) drain_issued(full, p.stages, issued);
    }
  } else if (warp == 1) {
    if ((!PAIR || rank == 0) && elect_one()) {
      const uint32_t idesc = instr_desc_i8(1u, 1u, PAIR ? 256u : 128u, (uint32_t)p.h);
      const uint64_t x_step = (uint64_t)(PAIR ? 128 : p.tok_box) * 8, w_step = (uint64_t)(PAIR ? p.h / 2 : p.h) * 8;      // from box to box, in 16 bytes
      int s = 0, it = 0;
      uint32_t par = 0u;
      bool ok = true;
      for (int id = first; ok && id < total; id += step, ++it) {
        const int b = it & 1;
        if (it >= 2) ok = mbar_wait(acc_empty + 8 * b, ((it >> 1) - 1) & 1, abort_flag, p.status, ST_ACCEMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + b * 256;
        for (int ks = ks0; ks < ks1; ++ks) {
          ok = mbar_wait(full + 8 * s, par, abort_flag, p.status, ST_FULL);
          if (!ok) break;
          tc_fence_after();
          uint64_t da = smem_desc_sw128(base + s * p.stage_bytes);
          uint64_t db = smem_desc_sw128(base + s * p.stage_bytes + p.a_bytes);
#pragma unroll
          for (int j = 0; j < KPS; ++j, da += x_step, db += w_step) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (PAIR) mma_i8_pair(d, da + 2 * i, db + 2 * i, idesc, ks > ks0 || j > 0 || i > 0);
              else mma_i8(d, da + 2 * i, db + 2 * i, idesc, ks > ks0 || j > 0 || i > 0);
            }
          }
          if constexpr (PAIR) tc_commit_pair(empty + 8 * s, 3); else tc_commit(empty + 8 * s);
          if (++s == p.stages) { s = 0; par ^= 1u; }
        }
        if (!ok) break;
        if constexpr (PAIR) tc_commit_pair(acc_full + 8 * b, 3); else tc_commit(acc_full + 8 * b);
      }
    }
  } else if (warp >= FIRST_EPI) {
    // ---- epilogue: lane quadrant = warp & 3 (tokens), column chunks of 32 shared by the two warps of a quadrant ----
    const int quad = warp & 3, half = (warp - FIRST_EPI) >> 2, etid = threadIdx.x - 32 * FIRST_EPI;
    const uint32_t stg = base + stg_off + (warp - FIRST_EPI) * 2048;
    grid_dep_wait();
    int it = 0;
    bool ok = true;                                        // a warp that has given up still goes to the barrier where the others expect it
    for (int id = first; id < total; id += step, ++it) {
      const Tile t = tile_at<GROUPED, GATED>(p, id);
      const int b = it & 1;
      float* sc = tab + b * 2 * TABLE;
      float* bi = sc + TABLE;
      {
        // scales of the tile's columns: thread i has column i (gated: gate columns, then up columns)
        const int width = GATED ? p.h / 2 : p.h, col = GATED && etid >= width ? etid - width : etid;
        float v = 0.f, w = 0.f;
        if (etid < p.h && col < t.cols) {
          const int64_t at = GATED ? (int64_t)(etid >= width ? t.w1 : t.w0) + col : (int64_t)t.w0 + col;
          v = load_scalar(p.ws, at, p.ws_dtype);
          if (p.bias) w = load_scalar(p.bias, t.n0 + col, p.out_bf16 ? B2Q_BF16 : B2Q_F16);
        }
        sc[etid] = v;
        bi[etid] = w;
      }
      const int trow = (PAIR ? (int)rank * 128 : 0) + quad * 32 + lane;      // this lane's token within the tile
      const float xs = trow < t.rows ? ld_f32(p.xs + t.tok0 + trow) : 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI) : "memory");
      ok = ok && mbar_wait_warp(acc_full + 8 * b, (it >> 1) & 1, abort_flag, p.status, ST_ACCFULL);
      if (!ok) continue;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + b * 256;
      const int row0 = (PAIR ? (int)rank * 128 : 0) + quad * 32;
      if constexpr (SPLIT) {
        // partial sums into this CTA's shared memory, whose stages nobody uses any more
        const int pitch = p.h + 4;
        for (int c = half * 32; row0 < t.rows && c < t.cols; c += 64) {
          uint32_t r[32];
          tmem_ld32(acc + c, r);
          tmem_ld_wait();
          const uint32_t at = base + (uint32_t)((quad * 32 + lane) * pitch + c) * 4;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (c + i < p.h) sts128(at + i * 4, r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      } else {
        if (GATED || (GROUPED && p.out_f32)) {
          // sixteen outputs in fp32 at a time
          float* out = reinterpret_cast<float*>(p.out) + (int64_t)(t.tok0 + row0) * p.ldo + t.n0;
          const float* us = sc + p.h / 2;
          const int end = row0 < t.rows ? t.cols : 0;
          uint32_t r[16], u[16], v[16];
          auto fetch = [&](int c) {
            tmem_ld16(acc + c, r);
            if constexpr (GATED) tmem_ld16(acc + p.h / 2 + c, u);
          };
          if (half * 16 < end) fetch(half * 16);
          for (int c = half * 16; c < end; c += 32) {
            tmem_ld_wait();
            const float4* g4 = reinterpret_cast<const float4*>(sc + c);
            const float4* u4 = reinterpret_cast<const float4*>(us + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 gs = g4[i], uv = GATED ? u4[i] : gs;
              const float gv[4] = {gs.x, gs.y, gs.z, gs.w}, uw[4] = {uv.x, uv.y, uv.z, uv.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float y = i8_scaled((int)r[4 * i + j], xs, gv[j]);
                v[4 * i + j] = __float_as_uint(GATED ? silu_mul_f(y, i8_scaled((int)u[4 * i + j], xs, uw[j])) : y);
              }
            }
            if (c + 32 < end) fetch(c + 32);               // on its way while these are stored
            stage_rows(stg, lane, v);
            if (p.vec_out && (t.cols - c) % 4 == 0) {
              store_rows(stg, lane, t.rows - row0, (t.cols - c) * 4, reinterpret_cast<uint8_t*>(out + c), p.ldo * 4);
            } else {
              for (int rr = 0; rr < 32 && row0 + rr < t.rows; ++rr) {
                const int i = lane & 15;
                uint32_t w;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(stg + rr * 64 + (((i >> 2) ^ ((rr >> 1) & 3)) << 4) + (i & 3) * 4) : "memory");
                if (lane < 16 && c + i < t.cols) out[rr * p.ldo + c + i] = __uint_as_float(w);
              }
            }
          }
        } else {
          uint16_t* out = p.out + (int64_t)(t.tok0 + row0) * p.ldo + t.n0;
          const int end = row0 < t.rows ? t.cols : 0;
          uint32_t r[32], o[16];
          if (half * 32 < end) tmem_ld32(acc + half * 32, r);
          for (int c = half * 32; c < end; c += 64) {
            tmem_ld_wait();
            const float4* s4 = reinterpret_cast<const float4*>(sc + c);
            const float4* b4 = reinterpret_cast<const float4*>(bi + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 sv = s4[i], bv = p.bias ? b4[i] : make_float4(0.f, 0.f, 0.f, 0.f);
              o[2 * i] = pack_out(i8_output((int)r[4 * i], xs, sv.x, bv.x), i8_output((int)r[4 * i + 1], xs, sv.y, bv.y), p.out_bf16);
              o[2 * i + 1] = pack_out(i8_output((int)r[4 * i + 2], xs, sv.z, bv.z), i8_output((int)r[4 * i + 3], xs, sv.w, bv.w), p.out_bf16);
            }
            if (c + 64 < end) tmem_ld32(acc + c + 64, r);  // on its way while this chunk is stored
            stage_rows(stg, lane, o);
            if (p.vec_out && (t.cols - c) % 8 == 0) {
              store_rows(stg, lane, t.rows - row0, (t.cols - c) * 2, reinterpret_cast<uint8_t*>(out + c), p.ldo * 2);
            } else {
              for (int rr = 0; rr < 32 && row0 + rr < t.rows; ++rr) {
                const int q = lane >> 3;
                uint16_t v;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(stg + rr * 64 + ((q ^ ((rr >> 1) & 3)) << 4) + (lane & 7) * 2) : "memory");
                if (c + lane < t.cols) out[rr * p.ldo + c + lane] = v;
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_cluster(map_to_cta(acc_empty + 8 * b, 0));
          else mbar_arrive(acc_empty + 8 * b);
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (SPLIT) {
    cluster_sync_all();                                    // every CTA's partial sums are there
    if (first < total && !*abort_flag) {
      const Tile t = tile_at<GROUPED, GATED>(p, first);
      const int pitch = p.h + 4, eights = (t.cols + 7) / 8, items = t.rows * eights;
      for (int i = (int)rank * THREADS + threadIdx.x; i < items; i += p.split * THREADS) {
        const int row = i / eights, c = (i - row * eights) * 8;
        int sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const uint32_t at = base + (uint32_t)(row * pitch + c) * 4;
        for (int j = 0; j < p.split; ++j) {
          const uint32_t from = map_to_cta(at, j);
          const uint4 a = ld_cluster(from), d = ld_cluster(from + 16);
          sum[0] += (int)a.x; sum[1] += (int)a.y; sum[2] += (int)a.z; sum[3] += (int)a.w;
          sum[4] += (int)d.x; sum[5] += (int)d.y; sum[6] += (int)d.z; sum[7] += (int)d.w;
        }
        const float xs = ld_f32(p.xs + t.tok0 + row);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = i8_output(sum[k], xs, tab[c + k], tab[TABLE + c + k]);
        uint16_t* out = p.out + (int64_t)(t.tok0 + row) * p.ldo + t.n0 + c;
        const uint4 o = make_uint4(pack_out(v[0], v[1], p.out_bf16), pack_out(v[2], v[3], p.out_bf16), pack_out(v[4], v[5], p.out_bf16),
                                   pack_out(v[6], v[7], p.out_bf16));
        if (p.vec_out && c + 8 <= t.cols) {
          *reinterpret_cast<uint4*>(out) = o;
        } else {
          const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (c + k < t.cols) out[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
        }
      }
    }
    cluster_sync_all();                                    // nobody leaves while its sums may be read
  }
  if constexpr (PAIR) cluster_sync_all();                  // nor while the partner may still signal it
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, 512); else tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace ui8 {
static int round_up(int v, int a) { return (v + a - 1) / a * a; }

template <int KPS, bool PAIR, bool SPLIT, bool GROUPED, bool GATED>
static int launch_form(const CUtensorMap& tx, const CUtensorMap& tw, Params& p, int grid, cudaStream_t st) {
  p.a_bytes = KPS * p.tok_box * 128;
  p.stage_bytes = p.a_bytes + KPS * (PAIR ? p.h / 2 : p.h) * 128;
  const int over = p.tok_box < 128 ? OVERREAD : 0, room = SMEM_MAX - 1024 - TAIL - over;
  p.stages = room / p.stage_bytes;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  int bytes = p.stages * p.stage_bytes;
  if (SPLIT && bytes < (p.tok_box < 32 ? 32 : p.tok_box) * (p.h + 4) * 4) return B2Q_ERR_LIMIT;      // partial sums use the stages' room
  // Never less than 165 KB (16 stages of 8 KB), so that no other CTA with tensor memory fits beside this one.  A kernel lets the next one begin before it has
  // allocated its own; were both on an SM, it could wait for columns that the next one holds while that waits for it.
  const int smem = 1024 + bytes + over + TAIL;
  auto kern = umma_i8_kernel<KPS, PAIR, SPLIT, GROUPED, GATED>;
  static thread_local bool configured[16] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX) != cudaSuccess) return B2Q_ERR_CUDA;
    if (dev < 16) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (PAIR || SPLIT) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = PAIR ? 2 : p.split; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (tls().overlap_mode > 0) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at; cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kern, tx, tw, p);               // launch_status() reports
  note_launch(PAIR ? "umma_i8_pair" : (SPLIT ? "umma_i8_split" : "umma_i8"));
  return launch_status();
}

template <bool SPLIT, bool GROUPED, bool GATED>
static int launch(int kps, const CUtensorMap& tx, const CUtensorMap& tw, Params& p, int grid, cudaStream_t st) {
  return kps == 1 ? launch_form<1, false, SPLIT, GROUPED, GATED>(tx, tw, p, grid, st) : launch_form<2, false, SPLIT, GROUPED, GATED>(tx, tw, p, grid, st);
}

// A stage costs its producers and the MMA's issuer some 150 ns whatever is in it, so low weight boxes come in twos (one / two / four per
// stage: 8 x 5120 x 5120, 48 rows, 9.1 / 8.0 / 8.0 us; 64 x 4096 x 4096, 32 rows, 7.8 / 6.9 / 7.3; 8 x 17408 x 5120, 128 rows, 16.0 / 16.5).
static int boxes_per_stage(int h) { return h <= 64 ? 2 : 1; }

// How a dense launch is divided: weight rows per tile, CTAs per tile, or pairs of CTAs with tiles of 256 tokens, by a fitted time in ns.
// A tile's 128 k cost 0.45 ns per token row of its box and 1.55 per weight row, 90 at least (a pair's 45 and 1.25 per weight row), and 1.2 and 0.3 more where K is no
// multiple of 128, so that a row of a box lies in two lines; its outputs 0.1 each, behind the next tile's k but for the last; a launch
// 3500, another round 500; the meeting of a split tile's sums 1800 and 0.22 per output; and all of it at least what the bytes take out of
// DRAM.  Over 46 shapes of 17 to 4096 tokens the choice took 1.02 times as long as the best division tried (16 x 1024 x 8192: one / two / four CTAs per
// tile 9.6 / 8.0 / 6.8 us, 256 x 4096 x 4096: 8.5 / 11.2 / 16.3, 1024 x 8192 x 8192: 53.0 alone, 47.3 in pairs of 256 rows, 45.8 of 224).  Eight CTAs per tile lost everywhere;
// of clusters of four 32 fit the SMs at a time, not 37.
struct Plan { int h, split; bool pair; };
static Plan plan(int M, int N, int K, int tok_box) {
  const int sms = sm_count(), nkb = (K + 127) / 128, m_tiles = (M + 127) / 128, rows = M < 128 ? M : 128;
  Plan best{256, 1, false};
  double least = 1e30;
  const double dram = ((double)N * nkb * 128 + (double)M * nkb * 128 + 2.0 * M * N) / 6300;
  for (int split = 1; split <= 4 && 2 * split <= nkb; split *= 2) {
    const int slots = split == 4 ? sms * 7 / 32 : sms / split;
    for (int rounds = 1; rounds <= (split > 1 ? 1 : 8); ++rounds) {
      const int strips = slots * rounds / m_tiles;
      if (strips == 0) continue;
      const int h = round_up((N + strips - 1) / strips, 16);
      if (h > 256) continue;
      const double k128 = fmax(90, 0.45 * tok_box + 1.55 * h) + (K % 128 ? 1.2 * tok_box + 0.3 * h : 0), drain = 0.1 * rows * h;
      double ns = fmax(dram, rounds * fmax(drain, (nkb + split - 1) / split * k128)) + 500.0 * (rounds - 1) + drain;
      if (split > 1) ns += 1800 + 0.22 * rows * h;
      if (ns < least) { least = ns; best = Plan{h, split, false}; }
    }
  }
  for (int h = 256; M > 128 && h >= 128; h -= 32) {        // a pair's columns come in 32s
    const double rounds = ((int64_t)(M + 255) / 256 * ((N + h - 1) / h) + sms / 2 - 1) / (sms / 2);
    const double ns = fmax(dram, rounds * fmax(13.0 * h, nkb * (45 + 1.25 * h))) + 500.0 * (rounds - 1) + 13.0 * h;
    if (ns < least) { least = ns; best = Plan{h, 1, true}; }
  }
  if (least >= 1e30) best.pair = M > 128;                  // more tiles than eight rounds hold
  return best;
}
}  // namespace ui8

int umma_i8_linear(const I8LinearArgs& a, cudaStream_t st) {
  using namespace ui8;
  if (!tensor_map_encoder()) return B2Q_ERR_CUDA;
  Params p{};
  p.xs = a.xs; p.ws = a.ws; p.ws_dtype = a.ws_dtype; p.bias = a.bias;
  p.out = reinterpret_cast<uint16_t*>(a.out); p.ldo = a.ldo; p.out_bf16 = a.out_bf16; p.vec_out = aligned16(a.out) && a.ldo % 8 == 0;
  p.M = a.M; p.N = a.N;
  const int nkb = (a.K + 127) / 128;
  p.early = tls().overlap_mode == 2;
  p.status = umma_status_ptr();
  if (!p.status) return B2Q_ERR_CUDA;
  const int sms = sm_count();
  p.tok_box = a.M <= 16 ? 16 : (a.M <= 32 ? 32 : (a.M <= 64 ? 64 : 128));
  const Plan pl = plan(a.M, a.N, a.K, p.tok_box);
  const bool pair = pl.pair;
  CUtensorMap tx, tw;
  p.h = pl.h; p.split = pl.split; p.tok_rows = pair ? 256 : 128;
  const int kps = pair ? 1 : boxes_per_stage(p.h);
  p.nks = (nkb + kps - 1) / kps;
  if (p.split > p.nks) p.split = p.nks;
  p.n_strips = (a.N + p.h - 1) / p.h;
  p.m_tiles = (a.M + p.tok_rows - 1) / p.tok_rows;
  p.m_group = p.m_tiles < 16 ? p.m_tiles : 16;
  if ((int64_t)p.n_strips * p.m_tiles > INT32_MAX / 8) return B2Q_ERR_LIMIT;
  p.total = p.n_strips * p.m_tiles;
  int rc = make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.xq, a.M, a.K, (uint64_t)a.ldx, p.tok_box, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.N, a.K, (uint64_t)a.K, pair ? p.h / 2 : p.h, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  if (pair) return launch_form<1, true, false, false, false>(tx, tw, p, 2 * (p.total < sms / 2 ? p.total : sms / 2), st);
  if (p.split > 1) return launch<true, false, false>(kps, tx, tw, p, p.total * p.split, st);
  return launch<false, false, false>(kps, tx, tw, p, p.total < sms ? p.total : sms, st);
}

// Token height of the tiles: an MMA has 128 token rows however few are loaded, so this is about bytes of tokens per tile only.
int i8_grouped_tile(int64_t rows, int E) {
  const int64_t avg = (rows + E - 1) / E;
  return avg <= 24 ? 32 : (avg <= 48 ? 64 : 128);
}

int umma_i8_grouped(const I8GroupedArgs& a, cudaStream_t st) {
  using namespace ui8;
  if (!tensor_map_encoder()) return B2Q_ERR_CUDA;
  Params p{};
  p.xs = a.xs; p.ws = a.ws; p.ws_dtype = a.ws_dtype;
  p.out = reinterpret_cast<uint16_t*>(a.out); p.ldo = a.N; p.out_bf16 = a.out_bf16; p.vec_out = aligned16(a.out) && a.N % 8 == 0;
  p.out_f32 = a.out_f32;
  p.M = a.rows; p.N = a.N;
  p.tiles = a.tiles; p.offsets = a.offsets; p.split = 1;
  p.status = umma_status_ptr();
  if (!p.status) return B2Q_ERR_CUDA;
  // Outputs of a tile: 128 gated, 256 otherwise, and half of that where there may be no more than two tiles per SM, which halves the last round
  // (6 tokens, 8 experts of 2048 x 2048, top-8, 37.4 -> 34.5 us; 16, 16 of 1024 x 4096, top-8, 56.0 -> 53.2; 24, 16 of 2048 x 2048, top-4, 53.9 -> 50.4).  With
  // more tiles it costs: 4096 tokens, 128 experts of 2048 x 768, top-8, 300 -> 392 us.
  const int token_tiles = (a.rows + a.tile - 1) / a.tile, experts = a.E < a.rows ? a.E : a.rows, likely = token_tiles > experts ? token_tiles : experts;
  int most = a.gated ? 128 : 256;
  if ((int64_t)likely * ((a.N + most - 1) / most) <= 2 * sm_count()) most /= 2;
  p.n_strips = (a.N + most - 1) / most;
  const int width = round_up((a.N + p.n_strips - 1) / p.n_strips, 16);
  p.h = a.gated ? 2 * width : width;
  p.tok_rows = p.tok_box = a.tile;
  const int kps = boxes_per_stage(p.h);
  p.nks = ((a.K + 127) / 128 + kps - 1) / kps;
  const int64_t w_rows = (int64_t)a.E * a.N * (a.gated ? 2 : 1);
  if (w_rows > INT32_MAX || (int64_t)a.tile_cap * p.n_strips > INT32_MAX / 2) return B2Q_ERR_LIMIT;
  CUtensorMap tx, tw;
  int rc = make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.xq, a.rows, a.K, (uint64_t)a.K, a.tile, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, w_rows, a.K, (uint64_t)a.K, width, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  const int most_tiles = a.tile_cap * p.n_strips, grid = most_tiles < sm_count() ? most_tiles : sm_count();
  return a.gated ? launch<false, true, true>(kps, tx, tw, p, grid, st) : launch<false, true, false>(kps, tx, tw, p, grid, st);
}

}  // namespace b2q
