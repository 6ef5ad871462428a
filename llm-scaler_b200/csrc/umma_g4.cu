// GEMM of many tokens on 4-bit group-quantised weights by tcgen05: out[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]), w = (q - z) s rounded once to the activations' type;
// dense where g4_stream.cu does not serve, and grouped by expert.
//
// 128 weight rows are the MMA's rows, a tile of NT tokens its columns.  Raw codes come by TMA; transform warps turn them into 16-bit values, a thread a row, and write
// them straight into tensor memory as the MMA's A operand; tokens come by TMA.  q - z is exact (the code is put below a power of two and that power plus z
// subtracted), times s is the one rounding; it is of the size of the output's own.
//
// Two CTAs share a tile of 256 rows (cta_group::2), each with its own 128 rows in tensor memory and half of the tokens in shared memory: a CTA alone would pull twice the
// tokens through L2, which at 9 TB/s is what bounds narrow tiles too (64 x 17408 x 5120: 89 MB of tokens, 45 in pairs, beside 46 of weights).
//
// A persistent CTA has separate warps for the weights' copies, the tokens' copies, the MMA, the epilogue and the transform, so that nothing of one tile stops the stream of the
// next.  An operand stage is 128 k; each ring stage stays with one group of four transform warps, since a parity wait cannot tell a phase from the one before the
// last.
//
//  * Where strips of 256 rows are fewer than pairs of SMs, k is cut into pieces; whoever delivers the last of a strip's partial sums adds them up in order (arrivals.cuh).
//  * GATED (expert up projection): a warp's 32 rows are 16 gate and 16 up rows of the same outputs, and the epilogue stores silu(gate) * up.
//
// In graphs: 4001 x 17408 x 5120 484 to 587 us by the GPU's power (1.22 to 1.47 PFLOP/s), 33 x 17408 x 5120 in groups of 32 22.0, 100 x 4096 x 4096 18.5.  Up to 128 tokens the
// transform sets the pace, 650 to 750 cycles for a stage, and no unit is full while it does: of 33 x 17408 x 5120 issue slots 52 %, the ALU pipe 45, the 16-bit one 26, tensor cores 26 (grouped
// 64, 54, 32, 32); fp16, whose decode has two operations fewer for a word, takes 24.0 us where bf16 takes 25.2 (cold, one launch).  Of the 9.6 cycles between two instructions of a warp 2.1 wait for
// loads, 1.7 at barriers, 1.1 for fixed latencies.  What would shorten the chain is not known; more groups and more slots did not.
//
// No multicast load; every mbarrier wait is bounded, as in the other tcgen05 kernels.
#include <type_traits>
#include "umma_gemm.cuh"
#include "sm100.cuh"
#include "arrivals.cuh"
#include "g4.cuh"

namespace b2q {

using namespace sm100;

namespace ug4 {
enum { ST_RAWEMPTY = 951, ST_RAWFULL = 952, ST_AEMPTY = 953, ST_FULL = 954, ST_XEMPTY = 955, ST_ACCEMPTY = 957, ST_ACCFULL = 958 };

template <int NT> struct Cfg {
  static constexpr int NBUF = NT <= 128 ? 2 : 1;             // accumulators
  static constexpr int COLS = NT, A_COL0 = NBUF * COLS;
  static constexpr int S = (512 - A_COL0) / 64 > 6 ? 6 : (512 - A_COL0) / 64;      // stages of 128 k: operand columns and tokens
  // Transform groups.  Two slots a group hide its waits where tensor memory has room for them; the accumulators of 128 tokens leave four slots, and four groups with one each
  // do better than two with two.
  static constexpr int DG = NT == 256 ? 2 : (NT == 128 ? 4 : 3);
  static constexpr int EW = NT <= 64 ? 4 : 8;                // epilogue warps
  static constexpr int FIRST_EPI = 4, FIRST_DEQ = FIRST_EPI + EW, THREADS = 32 * (FIRST_DEQ + 4 * DG);
  static constexpr int TOK = NT / 2;                         // tokens that a CTA loads
  static constexpr int X_BYTES = TOK * 256, RAW_BYTES = 8192;
  static constexpr int RS = NT == 256 ? 6 : (NT == 128 ? 8 : 9);      // raw stages, a multiple of DG
  static constexpr int STG = EW * 2048;                      // 32 tokens x 32 columns for every epilogue warp
  static constexpr int TABLE = 48;                           // tiles of a grouped launch that every role finds in shared memory
  static constexpr int USED = S * X_BYTES + RS * RAW_BYTES + STG + TABLE * 16 + 1024;
  static constexpr int SMEM = 1024 + (USED < 170 * 1024 ? 170 * 1024 : USED);      // one CTA with tensor memory on an SM: see umma_i8.cu
  static_assert(RS % DG == 0 && S % DG == 0 && S > 0 && SMEM <= 232448, "rings");
};

// Whether the tokens' k come permuted in eights (g4_position), which saves two operations of nine to seven for a word's eight codes (fp16: four).  A pass over the tokens pays
// where the conversion is what bounds the kernel.
template <int NT> constexpr bool permuted(bool grouped) { return grouped || NT < 256; }

struct Params {
  const uint16_t* s; const uint8_t* z; int64_t s_expert; int s_rows;      // scales [groups][s_rows]
  const uint16_t* bias; const float* out_w;
  uint16_t* out; int64_t ldo; int vec_out;
  int M, N, K, groups, nks;                                // nks: stages that K takes
  int n_strips, m_tiles, m_group, pieces, total;           // total: tiles of a dense launch
  float* partials; Arrivals* arrivals; Arrivals tag; const Arrivals* epoch;
  const int32_t* tiles; const int32_t* offsets;            // grouped
  int early;                                               // weights (grouped: and the tile list) may be read before the kernel in front is done
  uint32_t mask, magic;                                    // of the decode: as constants they take an operation each
  int* status;
};

// n0: first output column of the CTA or pair; w0: first weight row in memory (of an expert's gate half); k is walked from stage ks0 + turn on and round to it, since CTAs that all
// begin at the same k ask the same L2 lines for the tokens at the same time.
struct Tile {
  int tok0, rows, n0, w0, ks0, n, turn, piece, strip, e;
  __device__ __forceinline__ int stage(int j) const { const int i = j + turn; return ks0 + (i >= n ? i - n : i); }
};

// table: {first token, tokens, expert, strip} of this CTA's tiles, of which it has `known`; id is the n-th of them.
template <int NT, bool GROUPED, bool GATED> __device__ __forceinline__ Tile tile_at(const Params& p, int id, const int4* table, int n, int known) {
  constexpr int WIDTH = GATED ? 128 : 256;                 // output columns of a strip
  Tile t;
  t.piece = 0; t.ks0 = 0; t.n = p.nks; t.e = 0;
  int st;
  if constexpr (GROUPED) {
    int4 v;
    if (n < known) {
      v = table[n];
    } else {
      const int ti = id / p.n_strips, e = __ldcg(p.tiles + 4 + 2 * ti), tok0 = __ldcg(p.offsets + e) + __ldcg(p.tiles + 4 + 2 * ti + 1);
      v = make_int4(tok0, min(NT, __ldcg(p.offsets + e + 1) - tok0), e, id - ti * p.n_strips);
    }
    st = v.w;
    t.tok0 = v.x;
    t.rows = v.y;
    t.n0 = st * WIDTH;
    t.w0 = (GATED ? 2 : 1) * v.z * p.N + t.n0;
    t.strip = 0;
    t.e = v.z;
  } else {
    if (p.pieces > 1) {
      t.strip = id / p.pieces;
      t.piece = id - t.strip * p.pieces;
      t.ks0 = t.piece * p.nks / p.pieces;
      t.n = (t.piece + 1) * p.nks / p.pieces - t.ks0;
      id = t.strip;
    }
    const int per = p.m_group * p.n_strips, gi = id / per, left = id - gi * per, m0 = gi * p.m_group;
    const int gm = min(p.m_group, p.m_tiles - m0);
    st = left / gm;
    const int mt = m0 + left - st * gm;
    t.tok0 = mt * NT;
    t.rows = min(NT, p.M - t.tok0);
    t.n0 = st * WIDTH;
    t.w0 = t.n0;
  }
  t.turn = st * t.n / p.n_strips;                          // below 2^23, since a matrix has fewer than 2^31 scales
  return t;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint16_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory"); }
__device__ __forceinline__ uint32_t ld_u16(const uint16_t* p) { uint32_t v; asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v) : "l"(p)); return v; }
__device__ __forceinline__ uint32_t ld_u8(const uint8_t* p) { uint32_t v; asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v) : "l"(p)); return v; }

// Two 16-bit values at a time.
template <bool BF16> __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF16> __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma2_f16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// Eight codes of a word -> four registers of two values (q - z) s.  PERM: in the order 0, 4, 1, 5, 2, 6, 3, 7, else as they come.  zc: the power of two plus z, twice (fp16 and
// PERM: and -(64 + z) in zh); MORE: bf16, with what z has beyond 127 in more, for 128 + z has to fit eight bits.
template <bool BF16, bool PERM, bool MORE> __device__ __forceinline__ void decode(uint32_t w, uint32_t s2, uint32_t zc, uint32_t zh, uint32_t more, uint32_t MASK, uint32_t MAGIC, uint32_t* o) {
  if constexpr (PERM && !BF16) {
    const uint32_t w8 = w >> 8;
    o[0] = sub2<false>((w & MASK) | MAGIC, zc);
    o[2] = sub2<false>((w8 & MASK) | MAGIC, zc);
    o[1] = fma2_f16((w & (MASK << 4)) | MAGIC, 0x2C002C00u, zh);      // 2^-4 (1024 + 16 q) - (64 + z)
    o[3] = fma2_f16((w8 & (MASK << 4)) | MAGIC, 0x2C002C00u, zh);
  } else if constexpr (PERM) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = sub2<true>(((w >> 4 * i) & MASK) | MAGIC, zc);
  } else {
    const uint32_t w4 = w >> 4;
    o[0] = sub2<BF16>((__byte_perm(w, w4, 0x4400) & MASK) | MAGIC, zc);
    o[1] = sub2<BF16>((__byte_perm(w, w4, 0x5511) & MASK) | MAGIC, zc);
    o[2] = sub2<BF16>((__byte_perm(w, w4, 0x6622) & MASK) | MAGIC, zc);
    o[3] = sub2<BF16>((__byte_perm(w, w4, 0x7733) & MASK) | MAGIC, zc);
  }
  if constexpr (MORE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = sub2<true>(o[i], more);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = mul2<BF16>(o[i], s2);
}

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF16> __device__ __forceinline__ float half_f(uint32_t raw) { return BF16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half((unsigned short)raw)); }

// Sixteen tokens' values of a warp's rows (a lane has one row, tokens 2 i and 2 i + 1 in o[i]) through shared memory to out: rows of 32 consecutive columns.  cols, rows: how
// many there are.
__device__ __forceinline__ void store16(uint32_t stg, const uint32_t (&o)[8], uint16_t* out, int64_t ldo, int rows, int cols, bool vec) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sts16(stg + (2 * i) * 64 + lane * 2, (uint16_t)o[i]);
    sts16(stg + (2 * i + 1) * 64 + lane * 2, (uint16_t)(o[i] >> 16));
  }
  __syncwarp();
  if (vec && cols % 8 == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tk = i * 8 + (lane >> 2), c = (lane & 3) * 8;
      const uint4 v = lds128(stg + tk * 64 + c * 2);
      if (tk < rows && c < cols) *reinterpret_cast<uint4*>(out + tk * ldo + c) = v;
    }
  } else {
    for (int tk = 0; tk < 16 && tk < rows; ++tk) {
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(stg + tk * 64 + lane * 2) : "memory");
      if (lane < cols) out[tk * ldo + lane] = v;
    }
  }
}
}  // namespace ug4

template <bool BF16, int G, int NT, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(ug4::Cfg<NT>::THREADS, 1)
umma_g4_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const ug4::Params p) {
  using namespace ug4;
  using C = Cfg<NT>;
  constexpr bool PERM = permuted<NT>(GROUPED);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  // [token stages] [raw stages] [staging] [tiles] [barriers]
  const uint32_t raw0 = base + C::S * C::X_BYTES, stg0 = raw0 + C::RS * C::RAW_BYTES, tab0 = stg0 + C::STG, bar = tab0 + C::TABLE * 16;
  int4* table = reinterpret_cast<int4*>(gen + (tab0 - base));
  // A stage is full when its tokens have landed and both CTAs' operands are written; one barrier for both, since a wait costs the issuing thread some 125 cycles even when it is
  // over, and a commit 90.
  const uint32_t full = bar, empty = full + 8 * C::S, raw_full = empty + 8 * C::S, raw_empty = raw_full + 8 * C::RS, acc_full = raw_empty + 8 * C::RS, acc_empty = acc_full + 16,
                 tail = acc_empty + 16;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + (tail - base));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + (tail + 4 - base));
  volatile int* last_flag = reinterpret_cast<volatile int*>(gen + (tail + 8 - base));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int first = (int)blockIdx.x / 2, step = (int)gridDim.x / 2;

  if (!GROUPED) grid_dep_release();
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::S; ++i) { mbar_init(full + 8 * i, 9); mbar_init(empty + 8 * i, 1); }
    for (int i = 0; i < C::RS; ++i) { mbar_init(raw_full + 8 * i, 1); mbar_init(raw_empty + 8 * i, 4); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, 2 * C::EW); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // both CTAs' barriers exist before anything is signalled across
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int total = p.total, known = 0;
  if constexpr (GROUPED) {
    if (!p.early) grid_dep_wait();                         // early: the tile list was there when the kernel in front let this one begin
    total = __ldcg(p.tiles) * p.n_strips;
    const int mine = first < total ? (total - first + step - 1) / step : 0;
    known = min(mine, C::TABLE);
    // looked up once, all at a time: two loads that follow each other are 1500 cycles of every role at every tile
    if (threadIdx.x < known) {
      const Tile t = tile_at<NT, GROUPED, GATED>(p, first + threadIdx.x * step, table, 0, 0);
      table[threadIdx.x] = make_int4(t.tok0, t.rows, t.e, t.n0 / (GATED ? 128 : 256));
    }
    __syncthreads();
  }

  if (warp == 0) {
    // ---- raw codes ----
    if (elect_one()) {
      tma_prefetch_desc(&tm_w);
      if (!GROUPED && !p.early) grid_dep_wait();
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      for (int id = first, i = 0; ok && id < total; id += step, ++i) {
        const Tile t = tile_at<NT, GROUPED, GATED>(p, id, table, i, known);
        const int w = t.w0 + (int)rank * (GATED ? 64 : 128);
        for (int j = 0; j < t.n; ++j) {
          const int ks = t.stage(j);
          ok = mbar_wait(raw_empty + 8 * s, par, abort_flag, p.status, ST_RAWEMPTY);
          if (!ok) break;
          mbar_expect_tx(raw_full + 8 * s, C::RAW_BYTES);
          const uint32_t dst = raw0 + s * C::RAW_BYTES;
          tma_load_2d(dst, &tm_w, ks * 64, w, raw_full + 8 * s);
          if constexpr (GATED) tma_load_2d(dst + C::RAW_BYTES / 2, &tm_w, ks * 64, w + p.N, raw_full + 8 * s);
          ++issued;
          if (++s == C::RS) { s = 0; par ^= 1u; }
        }
      }
      if (!ok) drain_issued(raw_full, C::RS, issued);
    }
  } else if (warp == 2) {
    // ---- tokens ----
    if (elect_one()) {
      tma_prefetch_desc(&tm_x);
      grid_dep_wait();
      if (GROUPED) grid_dep_release();                     // the next one may read the tile list at once, and weights
      int s = 0, issued = 0;
      uint32_t par = 1u;
      bool ok = true;
      for (int id = first, q = 0; ok && id < total; id += step, ++q) {
        const Tile t = tile_at<NT, GROUPED, GATED>(p, id, table, q, known);
        for (int j = 0; j < t.n; ++j) {
          const int ks = t.stage(j);
          ok = mbar_wait(empty + 8 * s, par, abort_flag, p.status, ST_XEMPTY);
          if (!ok) break;
          const uint32_t dst = base + s * C::X_BYTES;
          if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * C::X_BYTES);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            tma_load_2d_pair(dst + i * C::TOK * 128, &tm_x, ks * 128 + i * 64, t.tok0 + (int)rank * C::TOK, map_to_cta(full + 8 * s, 0));
          }
          ++issued;
          if (++s == C::S) { s = 0; par ^= 1u; }
        }
      }
      if (!ok && rank == 0) drain_issued(full, C::S, issued);
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = instr_desc(BF16 ? 1u : 0u, BF16 ? 1u : 0u, 256u, (uint32_t)NT);
      int s = 0, it = 0;
      uint32_t par = 0u;
      bool ok = true;
      for (int id = first; ok && id < total; id += step, ++it) {
        const Tile t = tile_at<NT, GROUPED, GATED>(p, id, table, it, known);
        const int b = it % C::NBUF;
        if (it >= C::NBUF) ok = mbar_wait(acc_empty + 8 * b, (it / C::NBUF - 1) & 1, abort_flag, p.status, ST_ACCEMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + b * C::COLS;
        for (int ks = 0; ks < t.n; ++ks) {
          ok = mbar_wait(full + 8 * s, par, abort_flag, p.status, ST_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = tmem + C::A_COL0 + s * 64;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint64_t db = smem_desc_sw128(base + s * C::X_BYTES + i * C::TOK * 128);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma_f16_ts_pair(d, a + 32 * i + 8 * j, db + 2 * j, idesc, ks > 0 || i > 0 || j > 0);
            }
          }
          tc_commit_pair(empty + 8 * s, 3);
          if (++s == C::S) { s = 0; par ^= 1u; }
        }
        if (!ok) break;
        tc_commit_pair(acc_full + 8 * b, 3);
      }
    }
  } else if (warp >= C::FIRST_DEQ) {
    // ---- transform: group g of four warps has every DG-th stage, a thread a row ----
    const int grp = (warp - C::FIRST_DEQ) >> 2, quad = warp & 3;
    const int raw_row = GATED ? (lane < 16 ? 16 * quad + lane : 48 + 16 * quad + lane) : 32 * quad + lane;      // 64 + 16 quad + lane - 16
    const uint32_t row_at = raw_row * 64, f = (raw_row >> 1) & 3;      // 64-byte swizzle of the raw box
    constexpr int GS = 128 / G;
    if (!GROUPED && !p.early) grid_dep_wait();
    // This group's stages one after the other, whatever tile they are of.  All tiles of a CTA have the same number of stages: where k is cut into pieces, it has one tile.
    bool ok = true;
    uint32_t sc[2][GS], zc[2][GS];                         // of this group's next two stages
    struct Ahead { int id, q, j; Tile t; int64_t at; } ahead;      // of the stage whose scales are fetched next
    auto enter = [&]() {
      if (ahead.id >= total) return;
      const Tile t = ahead.t = tile_at<NT, GROUPED, GATED>(p, ahead.id, table, ahead.q, known);
      // this thread's row among the scales' rows; beyond the last it repeats it, and nobody looks at the sums
      int row;
      if constexpr (GATED) { const int h = min(t.n0 + (int)rank * 64 + 16 * quad + (lane & 15), p.N - 1); row = lane < 16 ? h : p.N + h; }
      else row = min(t.n0 + (int)rank * 128 + 32 * quad + lane, p.N - 1);
      ahead.at = (int64_t)t.e * p.s_expert + row;
    };
    ahead.id = first;
    ahead.q = 0;
    ahead.j = grp;
    enter();
    const int n = first < total ? ahead.t.n : 1;
    auto pass = [&]() {                                    // tiles that end before this group's next stage
      while (ahead.j >= n && ahead.id < total) {
        ahead.j -= n;
        ahead.id += step;
        ++ahead.q;
        enter();
      }
    };
    pass();
    auto fetch = [&](uint32_t (&s)[GS], uint32_t (&z)[GS]) {
      if (ahead.id >= total) return;
#pragma unroll
      for (int i = 0; i < GS; ++i) {
        const int64_t at = ahead.at + (int64_t)min(ahead.t.stage(ahead.j) * GS + i, p.groups - 1) * p.s_rows;
        s[i] = ld_u16(p.s + at);
        z[i] = p.z ? ld_u8(p.z + at) : 8u;
      }
      ahead.j += C::DG;
      pass();
    };
    fetch(sc[0], zc[0]);
    fetch(sc[1], zc[1]);
    const int tiles = first < total ? (total - first + step - 1) / step : 0, end = tiles * n;
    {
      for (int now = grp; now < end; now += C::DG) {
        const int rs = now % C::RS, as = now % C::S;
        uint32_t s2[GS], z2[GS], zh[GS], more[GS];
        bool has_more = false;
#pragma unroll
        for (int i = 0; i < GS; ++i) {
          s2[i] = sc[0][i] * 0x00010001u;
          const uint32_t z = zc[0][i];
          sc[0][i] = sc[1][i];
          zc[0][i] = zc[1][i];
          if (BF16) {
            const uint32_t low = min(z, 127u);
            z2[i] = 0x43004300u | low * 0x00010001u;
            more[i] = __float_as_uint((float)(z - low)) >> 16;
            more[i] |= more[i] << 16;
            has_more = has_more || z > 127u;
            zh[i] = 0;
          } else {
            z2[i] = 0x64006400u | z * 0x00010001u;
            zh[i] = __half_as_ushort(__float2half_rn(-64.f - (float)z)) * 0x00010001u;
            more[i] = 0;
          }
        }
        has_more = BF16 && __any_sync(0xffffffffu, has_more);
        fetch(sc[1], zc[1]);
        ok = mbar_wait_warp(raw_full + 8 * rs, (now / C::RS) & 1, abort_flag, p.status, ST_RAWFULL);
        if (!ok) break;
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = lds128(raw0 + rs * C::RAW_BYTES + row_at + ((i ^ f) << 4));
        if (now >= C::S) ok = mbar_wait_warp(empty + 8 * as, (now / C::S - 1) & 1, abort_flag, p.status, ST_AEMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a = tmem + C::A_COL0 + as * 64 + ((uint32_t)(quad * 32) << 16);
        auto convert = [&](auto with_more) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t o[32];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 r = raw[2 * h + i];
              const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const int of = (h * 64 + i * 32 + v * 8) / G;
                decode<BF16, PERM, decltype(with_more)::value>(w[v], s2[of], z2[of], zh[of], more[of], p.mask, p.magic, o + 16 * i + 4 * v);
              }
            }
            tmem_st32(a + 32 * h, o);
          }
        };
        if (has_more) convert(std::true_type{});
        else convert(std::false_type{});
        mbar_arrive_read(raw_empty + 8 * rs);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(full + 8 * as, 0));
        __syncwarp();
      }
    }
  } else if (warp >= C::FIRST_EPI) {
    // ---- epilogue: lane quadrant = warp & 3 (weight rows); tokens shared by the warps of a quadrant ----
    const int quad = warp & 3, half = (warp - C::FIRST_EPI) >> 2;
    constexpr int HALVES = C::EW / 4, MINE = NT / HALVES;  // tokens of a warp
    constexpr int CH = MINE < 32 ? 16 : 32;
    const uint32_t stg = stg0 + (warp - C::FIRST_EPI) * 2048;
    grid_dep_wait();
    int it = 0;
    bool ok = true;
    for (int id = first; id < total; id += step, ++it) {
      const Tile t = tile_at<NT, GROUPED, GATED>(p, id, table, it, known);
      const int b = it % C::NBUF;
      ok = ok && mbar_wait_warp(acc_full + 8 * b, (it / C::NBUF) & 1, abort_flag, p.status, ST_ACCFULL);
      if (!ok) {
        if (!GROUPED && p.pieces > 1) { asm volatile("bar.sync 1, %0;" ::"n"(32 * C::EW) : "memory"); asm volatile("bar.sync 1, %0;" ::"n"(32 * C::EW) : "memory"); }
        continue;
      }
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + b * C::COLS;
      const int c0 = t.n0 + (int)rank * (GATED ? 64 : 128) + quad * (GATED ? 16 : 32);      // this warp's first output column
      const int cols = p.N - c0;
      const int row = c0 + lane;
      float bias = 0.f;
      if (!GROUPED && p.bias && row < p.N) bias = half_f<BF16>(p.bias[row]);
      auto free_acc = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(acc_empty + 8 * b, 0));
        __syncwarp();
      };
      if (!GROUPED && p.pieces > 1) {
        // partial sums [strip][rank][piece][token][128 rows]; the last to deliver adds them up
        const int64_t at = 2 * t.strip + (int)rank;
        float* mine = p.partials + (at * p.pieces + t.piece) * NT * 128 + quad * 32 + lane;
        if (threadIdx.x == 32 * C::FIRST_EPI) arrivals_open(p.arrivals + at, p.tag, p.epoch);
        for (int c = half * MINE; c < (half + 1) * MINE && c < t.rows; c += 16) {
          uint32_t r[16];
          tmem_ld16(acc + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < t.rows) __stcg(mine + (int64_t)(c + i) * 128, __uint_as_float(r[i]));
        }
        free_acc();
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::EW) : "memory");
        if (threadIdx.x == 32 * C::FIRST_EPI) {
          *last_flag = arrivals_last(p.arrivals + at, p.pieces - 1);
          __threadfence();
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::EW) : "memory");
        if (*last_flag) {
          const float* from = p.partials + at * p.pieces * NT * 128 + quad * 32 + lane;
          for (int c = half * MINE; c < (half + 1) * MINE && c < t.rows; c += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = bias;
#pragma unroll 2
            for (int q = 0; q < p.pieces; ++q) {           // tokens beyond the last are read and not looked at
              float w[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = __ldcg(from + ((int64_t)q * NT + c + i) * 128);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] += w[i];
            }
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = pack2<BF16>(v[2 * i], v[2 * i + 1]);
            if (cols > 0) store16(stg, o, p.out + (int64_t)(t.tok0 + c) * p.ldo + c0, p.ldo, t.rows - c, min(cols, 32), p.vec_out);
          }
        }
        continue;
      }
      if constexpr (GATED) {
        const bool upper = lane >= 16;
        for (int c = half * MINE; c < (half + 1) * MINE && c < t.rows; c += 32) {
          uint32_t r[32];
          tmem_ld32(acc + c, r);
          tmem_ld_wait();
          uint16_t h[16];                                  // of token 2 i (lower lanes) or 2 i + 1
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float a = __uint_as_float(r[2 * i]), d = __uint_as_float(r[2 * i + 1]);
            const float got = __shfl_xor_sync(0xffffffffu, upper ? a : d, 16);
            const float gate = upper ? got : a, up = upper ? d : got;
            h[i] = (uint16_t)pack2<BF16>(gate / (1.f + expf(-gate)) * up, 0.f);
          }
          // through shared memory: [32 tokens][16 columns], the columns permuted in eights
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) sts16(stg + (2 * i + upper) * 32 + g4_position(lane & 15) * 2, h[i]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int tk = i * 16 + (lane >> 1), cc = (lane & 1) * 8;
            const uint4 v = lds128(stg + tk * 32 + cc * 2);
            if (c + tk < t.rows && cc < cols) *reinterpret_cast<uint4*>(p.out + (int64_t)(t.tok0 + c + tk) * p.ldo + c0 + cc) = v;
          }
        }
        free_acc();
      } else {
        // all of a warp's values first where the accumulator is the only one, so that the next tile can begin
        constexpr int KEEP = C::NBUF == 1 ? MINE : CH;
        for (int c1 = half * MINE; c1 < (half + 1) * MINE && c1 < t.rows; c1 += KEEP) {
          uint32_t o[KEEP / 2];
#pragma unroll
          for (int c = 0; c < KEEP; c += 16) {
            uint32_t r[16];
            tmem_ld16(acc + c1 + c, r);
            float w = 1.f;
            if (GROUPED) w = c1 + c + (lane & 15) < t.rows ? __ldcg(p.out_w + t.tok0 + c1 + c + (lane & 15)) : 0.f;
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float a = __uint_as_float(r[2 * i]) + bias, d = __uint_as_float(r[2 * i + 1]) + bias;
              if (GROUPED) { a *= __shfl_sync(0xffffffffu, w, 2 * i); d *= __shfl_sync(0xffffffffu, w, 2 * i + 1); }
              o[c / 2 + i] = pack2<BF16>(a, d);
            }
          }
          if (C::NBUF == 1) free_acc();
          if (cols > 0) {
#pragma unroll
            for (int c = 0; c < KEEP; c += 16) {
              if (c1 + c < t.rows) {
                uint32_t part[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) part[i] = o[c / 2 + i];
                store16(stg, part, p.out + (int64_t)(t.tok0 + c1 + c) * p.ldo + c0, p.ldo, t.rows - c1 - c, min(cols, 32), p.vec_out);
              }
            }
          }
        }
        if (C::NBUF > 1 || half * MINE >= t.rows) free_acc();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // nobody leaves while the partner may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Rows of x to contiguous rows: as they are, where x's do not start on 16 bytes as TMA wants them, or with the values of every eight permuted.
template <bool PERM> __global__ void __launch_bounds__(256) g4_rows_kernel(const uint16_t* x, int64_t ldx, int vec, uint4* to, int per) {
  grid_dep_release();
  grid_dep_wait();
  for (int i = threadIdx.x; i < per; i += 256) {
    const uint16_t* p = x + blockIdx.x * ldx + 8 * i;
    uint32_t w[4];
    if (vec) {
      const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (uint32_t)__ldcg(p + 2 * j) | (uint32_t)__ldcg(p + 2 * j + 1) << 16;
    }
    to[(int64_t)blockIdx.x * per + i] = PERM ? make_uint4(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632), __byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632))
                                             : make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- host ----
namespace ug4 {
constexpr uint32_t MASK = 0x000F000Fu, MAGIC_BF16 = 0x43004300u, MAGIC_F16 = 0x64006400u;      // 128 and 1024, whose lowest bits a code takes

template <bool BF16, int G, int NT, bool GROUPED, bool GATED>
static int launch(const CUtensorMap& tx, const CUtensorMap& tw, const Params& p, int grid, cudaStream_t st) {
  using C = Cfg<NT>;
  auto kern = umma_g4_kernel<BF16, G, NT, GROUPED, GATED>;
  static thread_local bool configured[16] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return B2Q_ERR_CUDA;
    if (dev < 16) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(C::THREADS); cfg.dynamicSmemBytes = C::SMEM; cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  at[n].id = cudaLaunchAttributeClusterDimension;
  at[n].val.clusterDim.x = 2; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
  ++n;
  if (tls().overlap_mode > 0) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at; cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kern, tx, tw, p);               // launch_status() reports
  note_launch("umma_g4");
  return launch_status();
}
template <int NT, bool GROUPED, bool GATED>
static int by_type(bool bf16, int G, const CUtensorMap& tx, const CUtensorMap& tw, const Params& p, int grid, cudaStream_t st) {
  if (bf16) {
    if (G == 128) return launch<true, 128, NT, GROUPED, GATED>(tx, tw, p, grid, st);
    if (G == 64) return launch<true, 64, NT, GROUPED, GATED>(tx, tw, p, grid, st);
    return launch<true, 32, NT, GROUPED, GATED>(tx, tw, p, grid, st);
  }
  if (G == 128) return launch<false, 128, NT, GROUPED, GATED>(tx, tw, p, grid, st);
  if (G == 64) return launch<false, 64, NT, GROUPED, GATED>(tx, tw, p, grid, st);
  return launch<false, 32, NT, GROUPED, GATED>(tx, tw, p, grid, st);
}
static size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

struct Plan { int nt, pieces, m_tiles, n_strips; };
// Heights, us in graphs, K = 5120, N = 17408: 32 tokens 19.8 in a tile of 32, 20.2 of 64; 48 tokens 32.9, 20.5 and 23.0 of 32, 64 and 128; 96 tokens 34.2, 24.0 and 33.4 of 64, 128 and 256; 128 tokens 34.5,
// 26.0, 33.9; 129 tokens 38.0 and 35.6 of 128 and 256, 256 tokens 41.4 and 37.6, 1024 142 and 127, 4001 581 and 506.  Where strips are few, 256 loses up to 512 tokens (4096 x 4096: 129 tokens
// 18.8 and 22.3, 512 21.3 and 26.5, 1024 33.8 and 31.2); the rule does not tell these apart.
// Pieces, at most eight: 24 x 512 x 14336 19.2 with four, 16.3 with eight, 18.3 with sixteen; 40 x 1024 x 8192 15.1, 15.6, 20.2; 100 x 1024 x 8192 20.4, 24.1, 34.2.  Of four stages at least: 40 x 1024 x 2048 12.7 of
// two, 10.4 of four, 9.8 of eight; 300 x 512 x 2048 27.4, 20.7, 19.1; 100 x 512 x 1024 13.4, 11.1, 6.8.
static Plan plan(int M, int N, int K) {
  Plan q{};
  q.nt = M <= 32 ? 32 : (M <= 64 ? 64 : (M <= 128 ? 128 : 256));
  q.m_tiles = (M + q.nt - 1) / q.nt;
  q.n_strips = (N + 255) / 256;
  const int64_t tiles = (int64_t)q.m_tiles * q.n_strips, pairs = sm_count() / 2;
  const int nks = (K + 127) / 128;
  q.pieces = tiles >= pairs ? 1 : (int)(pairs / tiles);
  if (q.pieces > nks / 4) q.pieces = nks / 4;
  if (q.pieces > 8) q.pieces = 8;
  if (q.pieces < 1) q.pieces = 1;
  return q;
}
static size_t partial_bytes(const Plan& q) { return align_up((size_t)q.m_tiles * q.n_strips * 2 * q.pieces * q.nt * 128 * 4, 256); }
static bool aligned_rows(const void* x, int64_t ldx) { return x && ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(2 * ldx)) & 15u) == 0; }
}  // namespace ug4

size_t umma_g4_bytes(const void* x, int64_t ldx, int M, int N, int K, int G) {
  using namespace ug4;
  const Plan q = plan(M, N, K);
  size_t n = q.nt < 256 || !aligned_rows(x, ldx) ? align_up((size_t)M * K * 2, 256) : 0;
  if (q.pieces > 1) n += partial_bytes(q) + align_up((size_t)q.m_tiles * q.n_strips * 2 * sizeof(Arrivals), 256);
  return n;
}

int umma_g4_linear(const G4LinearArgs& a, void* scratch, cudaStream_t st) {
  using namespace ug4;
  if (!tensor_map_encoder()) return B2Q_ERR_CUDA;
  const Plan q = plan(a.M, a.N, a.K);
  if ((int64_t)q.n_strips * q.m_tiles * q.pieces > INT32_MAX / 8) return B2Q_ERR_LIMIT;
  uint8_t* at = reinterpret_cast<uint8_t*>(scratch);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x);
  int64_t ldx = a.ldx;
  if (q.nt < 256 || !aligned_rows(a.x, a.ldx)) {
    launch_overlapped(q.nt < 256 ? g4_rows_kernel<true> : g4_rows_kernel<false>, dim3(a.M), dim3(256), 0, st, tls().overlap_mode > 0, x, a.ldx, (int)aligned_rows(a.x, a.ldx),
                      reinterpret_cast<uint4*>(at), a.K / 8);
    note_launch("g4_rows");
    x = reinterpret_cast<const uint16_t*>(at);
    at += align_up((size_t)a.M * a.K * 2, 256);
    ldx = a.K;
  }
  Params p{};
  p.s = reinterpret_cast<const uint16_t*>(a.scale); p.z = a.zero; p.s_rows = a.N;
  p.bias = reinterpret_cast<const uint16_t*>(a.bias); p.out = reinterpret_cast<uint16_t*>(a.out); p.ldo = a.ldo; p.vec_out = aligned16(a.out) && a.ldo % 8 == 0;
  p.M = a.M; p.N = a.N; p.K = a.K; p.groups = a.K / a.G; p.nks = (a.K + 127) / 128;
  // sixteen tiles of tokens take turns at a strip: 2048 x 8192 x 8192 191 us with 4 or 16, 197 with 8 or 32, 244 with 64 (which is none); 4001 x 17408 x 5120 482 to 508 with 4 to 32, 530 with 64
  p.n_strips = q.n_strips; p.m_tiles = q.m_tiles; p.m_group = q.m_tiles < 16 ? q.m_tiles : 16; p.pieces = q.pieces;
  p.total = q.n_strips * q.m_tiles * q.pieces;
  if (q.pieces > 1) {
    p.partials = reinterpret_cast<float*>(at);
    p.arrivals = reinterpret_cast<Arrivals*>(at + partial_bytes(q));
    p.tag = arrivals_tag();
    p.epoch = arrivals_epoch();
    if (!p.epoch) return B2Q_ERR_CUDA;
  }
  p.early = tls().overlap_mode == 2;
  p.mask = MASK; p.magic = a.bf16 ? MAGIC_BF16 : MAGIC_F16;
  p.status = umma_status_ptr();
  if (!p.status) return B2Q_ERR_CUDA;
  CUtensorMap tx, tw;
  int rc = make_tmap_2d(&tx, a.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, a.M, a.K, (uint64_t)ldx * 2, q.nt / 2, 64,
                        CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.N, a.K / 2, (uint64_t)a.K / 2, 128, 64, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc) return rc;
  const int pairs = sm_count() / 2, grid = 2 * (p.total < pairs ? p.total : pairs);
  if (q.nt == 32) return by_type<32, false, false>(a.bf16, a.G, tx, tw, p, grid, st);
  if (q.nt == 64) return by_type<64, false, false>(a.bf16, a.G, tx, tw, p, grid, st);
  if (q.nt == 128) return by_type<128, false, false>(a.bf16, a.G, tx, tw, p, grid, st);
  return by_type<256, false, false>(a.bf16, a.G, tx, tw, p, grid, st);
}

// Token height of the tiles, from the mean rows per expert (in brackets; us in graphs of the layer in tiles of 32, 64, 128): 64 experts of 2048 x 1408, top-8, groups of 64 [16] 109, 110, 133, [24] 113, 111, 135,
// [32] 149, 113, 137, [48] 191, 118, 141, [64] 233, 157, 143, [96] 315, 201, 151, [128] 399, 244, 203; 128 of 2048 x 768 [24] 117, 119, 143, [32] 151, 122, 146, [48] 203, 133, 153, [64] 246, 172, 158; 8 of
// 4096 x 4096, top-2 [24] 87, 90, 99, [32] 113, 90, 102, [48] 138, 93, 104, [64] 174, 125, 103.
int g4_grouped_tile(int64_t rows, int E) {
  const int64_t avg = (rows + E - 1) / E;
  return avg <= 24 ? 32 : (avg <= 48 ? 64 : 128);
}

int umma_g4_grouped(const G4GroupedArgs& a, cudaStream_t st) {
  using namespace ug4;
  if (!tensor_map_encoder()) return B2Q_ERR_CUDA;
  Params p{};
  p.s = reinterpret_cast<const uint16_t*>(a.scale); p.z = a.zero;
  p.s_rows = a.gated ? 2 * a.N : a.N; p.groups = a.K / a.G; p.s_expert = (int64_t)p.groups * p.s_rows;
  p.out_w = a.out_w; p.out = reinterpret_cast<uint16_t*>(a.out); p.ldo = a.N; p.vec_out = aligned16(a.out) && a.N % 8 == 0;
  p.M = a.rows; p.N = a.N; p.K = a.K; p.nks = (a.K + 127) / 128; p.pieces = 1;
  const int width = a.gated ? 128 : 256;
  p.n_strips = (a.N + width - 1) / width;
  p.tiles = a.tiles; p.offsets = a.offsets;
  p.mask = MASK; p.magic = a.bf16 ? MAGIC_BF16 : MAGIC_F16;
  p.status = umma_status_ptr();
  if (!p.status) return B2Q_ERR_CUDA;
  p.early = tls().overlap_mode > 0;
  const int64_t w_rows = (int64_t)a.E * p.s_rows;
  CUtensorMap tx, tw;
  int rc = make_tmap_2d(&tx, a.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.x, a.rows, a.K, (uint64_t)a.K * 2, a.tile / 2, 64,
                        CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, w_rows, a.K / 2, (uint64_t)a.K / 2, a.gated ? 64 : 128, 64, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc) return rc;
  const int pairs = sm_count() / 2, most = a.tile_cap * p.n_strips, grid = 2 * (most < pairs ? most : pairs);
  if (a.tile == 32) return a.gated ? by_type<32, true, true>(a.bf16, a.G, tx, tw, p, grid, st) : by_type<32, true, false>(a.bf16, a.G, tx, tw, p, grid, st);
  if (a.tile == 64) return a.gated ? by_type<64, true, true>(a.bf16, a.G, tx, tw, p, grid, st) : by_type<64, true, false>(a.bf16, a.G, tx, tw, p, grid, st);
  return a.gated ? by_type<128, true, true>(a.bf16, a.G, tx, tw, p, grid, st) : by_type<128, true, false>(a.bf16, a.G, tx, tw, p, grid, st);
}

}  // namespace b2q
