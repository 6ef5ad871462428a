// The inner part of the streaming kernels for 4-bit group-quantised weights of a few tokens: weights by cp.async through a ring of each warp's own to
// mma.sync m16n8k16.
//
// Mathematics.  out = sum_g s_g (sum_{k in g} x_k q_k - z_g X_g), X_g the sum of x over the group: the products of a group are added up by the MMA with q as it is, scale and
// zero point enter in fp32, so no weight is ever rounded.  A code is put into the lowest bits of an fp16, where it is the subnormal q 2^-24 (MMAs take
// those exactly), or four bits higher, as 16 q 2^-24: eight codes take five operations and no subtraction.  The activations that meet the latter are
// divided by 16 beforehand.  That loses nothing because every token's row is first scaled by a power of two that brings its largest value into
// [2^14, 2^15): bf16 and fp16 values down to 2^-24 of that stay exact, and smaller ones are off by no more than 2^-35 of it.
//
// What bounds such a kernel before memory does is a warp's chain of instructions.  Of the 7.3 cycles between two of them (1 x 28672 x 8192, four warps to a scheduler) 2.1 are fixed latencies, 1.0 a wait for
// its turn, 0.8 for the ALU pipe, 0.8 for shared memory; 55 % of the issue slots and 48 % of the ALU pipe are used, and no unit is full.  So a warp takes 32 rows at a time, for which the activations are read half
// as often (1 x 28672 x 8192: 29.0 us, 36 with 16 rows), and two steps at a time.  Codes by cp.async and not straight into registers, where a wait for one load was a wait for
// younger ones too (43 us).  An 8-bit mma.sync of e4m3, for which the bytes q need no more than masks, took 43 us where this took 36 at the time: half
// again as many instructions.
//
// Layout.  Rows of the weight are the rows of the MMA, tokens its columns.  With the k of a word of eight codes permuted alike on both sides, a word of row g and one of
// row g + 8 are the A operands of two MMAs.  Lane t of a quad has 8 VEC consecutive k, so that the quad's words of one index are of one group:
// VEC = G / 32.
#pragma once
#include "g4.cuh"

namespace b2q {
namespace g4s {

constexpr int STEP = 128;                                  // k of a step

// Tokens as the products read them, step by step: [M tokens][16 eights of values], then the group sums [STEP / G][8 TT] in units of 2^-24.  The sixteen bytes of an eight
// lie permuted so that the eight lanes of a quarter warp, two tokens' four eights, meet no bank twice.
__host__ __device__ constexpr int step_bytes(int M, int G, int tt) { return M * STEP * 2 + STEP / G * 8 * tt * 4; }
__host__ __device__ __forceinline__ constexpr int eight_at(int c, int m) { return (c ^ ((c >> 2) & 3) ^ ((m & 1) << 2)) * 16; }

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Sixteen bytes to shared memory; of which n are read, the others zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from, uint32_t n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Into registers of 32 bits as they are: a conversion behind the load would wait for it.
__device__ __forceinline__ uint32_t ld_scale(const uint16_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_zero(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
template <int W> __device__ __forceinline__ void lds_words(uint32_t a, uint32_t* v) {
  if constexpr (W == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
  else if constexpr (W == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a) : "memory");
  else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(a) : "memory");
}
__device__ __forceinline__ float2 lds64f(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
// D (+)= A B, 16 x 8 x 16, fp16 in, fp32 sums
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <bool BF16> __device__ __forceinline__ float half_f(uint32_t raw) {      // of the low 16 bits
  return BF16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half((unsigned short)raw));
}
template <bool BF16> __device__ __forceinline__ uint16_t to_half(float v) { return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v)); }

// One matrix: codes [N, K / 2], scales and zero points [K / G, N].
struct Matrix { const uint8_t* w; const uint16_t* s; const uint8_t* z; int64_t half; int64_t n; };      // half: K / 2, n: rows of the scales' pitch

// A warp takes its tiles of 32 rows two steps at a time.  Codes go by cp.async, a row's 64 bytes of a step by four lanes, into one of two slots of the warp's own in shared
// memory, the next two steps' while these are multiplied; the 16-byte pieces of a slot are permuted so that the words are read without bank conflicts,
// whatever the group.
constexpr int ROWS = 32, PART_BYTES = ROWS * STEP / 2, SLOT = 2 * PART_BYTES, WARP_BYTES = 2 * SLOT;
__device__ __forceinline__ int slot_piece(int row, int piece) {      // byte offset in a slot; row < 8
  const int f = (row >> 1 & 1) << 1 | (row >> 2 & 1);
  return row * 64 + ((piece ^ f) << 4);
}

template <int VEC> struct Lane {                           // what stays the same throughout
  uint32_t copy;                                           // where this lane's piece of its first row goes in a slot; the next rows 512 further each
  uint32_t word[4 / VEC];                                  // from where the words of the first row come, group by group
  uint32_t x[4];                                           // where the words find their activations in a token's 256 bytes of a step
  __device__ __forceinline__ Lane() {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    copy = slot_piece(g, t);
#pragma unroll
    for (int j = 0; j < 4 / VEC; ++j) {
      const int first = 4 * VEC * j + VEC * t;             // word of the step's sixteen
      word[j] = slot_piece(g, first >> 2) + (first & 3) * 4;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = eight_at(4 * VEC * (i / VEC) + VEC * t + i % VEC, g);
  }
};

// Scale in the low half as it is, zero point in the upper half as bf16, which holds every byte.
__device__ __forceinline__ uint32_t pack_scale(uint32_t s, uint32_t z) {
  return (__float_as_uint(__uint_as_float(0x4B000000u | z) - 8388608.f) & 0xFFFF0000u) | s;
}

// sum += a step's share, in units of 2^-24.  slot: the codes; xs: shared address of this lane's token (of each eight of tokens) at the step; xg: of the group sums at the
// step's first group and this lane's columns; packed: scales, of which the step's first group is in lane t0 of a quad; halves: sixteens of rows there are.
template <int VEC, int TT, bool BF16>
__device__ __forceinline__ void multiply(float (&sum)[2][TT][4], uint32_t slot, const Lane<VEC>& ln, const uint32_t (&xs)[TT], uint32_t xg, const uint32_t (&packed)[4], int t0,
                                         int halves) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 4 / VEC; ++j) {
    uint32_t x[VEC][TT][4];
#pragma unroll
    for (int v = 0; v < VEC; ++v)
#pragma unroll
      for (int n = 0; n < TT; ++n) lds_words<4>(xs[n] + ln.x[VEC * j + v], x[v][n]);
    float2 X[TT];
#pragma unroll
    for (int n = 0; n < TT; ++n) X[n] = lds64f(xg + (j * 8 * TT + 8 * n) * 4);
    const int from = (lane & ~3) + t0 + j;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && halves == 1) break;
      uint32_t wa[VEC], wb[VEC];
      lds_words<VEC>(slot + ln.word[j] + 1024 * h, wa);
      lds_words<VEC>(slot + ln.word[j] + 1024 * h + 512, wb);
      const uint32_t qa = __shfl_sync(0xffffffffu, packed[2 * h], from), qb = __shfl_sync(0xffffffffu, packed[2 * h + 1], from);
      float d[TT][4];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const uint32_t a = wa[v], b = wb[v], a8 = a >> 8, b8 = b >> 8;
        const uint32_t l0 = a & 0x000F000Fu, l1 = b & 0x000F000Fu, l2 = a8 & 0x000F000Fu, l3 = b8 & 0x000F000Fu;
        const uint32_t h0 = a & 0x00F000F0u, h1 = b & 0x00F000F0u, h2 = a8 & 0x00F000F0u, h3 = b8 & 0x00F000F0u;
#pragma unroll
        for (int n = 0; n < TT; ++n) {
          if (v == 0) mma_first(d[n], l0, l1, l2, l3, x[v][n][0], x[v][n][1]);
          else mma(d[n], l0, l1, l2, l3, x[v][n][0], x[v][n][1]);
          mma(d[n], h0, h1, h2, h3, x[v][n][2], x[v][n][3]);
        }
      }
      const float sa = half_f<BF16>(qa), sb = half_f<BF16>(qb), za = __uint_as_float(qa & 0xFFFF0000u), zb = __uint_as_float(qb & 0xFFFF0000u);
#pragma unroll
      for (int n = 0; n < TT; ++n) {
        sum[h][n][0] = fmaf(sa, fmaf(-za, X[n].x, d[n][0]), sum[h][n][0]);
        sum[h][n][1] = fmaf(sa, fmaf(-za, X[n].y, d[n][1]), sum[h][n][1]);
        sum[h][n][2] = fmaf(sb, fmaf(-zb, X[n].x, d[n][2]), sum[h][n][2]);
        sum[h][n][3] = fmaf(sb, fmaf(-zb, X[n].y, d[n][3]), sum[h][n][3]);
      }
    }
  }
}

// A tile's sums to [32 rows][8 TT], and zero.
template <int TT> __device__ __forceinline__ void flush(float (&sum)[2][TT][4], float* to) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int n = 0; n < TT; ++n) {
      float* at = to + (16 * h + g) * 8 * TT + 8 * n + 2 * t;
      *reinterpret_cast<float2*>(at) = make_float2(sum[h][n][0], sum[h][n][1]);
      *reinterpret_cast<float2*>(at + 64 * TT) = make_float2(sum[h][n][2], sum[h][n][3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[h][n][i] = 0.f;
    }
}

// A warp's run of units (a tile's step each): [u0, u1) of tiles with `steps` steps, the matrix's steps s0 on.  Tiles::rows(tile, row, off, base) gives the lane's four rows (of the
// codes), their scales' offsets from base, and how many sixteens of rows there are; Tiles::columns(tile, xs, xg) where its tokens and their group sums begin.
template <int VEC, int TT, bool BF16, bool PART, typename Tiles> struct Stream {      // PART: K is no multiple of 128
  static constexpr int G = 32 * VEC, GS = STEP / G;        // groups in a step
  static constexpr int SETS = GS == 4 ? 2 : 1;             // fours of groups in two steps
  const Matrix& m;
  Tiles& tiles;
  const Lane<VEC> ln;
  int K, steps, s0, u, u1;                                 // u: the next unit to load
  uint32_t ring;
  // of the two steps that are loaded next: where this lane copies from, and its scales
  const uint8_t* p[4];
  const uint16_t* scales; const uint8_t* zeros; uint32_t off[4];
  int tile, s, n, halves;
  uint32_t raw_s[SETS][4], raw_z[SETS][4];

  __device__ __forceinline__ Stream(const Matrix& m_, Tiles& tiles_, int K_, int steps_, int s0_, int u0_, int u1_, uint32_t ring_)
      : m(m_), tiles(tiles_), K(K_), steps(steps_), s0(s0_), u(u0_), u1(u1_), ring(ring_) {
    tile = steps ? u / steps : 0;
    s = u - tile * steps;
    n = 0;
    if (u < u1) enter();
  }
  __device__ __forceinline__ void enter() {                // the tile's rows, from step s on
    const int t = threadIdx.x & 3;
    int64_t row[4], base;
    halves = tiles.rows(tile, row, off, base);
    scales = m.s + base;
    zeros = m.z + base;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = m.w + row[i] * m.half + (s0 + s) * (STEP / 2) + 16 * t;
    n = min(2, min(steps - s, u1 - u));
  }
  // Loads two steps, or what is left of the tile, into the slot.  Rows beyond the last repeat it, and nobody looks at their sums; codes beyond K are zeros, and groups beyond K repeat
  // the last: their activations are zero.
  __device__ __forceinline__ void load(uint32_t slot) {
    if (u < u1) {
      const int t = threadIdx.x & 3, k0 = (s0 + s) * STEP;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && n == 1) break;
        const uint32_t to = slot + ln.copy + j * PART_BYTES, bytes = !PART || k0 + j * STEP + 32 * t < K ? 16 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i == 2 && halves == 1) break;
          if (PART) copy16(to + 512 * i, p[i] + j * (STEP / 2), bytes);
          else copy16(to + 512 * i, p[i] + j * (STEP / 2));
        }
      }
      const int g0 = (s0 + s) * GS, last = min(K / G - 1 - g0, n * GS - 1);
#pragma unroll
      for (int q = 0; q < SETS; ++q) {
        const uint32_t at = (uint32_t)(g0 + min(4 * q + t, last)) * (uint32_t)m.n;      // within a matrix's scales, below 2^31
#pragma unroll
        for (int i = 0; i < 4; ++i) raw_s[q][i] = ld_scale(scales + (at + off[i]));
#pragma unroll
        for (int i = 0; i < 4; ++i) raw_z[q][i] = 8;
        if (m.z) {
#pragma unroll
          for (int i = 0; i < 4; ++i) raw_z[q][i] = ld_zero(zeros + (at + off[i]));
        }
      }
    }
    copy_commit();
  }
  __device__ __forceinline__ void advance() {              // behind load()
    u += n;
    s += n;
    if (s == steps) {
      s = 0;
      ++tile;
      if (u < u1) enter();
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] += STEP;
      n = min(2, min(steps - s, u1 - u));
    }
  }
  // Everything, behind load() of the first slot and the staging of the tokens.  A tile's sums go to slots[tile + warp].
  __device__ __forceinline__ void run(uint32_t x_stride, uint32_t xg_stride, float* slots, int warp) {
    float sum[2][TT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[h][i][j] = 0.f;
    uint32_t at[TT], xg = 0, slot = ring;
    bool fresh = true;
    while (u < u1) {
      const int now_tile = tile, now_s = s, now_n = n, now_halves = halves;
      uint32_t packed[SETS][4];
#pragma unroll
      for (int q = 0; q < SETS; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) packed[q][i] = pack_scale(raw_s[q][i], raw_z[q][i]);
      advance();
      load(2 * ring + SLOT - slot);
      if (fresh) {
        tiles.columns(now_tile, at, xg);
#pragma unroll
        for (int i = 0; i < TT; ++i) at[i] += now_s * x_stride;
        xg += now_s * xg_stride;
        fresh = false;
      }
      copy_wait<1>();
      __syncwarp();                                        // other lanes' pieces are there
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && now_n == 1) break;
        multiply<VEC, TT, BF16>(sum, slot + j * PART_BYTES, ln, at, xg, packed[j * GS / 4], j * GS % 4, now_halves);
#pragma unroll
        for (int i = 0; i < TT; ++i) at[i] += x_stride;
        xg += xg_stride;
      }
      if (u >= u1 || tile != now_tile) {
        flush<TT>(sum, slots + (now_tile + warp) * ROWS * 8 * TT);
        fresh = true;
      }
      __syncwarp();                                        // all have read what the copies after the next replace
      slot = 2 * ring + SLOT - slot;
    }
    copy_wait<0>();
  }
};

// ---- tokens ----
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }      // |k| < 127
// 2^shift brings a row whose largest magnitude has the bits mx into [2^14, 2^15); 0 for a row that is not finite, whose sums will not be either.
template <bool BF16> __device__ __forceinline__ int row_shift(uint32_t mx) {
  const int ex = (int)(__float_as_uint(half_f<BF16>(mx)) >> 23);
  return mx == 0 || ex == 255 ? 0 : min(126, max(-126, 14 - (ex - 127)));
}
// v 2^(24 - shift), in two halves, so that what lies between them is beyond fp32 only where v or the result is
__device__ __forceinline__ float unshift(float v, int shift) { const int e = 24 - shift, half = e >> 1; return v * pow2(half) * pow2(e - half); }
__device__ __forceinline__ uint32_t max_bits(const uint4& v) {      // of eight magnitudes, which order as their bits
  const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
  return max(m & 0xFFFFu, m >> 16);
}
__device__ __forceinline__ uint4 ld_eight(const uint16_t* p, bool vec) {
  uint4 v;
  if (vec) {
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned short lo, hi;
      asm volatile("ld.global.u16 %0, [%1];" : "=h"(lo) : "l"(p + 2 * j));
      asm volatile("ld.global.u16 %0, [%1];" : "=h"(hi) : "l"(p + 2 * j + 1));
      w[j] = (uint32_t)lo | (uint32_t)hi << 16;
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
// Eight values as the products read them, and their sum: the k of low nibbles (0, 4), (2, 6), then those of high ones (1, 5), (3, 7), divided by 16.
template <bool BF16> __device__ __forceinline__ uint4 scaled_eight(const uint4& v, float f, float& sum) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) { x[2 * j] = half_f<BF16>(w[j] & 0xFFFFu) * f; x[2 * j + 1] = half_f<BF16>(w[j] >> 16) * f; }
  sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
  auto pack = [](float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); };
  constexpr float T = 1.f / 16;
  return make_uint4(pack(x[0], x[4]), pack(x[2], x[6]), pack(x[1] * T, x[5] * T), pack(x[3] * T, x[7] * T));
}
// Eight c of the row of token m, c counted from the image's first value, into the image `to`; whole half warps, which have consecutive c of one token.
template <int G, int TT, bool BF16> __device__ __forceinline__ void put_eight(uint8_t* to, int M, int m, int c, const uint4& v, float f, bool valid) {
  float sum = 0.f;
  uint8_t* step = to + (int64_t)(c >> 4) * step_bytes(M, G, TT);
  if (valid) *reinterpret_cast<uint4*>(step + m * STEP * 2 + eight_at(c & 15, m)) = scaled_eight<BF16>(v, f, sum);
#pragma unroll
  for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (valid && c % (G / 8) == 0) reinterpret_cast<float*>(step + M * STEP * 2)[(c & 15) / (G / 8) * 8 * TT + m] = sum * 5.9604644775390625e-8f;      // 2^-24
}
#endif

}  // namespace g4s
}  // namespace b2q
