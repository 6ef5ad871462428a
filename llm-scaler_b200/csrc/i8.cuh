// What the 8-bit integer operators share: the rounding of a row to int8, early starts, and their host interface.
#pragma once
#include "common.cuh"

namespace b2q {

// Smallest row maximum a scale is made from, as for the FP8 quantisers.
constexpr float I8_MIN_AMAX = 1e-12f;

// up to this many tokens the streaming kernels serve a call: one m16n8k32 MMA takes sixteen rows of codes
constexpr int I8_STREAM_MAX_TOK = 16;

int sm_count();                                            // of the current device; 148 where there is none

struct I8LinearArgs {
  const int8_t* xq; int64_t ldx; const float* xs;          // codes [M, ldx], scales [M]; or, with x16 set,
  const void* x16; int64_t ldx16; bool x_bf16;             // the 16-bit rows to be quantised first (streaming kernel only)
  const int8_t* w; const void* ws; int ws_dtype;           // [N, K], [N]
  const void* bias;                                        // [N] in the output type, or null
  void* out; int64_t ldo; bool out_bf16;
  int M, N, K;
};
bool i8_stream_from16(int64_t M, int64_t N, int64_t K);    // whether the 16-bit form is worth its quantising in every CTA
bool i8_stream_preferred(int64_t M, int64_t N, int64_t K);
int i8_stream_linear(const I8LinearArgs& a, cudaStream_t st);
int umma_i8_linear(const I8LinearArgs& a, cudaStream_t st);

// Grouped form: rows [offsets[e], offsets[e + 1]) of xq meet expert e's [N, K] of w.  gated: N is I and w holds 2 I rows per expert, gate then
// up; the output is silu(gate) * up.
struct I8GroupedArgs {
  const int8_t* xq; const float* xs; const int8_t* w; const void* ws; int ws_dtype;
  const int32_t* offsets; const int32_t* tiles; int tile, tile_cap, E;      // tile list of this height (i8_grouped_tile)
  void* out; bool out_bf16, out_f32; int rows, N, K; bool gated;      // gated: out is fp32 too
};
int i8_grouped_tile(int64_t rows, int E);
int umma_i8_grouped(const I8GroupedArgs& a, cudaStream_t st);

// A whole expert layer of up to sixteen tokens in one kernel (moe_i8.cu).
struct I8FewArgs {
  const void* x; bool bf16; const void* logits; int logits_dtype;
  const int8_t* w13; const void* s13; int s13_dtype; const int8_t* w2; const void* s2; int s2_dtype;
  void* out; int T, E, k, H, I; bool renorm;
  void* scratch;                                           // moe_i8_few_bytes(), 256-byte aligned
};
constexpr int I8_FEW_LOAD = 40960;                         // most of T (4 k I + H)
bool moe_i8_few_preferred(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I);
size_t moe_i8_few_bytes(int64_t T, int64_t k, int64_t I);
int moe_i8_few(const I8FewArgs& a, cudaStream_t st);

// q [M, K] codes, s [M] scales of rows of x; x_dtype B2Q_BF16 / F16 / F32.
int quantize_i8(const void* x, int x_dtype, int64_t ldx, int8_t* q, float* s, int64_t M, int K, cudaStream_t st);
// codes of the first *n_valid of M fp32 rows, a number that only the device knows; the rows are results themselves, so that halves are not decided
// to the last bit.  x 16-byte aligned, K % 8 == 0
int quantize_i8_computed(const float* x, const int32_t* n_valid, int8_t* q, float* s, int64_t M, int K, cudaStream_t st);
// the same with a copy of row r for each of its k pairs, at rows[pair] = base[r / run, ids[pair]] + place[pair] (moe_i8_route), which it also writes;
// -1, and no copy, where the pair has no expert.  x contiguous, 16 bit, K % 8 == 0
struct I8Copies {
  const int32_t *ids, *place, *base;
  int32_t* rows;
  int k, E, run;
};
int quantize_i8_copies(const void* x, bool bf16, const I8Copies& to, int8_t* q, float* s, int64_t M, int K, cudaStream_t st);
int silu_mul_quantize_i8(const void* gate_up, bool bf16, int64_t ldx, int8_t* q, float* s, int64_t M, int K, cudaStream_t st);
int resadd_rmsnorm_quantize_i8(const void* hidden, const void* residual, const void* w, void* residual_out, bool bf16, float eps, int8_t* q, float* s,
                               int64_t M, int K, cudaStream_t st);

// The expert layer of many tokens (moe_i8_many.cu): routing, with base for moe_i8_route_ctas(T) runs of ceil(T / that) tokens; weighted sum.
int moe_i8_route_ctas(int64_t T);
int moe_i8_route(const void* logits, int dt, int64_t T, int E, int k, bool renorm, int tile, float* weights, int32_t* ids, int32_t* place, int32_t* base,
                 int32_t* offsets, int32_t* tiles, void* count, cudaStream_t st);
struct I8Outputs {                                         // what the outputs are made of: codes and scales of h by row, the experts' matrices, the pairs' experts
  const int8_t* q; const float* s; const int8_t* w; const void* ws; int ws_dt; const int32_t* ids; int I;
};
int moe_i8_sum(const void* y, bool y_f32, const float* weights, const int32_t* rows, const I8Outputs& of, void* out, bool bf16, int64_t T, int k, int H, cudaStream_t st);

#ifdef __CUDACC__
// As in moe_aux.cu: a grid that fills the GPU lets the next one begin later.
__device__ __forceinline__ void grid_dep_enter() {
  const bool few = gridDim.x <= 148;
  if (few) grid_dep_release();
  grid_dep_wait();
  if (!few) grid_dep_release();
}

// Ordinary loads, never by the read-only path: these kernels begin while the kernel that writes their inputs is still running.  Volatile
// keeps them behind the wait for it; without a memory clobber several are on their way at a time.
__device__ __forceinline__ uint4 ld_vec(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_u16(const uint16_t* p) {
  unsigned short v;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_f32(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
// Sixteen bytes of a weight: read once per call by one thread, so not worth a line of L1.
__device__ __forceinline__ uint4 ld_weight(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <bool BF16> __device__ __forceinline__ void unpack2(uint32_t v, float& a, float& b) {
  if constexpr (BF16) { a = __uint_as_float(v << 16); b = __uint_as_float(v & 0xFFFF0000u); }
  else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v)); a = f.x; b = f.y; }
}
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {      // a in the lower half
  if constexpr (BF16) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
  else { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
}

// What the codes of a row need of its largest value: rint(127 x / a), halves to even, decided exactly.  The quotient of y = 127 x by a is
// corrected once by its remainder, which is exact in fp32, and is good to about 2^-24 of itself then; a quotient that is a half comes out as one, and of
// 16-bit values no other is nearer to a half than 2^-18.9 of it (by enumeration: fp16 a = 2047, x = 1910; bf16 2^-16.0; bf16 rows below the floor
// 2^-14.3).  (A bf16 row has exact halves by the dozen: every value that is half its row's largest.  Deciding the near ones in a branch of their own
// cost more than this: three of ten warps went there.)  Rows of huge values are taken 2^-40 of.
struct I8Row {
  float c, a, ra;                                          // 127, a, 1 / a, or the first two 2^-40 times that
};
__device__ __forceinline__ I8Row i8_row(float a) {
  const float f = a > 1e30f ? 9.094947e-13f : 1.f;
  return I8Row{127.f * f, a * f, 1.f / (a * f)};
}
constexpr float I8_ROUND = 12582912.f;                     // 1.5 * 2^23: added, it leaves a small value's nearest integer in the low byte
__device__ __forceinline__ uint32_t i8_pack4(const float (&m)[4]) {      // values plus I8_ROUND -> four codes, lowest byte first
  return __byte_perm(__byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x0040), __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x0040), 0x5410);
}
// WIDE: x has more than eleven significant bits, so that 127 x needs a second word.
template <bool WIDE> __device__ __forceinline__ float i8_place(float x, const I8Row& r) {
  const float y = __fmul_rn(x, r.c), t = __fmul_rn(y, r.ra);
  float rem = __fmaf_rn(-t, r.a, y);
  if constexpr (WIDE) {
    const float low = __fmaf_rn(x, r.c, -y), q = __fmaf_rn(__fadd_rn(rem, low), r.ra, t);
    // the quotient may be rounded to a half without being one: its own remainder tells
    rem = __fadd_rn(__fmaf_rn(-q, r.a, y), low);
    return fabsf(q - rintf(q)) == 0.5f && rem != 0.f ? q + copysignf(0.0009765625f, rem) : q;
  } else {
    return __fmaf_rn(rem, r.ra, t);
  }
}
template <bool WIDE> __device__ __forceinline__ uint32_t i8_codes4(const float (&x)[4], const I8Row& r) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __fadd_rn(i8_place<WIDE>(x[i], r), I8_ROUND);
  return i8_pack4(m);
}
// Of values that are rounded themselves, where the last bit of the quotient means nothing: r = 127 / a.
__device__ __forceinline__ uint32_t i8_codes4_computed(const float (&x)[4], float r) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __fmaf_rn(x[i], r, I8_ROUND);
  return i8_pack4(m);
}
// Never contracted, so that every kernel gives the same bits.
__device__ __forceinline__ float i8_scaled(int sum, float scale, float wscale) { return __fmul_rn(__fmul_rn((float)sum, scale), wscale); }
__device__ __forceinline__ float i8_output(int sum, float scale, float wscale, float bias) { return __fadd_rn(i8_scaled(sum, scale, wscale), bias); }
__device__ __forceinline__ float rcp_f(float v) {      // of 1 and more: to a unit in the last place, zero beyond 2^126
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// To within a few units in the last place: codes are made from it, and each that lands on the other side of a half is a step off (with the
// fast exponential an fp16 layer of 14336 wide experts was off by 4.3e-4 of its norm instead of 2.1e-4).
__device__ __forceinline__ float silu_mul_f(float g, float u) { return g * rcp_f(1.f + expf(-g)) * u; }

// Bytes between two tokens' codes in shared memory: 64 apart in the banks, so that a quarter warp reads two tokens' 64 bytes without a conflict.
__host__ __device__ constexpr int i8_code_pitch(int K) { return (K + 127) / 128 * 128 + 64; }

// All codes of M rows x [M, ldx] into shared memory, by the first THREADS threads of a CTA, in three steps with a barrier of theirs between two:
// maximum, rows, codes.  tok.max is zero before, K % 8 == 0.  A thread's pieces of eight stay in registers from the first step to the
// last, V of them; more are read twice.
struct I8Tokens {
  uint32_t max[I8_STREAM_MAX_TOK];
  float scale[I8_STREAM_MAX_TOK];
  I8Row row[I8_STREAM_MAX_TOK];
  int16_t list[I8_STREAM_MAX_TOK];                         // of the tokens that are wanted, where that is not all of them
  int count;
};
template <bool BF16, int THREADS, int V> struct I8TokenCodes {
  const uint16_t* x; int64_t ldx;
  bool vec;                                                // rows are 16-byte aligned
  int M, n8, total;
  uint32_t inv;                                            // i / n8 = i * inv >> 32 for the sizes that fit shared memory (i < 2^17, n8 < 2^14)
  const int16_t* list = nullptr;
  uint4 v[V];
  __device__ __forceinline__ void only(const I8Tokens& tok) {      // those of tok.list
    list = tok.list;
    M = tok.count;
    total = M * n8;
  }
  __device__ __forceinline__ int actual(int m) const { return list ? list[min(m, M - 1)] : m; }
  __device__ __forceinline__ I8TokenCodes(const uint16_t* x_, int64_t ldx_, int M_, int K) : x(x_), ldx(ldx_), M(M_), n8(K >> 3), total(M_ * (K >> 3)) {
    vec = ((reinterpret_cast<uintptr_t>(x_) | (uintptr_t)(2 * ldx_)) & 15u) == 0;
    inv = 0xFFFFFFFFu / (uint32_t)n8 + 1;
  }
  __device__ __forceinline__ int token(int i) const { return n8 == 1 ? i : (int)__umulhi((uint32_t)i, inv); }
  __device__ __forceinline__ void fetch(int base = 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = base + j * THREADS + threadIdx.x, m = token(i);
      v[j] = make_uint4(0, 0, 0, 0);
      if (i < total) {
        const uint16_t* at = x + actual(m) * ldx + 8 * (i - m * n8);
        if (vec) v[j] = ld_vec(at);
        else v[j] = make_uint4(ld_u16(at) | ld_u16(at + 1) << 16, ld_u16(at + 2) | ld_u16(at + 3) << 16, ld_u16(at + 4) | ld_u16(at + 5) << 16, ld_u16(at + 6) | ld_u16(at + 7) << 16);
      }
    }
  }
  __device__ __forceinline__ void maximum(I8Tokens& tok) { // behind fetch()
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < total; base += V * THREADS) {
      if (base) fetch(base);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i0 = base + j * THREADS + (int)(threadIdx.x & ~31u);
        if (i0 >= total) break;                            // whole warps
        const uint32_t e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        uint32_t mx = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float a, b;
          unpack2<BF16>(e[c], a, b);
          mx = max(mx, max(__float_as_uint(a) & 0x7FFFFFFFu, __float_as_uint(b) & 0x7FFFFFFFu));
        }
        const int m = token(i0);
        if (token(i0 + 31) == m) {
          mx = __reduce_max_sync(0xffffffffu, mx);
          if (lane == 0) atomicMax(&tok.max[actual(m)], mx);
        } else if (i0 + lane < total) {                    // a warp that straddles tokens
          atomicMax(&tok.max[actual(token(i0 + lane))], mx);
        }
        __syncwarp();
      }
    }
  }
  __device__ __forceinline__ void rows(I8Tokens& tok) const {
    if (threadIdx.x < M) {
      const int m = actual(threadIdx.x);
      const uint32_t bits = tok.max[m];
      const float a = fmaxf(__uint_as_float(bits), I8_MIN_AMAX);
      I8Row r = i8_row(a);
      if (bits >= 0x7F800000u) r = I8Row{0.f, 0.f, 0.f};   // not finite
      tok.row[m] = r;
      tok.scale[m] = bits < 0x7F800000u ? a / 127.f : __uint_as_float(0x7FC00000u);
    }
    __syncwarp();
  }
  __device__ __forceinline__ void codes(const I8Tokens& tok, uint8_t* to, int pitch) {
    for (int base = 0; base < total; base += V * THREADS) {
      if (total > V * THREADS) fetch(base);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = base + j * THREADS + threadIdx.x;
        if (i >= total) break;
        const int n = token(i), m = actual(n);
        const I8Row r = tok.row[m];
        float lo[4], hi[4];
        unpack2<BF16>(v[j].x, lo[0], lo[1]); unpack2<BF16>(v[j].y, lo[2], lo[3]); unpack2<BF16>(v[j].z, hi[0], hi[1]); unpack2<BF16>(v[j].w, hi[2], hi[3]);
        uint2 o = make_uint2(0, 0);
        if (r.c != 0.f) o = make_uint2(i8_codes4<false>(lo, r), i8_codes4<false>(hi, r));
        *reinterpret_cast<uint2*>(to + m * pitch + 8 * (i - n * n8)) = o;
      }
    }
    __syncwarp();
  }
};
__device__ __forceinline__ void add_shared(int* p, int v) {
  asm volatile("red.shared.add.s32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(p)), "r"(v) : "memory");
}

// D += A * B, 16 x 8 x 32, signed bytes: A rows are tokens, B columns weight rows
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
#endif

}  // namespace b2q
