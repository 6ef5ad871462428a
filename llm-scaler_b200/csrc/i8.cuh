// What the 8-bit integer operators share: the rounding of a row to int8, early starts, and their host interface.
#pragma once
#include "common.cuh"

namespace b2q {

// Smallest row maximum a scale is made from, as for the FP8 quantisers.
constexpr float I8_MIN_AMAX = 1e-12f;

// up to this many tokens the streaming kernels serve a call: one m16n8k32 MMA takes sixteen rows of codes
constexpr int I8_STREAM_MAX_TOK = 16;

struct I8LinearArgs {
  const int8_t* xq; int64_t ldx; const float* xs;          // codes [M, ldx], scales [M]; or, with x16 set,
  const void* x16; int64_t ldx16; bool x_bf16;             // the 16-bit rows to be quantised first (streaming kernel only)
  const int8_t* w; const void* ws; int ws_dtype;           // [N, K], [N]
  const void* bias;                                        // [N] in the output type, or null
  void* out; int64_t ldo; bool out_bf16;
  int M, N, K;
};
bool i8_stream_supported(const I8LinearArgs& a);           // of the 16-bit form: whether its codes fit the CTA's shared memory
int i8_stream_linear(const I8LinearArgs& a, cudaStream_t st);
int umma_i8_linear(const I8LinearArgs& a, cudaStream_t st);

// Grouped form: rows [offsets[e], offsets[e + 1]) of xq meet expert e's [N, K] of w.  gated: N is I and w holds 2 I rows per expert, gate then
// up; the output is silu(gate) * up in fp32.  Otherwise y in fp32.
struct I8GroupedArgs {
  const int8_t* xq; const float* xs; const int8_t* w; const void* ws; int ws_dtype;
  const int32_t* offsets; const int32_t* tiles; int tile_cap; int E;
  float* out; int rows, N, K; bool gated;
};
constexpr int I8_GROUPED_TILE = 128;
int umma_i8_grouped(const I8GroupedArgs& a, cudaStream_t st);

// q [M, K] codes, s [M] scales of rows of x; x_dtype B2Q_BF16 / F16 / F32.
int quantize_i8(const void* x, int x_dtype, int64_t ldx, int8_t* q, float* s, int64_t M, int K, cudaStream_t st);
// row r of the output belongs to row idx[r] / div of x (16 bit); rows from *n_valid on are left alone
int quantize_i8_gather(const void* x, bool bf16, int64_t ldx, const int32_t* idx, int div, const int32_t* n_valid, int8_t* q, float* s, int64_t rows, int K,
                       cudaStream_t st);
int silu_mul_quantize_i8(const void* gate_up, bool bf16, int64_t ldx, int8_t* q, float* s, int64_t M, int K, cudaStream_t st);
int resadd_rmsnorm_quantize_i8(const void* hidden, const void* residual, const void* w, void* residual_out, bool bf16, float eps, int8_t* q, float* s,
                               int64_t M, int K, cudaStream_t st);

#ifdef __CUDACC__
// Ordinary loads, never by the read-only path: these kernels begin while the kernel that writes their inputs is still running.
__device__ __forceinline__ uint4 ld_vec(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float ld_f32(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
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

// rint(127 x / a), half to even, decided exactly.  r = 127 / a rounded; x * r is then off by 2e-5 at most, and only within that of a half
// can the two round differently (a bf16 row holds exact halves often: every value that is half its row's largest).
__device__ __forceinline__ int i8_code_exact(float x, float a, float r) {
  const float t = fabsf(x) * r;
  float k = floorf(t);
  if (fabsf(t - k - 0.5f) < 1e-4f) {
    const double d = 254.0 * (double)fabsf(x), h = (2.0 * (double)k + 1.0) * (double)a;      // both exact
    if (d > h || (d == h && ((int)k & 1))) k += 1.f;
  } else {
    k = rintf(t);
  }
  return x < 0.f ? -(int)k : (int)k;
}
// Four codes, lowest byte first.  Adding 1.5 * 2^23 leaves the rounded product in the low byte; what the product is off from it says
// whether one of the four is near a half.
__device__ __forceinline__ uint32_t i8_codes4(const float (&x)[4], float a, float r) {
  constexpr float MAGIC = 12582912.f;
  uint32_t b[4];
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m = fmaf(x[i], r, MAGIC);
    off = fmaxf(off, fabsf(fmaf(x[i], r, -(m - MAGIC))));
    b[i] = __float_as_uint(m);
  }
  if (off > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = (uint32_t)i8_code_exact(x[i], a, r);
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
// Never contracted, so that every kernel gives the same bits.
__device__ __forceinline__ float i8_scaled(int sum, float scale, float wscale) { return __fmul_rn(__fmul_rn((float)sum, scale), wscale); }
__device__ __forceinline__ float i8_output(int sum, float scale, float wscale, float bias) { return __fadd_rn(i8_scaled(sum, scale, wscale), bias); }
__device__ __forceinline__ float silu_mul_f(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// D += A * B, 16 x 8 x 32, signed bytes: A rows are tokens, B columns weight rows
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
#endif

}  // namespace b2q
