// Rows to int8 codes and one scale per row: a = max(max |x|, 1e-12), scale = a / 127, code = rint(127 x / a) with halves to even, decided
// exactly (i8.cuh).  A row that holds an infinity or a NaN gets the scale NaN and zero codes, so that everything made from it is NaN.
//
// Three forms of x: a row of 16-bit (or fp32) values; silu(gate) * up; and the RMSNorm of hidden + residual, whose codes need no
// 1 / rms: it cancels out of v w / max |v w|, so that one reduction gives both the sum of squares and the maximum.  Where that sum overflows (bf16
// rows of rms above some 1e17) it is made again of 2^-80 v; other rows pay one test for it, behind the reduction.
//
// Memory-bound: a row is read once and stays in registers between the maximum and the codes.  Rows of up to 1024 values take a warp
// each, longer ones a CTA with one barrier; what is not 16-byte aligned, or longer than 1024 threads hold, is read twice.  The exponential
// and the division of SiLU keep an SM busy for half as long as the bytes take: where a row fills it (2048 x 28672: 68 us for 45 of bytes) the two add
// up.  A ring of bulk copies ahead of such rows took 59 us, but 20 % longer than this with two CTAs per SM.
#include "i8.cuh"

namespace b2q {

namespace i8q {
enum { PLAIN, SILU, NORM, COPIES, COMPUTED };              // COMPUTED: fp32 rows that are results themselves

struct Params {
  const void* x; int64_t ldx;                              // elements
  const void* residual; const void* nw; void* residual_out; float eps;
  const int32_t* n_valid;
  I8Copies to;                                             // COPIES
  int8_t* q; float* s; int64_t M; int K;
};

// The largest magnitude, NaN above all: half an instruction per value (as integers two: norm of 2047 x 8192 19.6 us for 17.0, SiLU 18.2 for 17.6).
__device__ __forceinline__ float abs_max(float m, float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
template <bool BF16> __device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t v) {      // of two packed values at a time
  uint32_t r;
  if constexpr (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(v & 0x7FFF7FFFu));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(v & 0x7FFF7FFFu));
  return r;
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }      // orders as |v|, NaN above all

// What a row's codes are made with: a stored row's exactly (row), a computed one's by r = 127 / a.
struct Scale {
  I8Row row;
  float r, scale;
  bool finite;
};
template <int MODE> __device__ __forceinline__ Scale row_scale(uint32_t mx, float sum, int K, float eps) {
  Scale s;
  if constexpr (MODE == NORM) {
    // codes of v w, whose maximum stands for the normed row's; of a row that is nearly nothing, of v w against the floor over 1 / rms
    const float rstd = rsqrtf(sum / (float)K + eps), an = __uint_as_float(mx) * rstd;
    s.finite = abs_bits(an) < 0x7F800000u && mx < 0x7F800000u && abs_bits(sum) <= 0x7F800000u;
    s.scale = fmaxf(an, I8_MIN_AMAX) / 127.f;
    s.r = 127.f / fmaxf(__uint_as_float(mx), I8_MIN_AMAX / rstd);
  } else {
    const float a = fmaxf(__uint_as_float(mx), I8_MIN_AMAX);
    s.finite = mx < 0x7F800000u;
    s.scale = a / 127.f;
    if constexpr (MODE == PLAIN || MODE == COPIES) s.row = i8_row(a); else s.r = 127.f / a;
  }
  if (!s.finite) s.scale = __uint_as_float(0x7FC00000u);
  return s;
}

constexpr float HUGE_UNIT = 8.271806125530277e-25f;        // 2^-80: 2^31 squares of it times the largest number add up to less than 2^128
// Of a row of the NORM form whose sum of squares overflows, from each thread's sum of the squares of HUGE_UNIT v; eps is nothing beside them.
template <bool WARP> __device__ __forceinline__ Scale huge_scale(float sum, uint32_t mx, int K, float* red) {
  const int lane = threadIdx.x & 31;
  auto add = [](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  sum = add(sum);
  if constexpr (!WARP) {
    __syncthreads();                                       // red is being read
    if (lane == 0) red[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = add(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.f);
  }
  const float a = __uint_as_float(mx), an = a * HUGE_UNIT * rsqrtf(sum / (float)K);
  Scale s;
  s.finite = abs_bits(an) < 0x7F800000u && mx < 0x7F800000u;
  s.scale = s.finite ? fmaxf(an, I8_MIN_AMAX) / 127.f : __uint_as_float(0x7FC00000u);
  s.r = 127.f / fmaxf(a, I8_MIN_AMAX / rsqrtf(sum / (float)K) / HUGE_UNIT);
  return s;
}

template <int DT> __device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  constexpr bool BF16 = DT == B2Q_BF16;
  unpack2<BF16>(v.x, f[0], f[1]); unpack2<BF16>(v.y, f[2], f[3]); unpack2<BF16>(v.z, f[4], f[5]); unpack2<BF16>(v.w, f[6], f[7]);
}

// Eight values of a row as they are to be quantised.  16-bit PLAIN keeps the raw words, the other forms the eight floats.
template <int MODE, int DT> struct Piece {
  float f[8];
  __device__ __forceinline__ void get(float (&o)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = f[i];
  }
};
template <int DT> struct RawPiece {
  uint4 v;
  __device__ __forceinline__ void get(float (&o)[8]) const { unpack8<DT>(v, o); }
};
template <> struct Piece<PLAIN, B2Q_BF16> : RawPiece<B2Q_BF16> {};
template <> struct Piece<PLAIN, B2Q_F16> : RawPiece<B2Q_F16> {};
template <> struct Piece<COPIES, B2Q_BF16> : RawPiece<B2Q_BF16> {};
template <> struct Piece<COPIES, B2Q_F16> : RawPiece<B2Q_F16> {};

// WARP: a row per warp, V pieces per lane.  Otherwise a row per CTA, V pieces per thread.
template <int MODE, int DT, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : (V == 8 ? 512 : 1024)) quantize_i8_kernel(const Params p) {
  __shared__ uint32_t red_max[32];
  __shared__ float red_sum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int step = WARP ? 32 : blockDim.x, first = WARP ? lane : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : (int64_t)blockIdx.x;
  if constexpr (MODE == COPIES) {                          // the grouped GEMM behind reads the routing's tile list as soon as it begins
    grid_dep_wait();
    grid_dep_release();
  } else {
    grid_dep_enter();
  }
  if (row >= p.M) return;                                  // whole warps, or the whole CTA
  if constexpr (MODE == PLAIN || MODE == COMPUTED) {
    if (p.n_valid && row >= *reinterpret_cast<const volatile int32_t*>(p.n_valid)) return;
  }
  const int n8 = p.K >> 3;
  constexpr bool BF16 = DT == B2Q_BF16;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.x) + row * p.ldx * (DT == B2Q_F32 ? 2 : 1);
  Piece<MODE, DT> pc[V];
  float top = 0.f;
  float sum = 0.f;
  if constexpr (MODE == PLAIN || MODE == COPIES || MODE == COMPUTED) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = first + i * step;
      if constexpr (DT == B2Q_F32) {
        const uint4 a = c < n8 ? ld_vec(x + 16 * c) : make_uint4(0, 0, 0, 0), b = c < n8 ? ld_vec(x + 16 * c + 8) : make_uint4(0, 0, 0, 0);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) pc[i].f[j] = __uint_as_float(w[j]);
      } else {
        pc[i].v = c < n8 ? ld_vec(x + 8 * c) : make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (DT == B2Q_F32) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) top = abs_max(top, pc[i].f[j], pc[i].f[j + 1]);
      }
    } else {
      uint32_t two = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) two = abs_max2<BF16>(abs_max2<BF16>(abs_max2<BF16>(abs_max2<BF16>(two, pc[i].v.x), pc[i].v.y), pc[i].v.z), pc[i].v.w);
      float a, b;
      unpack2<BF16>(two, a, b);
      top = abs_max(0.f, a, b);
    }
  } else if constexpr (MODE == SILU) {
    uint4 g[V], u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = first + i * step;
      const bool in = c < n8;
      g[i] = in ? ld_vec(x + 8 * c) : make_uint4(0, 0, 0, 0);
      u[i] = in ? ld_vec(x + p.K + 8 * c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a[8], b[8];
      unpack8<DT>(g[i], a);
      unpack8<DT>(u[i], b);
#pragma unroll
      for (int j = 0; j < 8; ++j) pc[i].f[j] = silu_mul_f(a[j], b[j]);
#pragma unroll
      for (int j = 0; j < 8; j += 2) top = abs_max(top, pc[i].f[j], pc[i].f[j + 1]);
    }
  } else {
    const uint16_t* rs = reinterpret_cast<const uint16_t*>(p.residual) + row * p.K;
    uint16_t* ro = reinterpret_cast<uint16_t*>(p.residual_out) + row * p.K;
    uint4 h[V], r[V], w[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = first + i * step;
      const bool in = c < n8;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      h[i] = in ? ld_vec(x + 8 * c) : zero;
      r[i] = in ? ld_vec(rs + 8 * c) : zero;
      w[i] = in ? ld_vec(reinterpret_cast<const uint16_t*>(p.nw) + 8 * c) : zero;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = first + i * step;
      float a[8], b[8];
      unpack8<DT>(h[i], a);
      unpack8<DT>(r[i], b);
#pragma unroll
      for (int j = 0; j < 8; ++j) { a[j] += b[j]; sum = fmaf(a[j], a[j], sum); }
      if (c < n8)
        *reinterpret_cast<uint4*>(ro + 8 * c) =
            make_uint4(pack2<BF16>(a[0], a[1]), pack2<BF16>(a[2], a[3]), pack2<BF16>(a[4], a[5]), pack2<BF16>(a[6], a[7]));
      unpack8<DT>(w[i], b);
#pragma unroll
      for (int j = 0; j < 8; ++j) pc[i].f[j] = a[j] * b[j];
#pragma unroll
      for (int j = 0; j < 8; j += 2) top = abs_max(top, pc[i].f[j], pc[i].f[j + 1]);
    }
  }
  uint32_t mx = __reduce_max_sync(0xffffffffu, abs_bits(top));
  if constexpr (MODE == NORM) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if constexpr (!WARP) {                                   // every warp finishes the reduction itself: one barrier
    const bool in = lane < (int)(blockDim.x >> 5);
    if (lane == 0) { red_max[warp] = mx; if constexpr (MODE == NORM) red_sum[warp] = sum; }
    __syncthreads();
    mx = __reduce_max_sync(0xffffffffu, in ? red_max[lane] : 0u);
    if constexpr (MODE == NORM) {
      sum = in ? red_sum[lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
  }
  const Scale sc = row_scale<MODE>(mx, sum, p.K, p.eps);
  int32_t copy = -1;                                       // lane n: the row of the n-th copy
  if constexpr (MODE == COPIES) {
    if (lane < p.to.k) {
      const int64_t pair = row * p.to.k + lane;
      const int32_t e = __ldcg(p.to.ids + pair);
      if (e >= 0) copy = __ldcg(p.to.base + row / p.to.run * p.to.E + e) + __ldcg(p.to.place + pair);
      if (WARP || warp == 0) {
        p.to.rows[pair] = copy;
        if (copy >= 0) p.s[copy] = sc.scale;
      }
    }
    __syncwarp();
  } else {
    if (first == 0) p.s[row] = sc.scale;
  }
  uint8_t* q = reinterpret_cast<uint8_t*>(p.q) + (MODE == COPIES ? 0 : row * p.K);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = first + i * step;
    float f[8];
    pc[i].get(f);
    const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
    uint2 o = make_uint2(0, 0);
    if (sc.finite) {
      if constexpr (MODE == PLAIN || MODE == COPIES) o = make_uint2(i8_codes4<DT == B2Q_F32>(lo, sc.row), i8_codes4<DT == B2Q_F32>(hi, sc.row));
      else o = make_uint2(i8_codes4_computed(lo, sc.r), i8_codes4_computed(hi, sc.r));
    }
    if constexpr (MODE == COPIES) {
      for (int n = 0; n < p.to.k; ++n) {
        const int32_t r = __shfl_sync(0xffffffffu, copy, n);
        if (r >= 0 && c < n8) *reinterpret_cast<uint2*>(q + (int64_t)r * p.K + 8 * c) = o;
      }
    } else {
      if (c < n8) *reinterpret_cast<uint2*>(q + 8 * c) = o;
    }
  }
  if constexpr (MODE == NORM && BF16) {
    if (!(sum < INFINITY)) {                               // the same for the whole row; what was stored above is replaced
      // In front of the codes, or out of line, this cost ordinary rows registers (4096 x 1024 up to 7.2 us for 5.7).  v is what is left of it: v w over w,
      // and where w is 0 the rounded v that this thread has written.
      __syncwarp();                                        // those writes stay in front of the loads
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = first + i * step;
        float f[8];
        pc[i].get(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c >= n8) continue;
          const float w = scalar_from_raw(ld_u16(reinterpret_cast<const uint16_t*>(p.nw) + 8 * c + j), DT);
          const float v = w != 0.f ? __fdividef(f[j], w) : scalar_from_raw(ld_u16(reinterpret_cast<const uint16_t*>(p.residual_out) + row * p.K + 8 * c + j), DT);
          sum = fmaf(v * HUGE_UNIT, v * HUGE_UNIT, sum);
        }
      }
      __syncwarp();
      const Scale huge = huge_scale<WARP>(sum, mx, p.K, red_sum);
      if (first == 0) p.s[row] = huge.scale;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = first + i * step;
        float f[8];
        pc[i].get(f);
        const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
        if (c < n8) *reinterpret_cast<uint2*>(q + 8 * c) = huge.finite ? make_uint2(i8_codes4_computed(lo, huge.r), i8_codes4_computed(hi, huge.r)) : make_uint2(0, 0);
      }
    }
  }
}

// Any K, any alignment: element by element, the row read twice.
template <int MODE, int DT>
__global__ void __launch_bounds__(512) quantize_i8_any_kernel(const Params p) {
  __shared__ uint32_t red_max[16];
  __shared__ float red_sum[16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  grid_dep_enter();
  if constexpr (MODE == PLAIN) {
    if (p.n_valid && row >= *reinterpret_cast<const volatile int32_t*>(p.n_valid)) return;
  }
  auto at = [&](const void* b, int64_t i) -> float {
    if constexpr (DT == B2Q_F32) return reinterpret_cast<const volatile float*>(b)[i];
    else return scalar_from_raw(reinterpret_cast<const volatile unsigned short*>(b)[i], DT);
  };
  uint32_t mx = 0;
  float sum = 0.f;
  for (int c = threadIdx.x; c < p.K; c += 512) {
    float v = at(p.x, row * p.ldx + c);
    if constexpr (MODE == SILU) v = silu_mul_f(v, at(p.x, row * p.ldx + p.K + c));
    if constexpr (MODE == NORM) {
      v += at(p.residual, row * p.K + c);
      sum = fmaf(v, v, sum);
      v *= at(p.nw, c);
    }
    mx = max(mx, abs_bits(v));
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) { red_max[warp] = mx; red_sum[warp] = sum; }
  __syncthreads();
  mx = __reduce_max_sync(0xffffffffu, lane < 16 ? red_max[lane] : 0u);
  sum = lane < 16 ? red_sum[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  Scale sc = row_scale<MODE>(mx, sum, p.K, p.eps);
  if constexpr (MODE == NORM && DT == B2Q_BF16) {
    if (!(sum < INFINITY)) {                               // the same for the whole row, and residual_out is not written yet
      sum = 0.f;
      for (int c = threadIdx.x; c < p.K; c += 512) {
        const float v = (at(p.x, row * p.ldx + c) + at(p.residual, row * p.K + c)) * HUGE_UNIT;
        sum = fmaf(v, v, sum);
      }
      __syncwarp();
      sc = huge_scale<false>(sum, mx, p.K, red_sum);
    }
  }
  if (threadIdx.x == 0) p.s[row] = sc.scale;
  for (int c = threadIdx.x; c < p.K; c += 512) {
    float v = at(p.x, row * p.ldx + c);
    if constexpr (MODE == SILU) v = silu_mul_f(v, at(p.x, row * p.ldx + p.K + c));
    if constexpr (MODE == NORM) {
      v += at(p.residual, row * p.K + c);
      store_scalar(p.residual_out, row * p.K + c, DT, v);
      v *= at(p.nw, c);
    }
    float m;
    if constexpr (MODE == PLAIN) m = __fadd_rn(i8_place<DT == B2Q_F32>(v, sc.row), I8_ROUND);
    else m = __fmaf_rn(v, sc.r, I8_ROUND);
    p.q[row * p.K + c] = sc.finite ? (int8_t)(__float_as_uint(m) & 255u) : (int8_t)0;
  }
}

template <typename... KArgs, typename... Args>
static int launch(void (*kern)(KArgs...), int64_t grid, int block, cudaStream_t st, Args&&... args) {
  if (grid > INT32_MAX) return B2Q_ERR_LIMIT;
  launch_overlapped(kern, dim3((unsigned)grid), dim3(block), 0, st, tls().overlap_mode > 0, args...);
  note_launch("quantize_i8");
  return launch_status();
}

template <int MODE, int DT> static int run_vec(const Params& p, cudaStream_t st) {
  const int n8 = p.K / 8;
  // short rows, and enough of them to fill the SMs: a warp each
  if (n8 <= 128 && p.M >= 148) {
    const int64_t grid = (p.M + 7) / 8;
    if (n8 <= 32) return launch(quantize_i8_kernel<MODE, DT, 1, true>, grid, 256, st, p);
    if (n8 <= 64) return launch(quantize_i8_kernel<MODE, DT, 2, true>, grid, 256, st, p);
    return launch(quantize_i8_kernel<MODE, DT, 4, true>, grid, 256, st, p);
  }
  auto block = [&](int v) { return (n8 + 32 * v - 1) / (32 * v) * 32; };
  // one CTA per SM at most: as many threads as a row gives work to
  if (p.M <= 148) {
    if (n8 <= 1024) return launch(quantize_i8_kernel<MODE, DT, 1, false>, p.M, block(1), st, p);
    if (n8 <= 2048) return launch(quantize_i8_kernel<MODE, DT, 2, false>, p.M, block(2), st, p);
    return launch(quantize_i8_kernel<MODE, DT, 4, false>, p.M, block(4), st, p);
  }
  // Two CTAs per SM at most (256 x 8192, with two / four / eight pieces a thread: stored rows 2.4 / 2.5 / 2.7 us, SiLU 3.5 / 4.2; norm 3.5 / 3.3).
  if (MODE != NORM && p.M <= 296 && n8 <= 2048) return launch(quantize_i8_kernel<MODE, DT, 2, false>, p.M, block(2), st, p);
  // Many rows: smaller CTAs with more in flight each.  Two / four / eight pieces: stored rows of 16384 x 1536 17.6 / 17.9 / 17.6 us, 4096 x 5120 13.2 / 11.8 /
  // 12.9, 2047 x 8192 11.1 / 10.0 / 9.7 (5.2 TB/s), 2048 x 28672 - / 44.8 / 35.2 (5.0 TB/s).  The other forms hold floats, and eight pieces of those do
  // not fit the registers: SiLU 16384 x 1536 24.9 / 28.5, 4096 x 2048 9.3 / 9.4, 4096 x 5120 21.8 / 20.4, 2047 x 8192 19.7 / 17.2; norm 4096 x 2048
  // 8.5 / 7.7, 4096 x 5120 23.3 / 21.5, 2047 x 8192 21.2 / 17.0.
  if (n8 < 256) return launch(quantize_i8_kernel<MODE, DT, 2, false>, p.M, block(2), st, p);
  if constexpr (MODE == PLAIN || MODE == COPIES) {
    if (n8 > 768) return launch(quantize_i8_kernel<MODE, DT, 8, false>, p.M, block(8), st, p);
  }
  return launch(quantize_i8_kernel<MODE, DT, 4, false>, p.M, block(4), st, p);
}

template <int MODE> static int run(const Params& p, int dt, bool vec, cudaStream_t st) {
  if (p.M == 0) return B2Q_OK;
  if (vec && p.K % 8 == 0 && p.K <= 32768) {
    if (dt == B2Q_BF16) return run_vec<MODE, B2Q_BF16>(p, st);
    if (dt == B2Q_F16) return run_vec<MODE, B2Q_F16>(p, st);
    if constexpr (MODE == PLAIN) return run_vec<MODE, B2Q_F32>(p, st);
  }
  if (dt == B2Q_BF16) return launch(quantize_i8_any_kernel<MODE, B2Q_BF16>, p.M, 512, st, p);
  if (dt == B2Q_F16) return launch(quantize_i8_any_kernel<MODE, B2Q_F16>, p.M, 512, st, p);
  if constexpr (MODE == PLAIN) return launch(quantize_i8_any_kernel<MODE, B2Q_F32>, p.M, 512, st, p);
  return B2Q_ERR_DTYPE;
}
static bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }
}  // namespace i8q

int quantize_i8(const void* x, int x_dtype, int64_t ldx, int8_t* q, float* s, int64_t M, int K, cudaStream_t st) {
  i8q::Params p{};
  p.x = x; p.ldx = ldx; p.q = q; p.s = s; p.M = M; p.K = K;
  return i8q::run<i8q::PLAIN>(p, x_dtype, aligned16(x) && i8q::aligned8(q) && ldx % 8 == 0, st);
}
int quantize_i8_computed(const float* x, const int32_t* n_valid, int8_t* q, float* s, int64_t M, int K, cudaStream_t st) {
  i8q::Params p{};
  p.x = x; p.ldx = K; p.n_valid = n_valid; p.q = q; p.s = s; p.M = M; p.K = K;
  return K <= 32768 ? i8q::run_vec<i8q::COMPUTED, B2Q_F32>(p, st) : i8q::run<i8q::PLAIN>(p, B2Q_F32, false, st);
}
int quantize_i8_copies(const void* x, bool bf16, const I8Copies& to, int8_t* q, float* s, int64_t M, int K, cudaStream_t st) {
  using namespace i8q;
  if (K > 32768) return B2Q_ERR_LIMIT;
  Params p{};
  p.x = x; p.ldx = K; p.to = to; p.q = q; p.s = s; p.M = M; p.K = K;
  return bf16 ? run_vec<COPIES, B2Q_BF16>(p, st) : run_vec<COPIES, B2Q_F16>(p, st);
}
int silu_mul_quantize_i8(const void* gate_up, bool bf16, int64_t ldx, int8_t* q, float* s, int64_t M, int K, cudaStream_t st) {
  i8q::Params p{};
  p.x = gate_up; p.ldx = ldx; p.q = q; p.s = s; p.M = M; p.K = K;
  return i8q::run<i8q::SILU>(p, bf16 ? B2Q_BF16 : B2Q_F16, aligned16(gate_up) && i8q::aligned8(q) && ldx % 8 == 0, st);
}
int resadd_rmsnorm_quantize_i8(const void* hidden, const void* residual, const void* w, void* residual_out, bool bf16, float eps, int8_t* q, float* s,
                               int64_t M, int K, cudaStream_t st) {
  i8q::Params p{};
  p.x = hidden; p.ldx = K; p.residual = residual; p.nw = w; p.residual_out = residual_out; p.eps = eps; p.q = q; p.s = s; p.M = M; p.K = K;
  return i8q::run<i8q::NORM>(p, bf16 ? B2Q_BF16 : B2Q_F16,
                             aligned16(hidden) && aligned16(residual) && aligned16(w) && aligned16(residual_out) && i8q::aligned8(q), st);
}

}  // namespace b2q
