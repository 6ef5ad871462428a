// Int8 linear of up to sixteen tokens and 20 Mi weights: out[m, n] = scale[m] wscale[n] sum_k codes[m, k] w[n, k] (+ bias[n]).
//
// HBM-bound: the weights are read once and nothing else is large.  They go from global memory straight into the registers that
// mma.sync m16n8k32 takes them from: with the k of a 64-byte piece permuted the same way on both sides, a lane's sixteen bytes of a weight
// row are the B operands of two MMAs (rows as the MMA's columns, tokens as its rows), so there is nothing to stage, convert or wait for
// but the loads themselves.
//
// Every CTA has rows of its own, dealt out evenly over two CTAs per SM.  Its eight warps share the work in units of eight 16-byte
// loads per lane (32 rows x 128 k, 16 x 256 or 8 x 512), an equal run of units each; the next unit's loads are on their way while a unit is
// multiplied.  Integer sums are exact in any order, so warps that share rows add into shared memory by atomics and every result is
// bit-identical whatever the division.
//
// 3 x 17408 x 5120 ran at 5.6 TB/s in umma_i8.cu, whose ring keeps more in flight per SM; below 20 Mi weights there is too little of that to matter, and
// this starts sooner: 1 x 2048 x 2048 3.1 us, of which 0.65 are the bytes'.
//
// The 16-bit form quantises the tokens by itself: each CTA makes all codes in its shared memory while its first weights arrive.
#include "i8.cuh"

namespace b2q {

namespace i8s {
constexpr int WARPS = 8, THREADS = 32 * WARPS, LOADS = 8;
// Values that the 16-bit form quantises in every CTA; beyond, a launch of its own costs less (2048 x 2048, 1 / 2 / 4 / 8 tokens 3.6 / 3.9 / 4.6 / 6.7 us
// in one launch, where codes given beforehand take 3.1 / 3.1 / 3.1 / 3.2 and a quantiser in front 1.2 more).
constexpr int FROM16_MAX = 8192;

struct Params {
  const int8_t* xq; int64_t ldx; const float* xs;
  const uint16_t* x16; int64_t ldx16;
  const int8_t* w; const void* ws; int ws_dtype; const void* bias;
  void* out; int64_t ldo;
  int M, N, K;
  int row_cap, code_pitch;                                 // rows of sums per token; bytes between two tokens' codes
  int early;                                               // weights may be read before the kernels in front are done
};

// R: eights of rows in a unit
template <int R, bool FROM16, bool BF16>
__global__ void __launch_bounds__(THREADS, 2) i8_stream_kernel(const Params p) {
  constexpr int S = LOADS / R, ROWS = 8 * R, KU = 64 * S;
  extern __shared__ __align__(16) uint8_t smem[];
  int* sums = reinterpret_cast<int*>(smem);                // [M][row_cap]
  uint8_t* codes = smem + (size_t)p.M * p.row_cap * 4;     // [M][code_pitch]
  __shared__ I8Tokens tok;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int r0 = (int)((int64_t)blockIdx.x * p.N / gridDim.x), rows = (int)((int64_t)(blockIdx.x + 1) * p.N / gridDim.x) - r0;
  const int nck = (p.K + KU - 1) / KU, units = (rows + ROWS - 1) / ROWS * nck;
  const int u0 = (int)((int64_t)warp * units / WARPS), u1 = (int)((int64_t)(warp + 1) * units / WARPS);

  grid_dep_release();
  uint4 cur[LOADS], nxt[LOADS];
  auto load = [&](int u, uint4 (&v)[LOADS]) {
    const int group = u / nck, k0 = (u - group * nck) * KU + 16 * t;
    const int8_t* base = p.w + (int64_t)(r0 + group * ROWS + g) * p.K + k0;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const bool in = group * ROWS + 8 * i + g < rows && k0 + 64 * j < p.K;
        v[i * S + j] = in ? ld_weight(base + (int64_t)(8 * i) * p.K + 64 * j) : make_uint4(0, 0, 0, 0);
      }
  };
  if (!p.early) grid_dep_wait();
  if (u0 < u1) load(u0, cur);
  for (int i = threadIdx.x; i < p.M * p.row_cap; i += THREADS) sums[i] = 0;
  if (FROM16 && threadIdx.x < I8_STREAM_MAX_TOK) tok.max[threadIdx.x] = 0;
  if (p.early) grid_dep_wait();
  __syncthreads();

  if constexpr (FROM16) {
    I8TokenCodes<BF16, THREADS, 4> tc(p.x16, p.ldx16, p.M, p.K);
    tc.fetch();
    tc.maximum(tok);
    __syncthreads();
    tc.rows(tok);
    __syncthreads();
    tc.codes(tok, codes, p.code_pitch);
    __syncthreads();
  }

  int acc[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[i][c] = 0;
  auto multiply = [&](int u, const uint4 (&v)[LOADS]) {
    const int group = u / nck, k0 = (u - group * nck) * KU + 16 * t;
    uint4 xa[S], xb[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const int k = k0 + 64 * j;
      xa[j] = xb[j] = make_uint4(0, 0, 0, 0);
      if constexpr (FROM16) {
        if (g < p.M && k < p.K) xa[j] = *reinterpret_cast<const uint4*>(codes + g * p.code_pitch + k);
        if (g + 8 < p.M && k < p.K) xb[j] = *reinterpret_cast<const uint4*>(codes + (g + 8) * p.code_pitch + k);
      } else {
        if (g < p.M && k < p.K) xa[j] = ld_vec(p.xq + g * p.ldx + k);
        if (g + 8 < p.M && k < p.K) xb[j] = ld_vec(p.xq + (g + 8) * p.ldx + k);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const uint4 w = v[i * S + j];
        mma_s8(acc[i], xa[j].x, xb[j].x, xa[j].y, xb[j].y, w.x, w.y);
        mma_s8(acc[i], xa[j].z, xb[j].z, xa[j].w, xb[j].w, w.z, w.w);
      }
  };
  auto flush = [&](int group) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int m = g + (c & 2) * 4, r = group * ROWS + 8 * i + 2 * t + (c & 1);
        if (m < p.M && r < rows) add_shared(sums + m * p.row_cap + r, acc[i][c]);
        acc[i][c] = 0;
      }
    }
  };
  for (int u = u0; u < u1; ++u) {
    if (u + 1 < u1) load(u + 1, nxt);
    multiply(u, cur);
    const int group = u / nck;
    if (u + 1 == u1 || (u + 1) / nck != group) flush(group);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) cur[i] = nxt[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.M * rows; i += THREADS) {
    const int m = i / rows, r = i - m * rows, n = r0 + r;
    const float s = FROM16 ? tok.scale[m] : ld_f32(p.xs + m);
    const float v = i8_output(sums[m * p.row_cap + r], s, load_scalar(p.ws, n, p.ws_dtype), p.bias ? load_scalar(p.bias, n, BF16 ? B2Q_BF16 : B2Q_F16) : 0.f);
    reinterpret_cast<uint16_t*>(p.out)[m * p.ldo + n] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
  }
}


template <int R, bool FROM16, bool BF16> static int launch(Params& p, int grid, cudaStream_t st) {
  p.row_cap = (p.N + grid - 1) / grid;
  p.row_cap = (p.row_cap + 3) / 4 * 4;                     // the codes behind the sums stay 16-byte aligned
  p.code_pitch = i8_code_pitch(p.K);
  const int smem = p.M * p.row_cap * 4 + (FROM16 ? p.M * p.code_pitch : 0);
  auto kern = i8_stream_kernel<R, FROM16, BF16>;
  launch_overlapped(kern, dim3(grid), dim3(THREADS), smem, st, tls().overlap_mode > 0, p);
  note_launch("i8_stream");
  return launch_status();
}

template <bool FROM16, bool BF16> static int pick(Params& p, cudaStream_t st) {
  // two CTAs per SM; more where the sums of that many rows would not fit the default shared memory beside the codes
  int grid = 2 * sm_count();
  while ((int64_t)p.M * ((p.N + grid - 1) / grid + 4) * 4 > 24 * 1024) grid *= 2;
  if (grid > p.N) grid = p.N;
  const int rows = (p.N + grid - 1) / grid;
  if (rows <= 8) return launch<1, FROM16, BF16>(p, grid, st);
  if (rows <= 16) return launch<2, FROM16, BF16>(p, grid, st);
  return launch<4, FROM16, BF16>(p, grid, st);
}
}  // namespace i8s

// Up to sixteen tokens and 20 Mi weights: straight from global memory (1 / 16 tokens, 2048 x 2048 3.1 / 3.5 us against 4.3 / 4.8 on tcgen05, 4096 x
// 4096 5.2 / 5.8 against 6.7 / 6.6, 2048 x 8192 6.4 / 8.2 against 7.8 / 8.2); more weights want the deeper ring (5120 x 5120 9.0 / 9.7 and
// 7.9 / 8.4, 17408 x 5120 19.4 / 22.4 and 15.6 / 16.0).
bool i8_stream_preferred(int64_t M, int64_t N, int64_t K) { return M <= I8_STREAM_MAX_TOK && N * K <= (int64_t)20 << 20; }
bool i8_stream_from16(int64_t M, int64_t N, int64_t K) { return i8_stream_preferred(M, N, K) && M * K <= i8s::FROM16_MAX; }

int i8_stream_linear(const I8LinearArgs& a, cudaStream_t st) {
  i8s::Params p{};
  p.xq = a.xq; p.ldx = a.ldx; p.xs = a.xs; p.x16 = reinterpret_cast<const uint16_t*>(a.x16); p.ldx16 = a.ldx16;
  p.w = a.w; p.ws = a.ws; p.ws_dtype = a.ws_dtype; p.bias = a.bias; p.out = a.out; p.ldo = a.ldo; p.M = a.M; p.N = a.N; p.K = a.K;
  p.early = tls().overlap_mode == 2;
  if (a.x16) return a.out_bf16 ? i8s::pick<true, true>(p, st) : i8s::pick<true, false>(p, st);
  return a.out_bf16 ? i8s::pick<false, true>(p, st) : i8s::pick<false, false>(p, st);
}

}  // namespace b2q
