// 4-bit group-quantised weights, any number of tokens: tiles of 64 x 64 outputs in fp32, dense and by expert.
#include "g4.cuh"

namespace b2q {
namespace g4t {
constexpr int TM = 64, TN = 64, TK = 32, THREADS = 256;

struct Params {
  const void* x; int64_t ldx; int bf16;
  const uint8_t* w; const void* s; const uint8_t* z;
  const void* bias; void* out; int64_t ldo; int out_f32;
  int M, N, K, G;
  const int32_t* ids; int E, k, x_div; const float* weights;      // by expert: rows are pairs, x row = pair / x_div
};

template <bool BF16, bool MOE> __global__ void __launch_bounds__(THREADS) g4_tile_kernel(const Params p) {
  __shared__ float xs[TK][TM + 1], ws[TK][TN + 1];
  __shared__ int list[TM];
  __shared__ int found;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n0 = blockIdx.x * TN, e = MOE ? blockIdx.y : 0;
  constexpr int DT = BF16 ? B2Q_BF16 : B2Q_F16;
  const uint8_t* w = p.w + (int64_t)e * p.N * (p.K / 2);
  const int64_t sg = (int64_t)e * (p.K / p.G) * p.N;
  grid_dep_release();
  grid_dep_wait();
  int next = MOE ? 0 : blockIdx.y * TM;
  for (;;) {
    int rows;
    if (MOE) {
      if (threadIdx.x == 0) {
        int n = 0;
        for (; next < p.M && n < TM; ++next)
          if (p.ids[next] == e) list[n++] = next;
        found = n;
      }
      __syncthreads();
      rows = found;
      if (rows == 0) return;
    } else {
      rows = min(TM, p.M - next);
    }
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += TK) {
      for (int i = threadIdx.x; i < TM * TK; i += THREADS) {
        const int r = i / TK, kk = i % TK;
        float v = 0.f;
        if (r < rows) {
          const int64_t row = MOE ? list[r] / p.x_div : next + r;
          v = load_scalar(p.x, row * p.ldx + k0 + kk, DT);
        }
        xs[kk][r] = v;
      }
      for (int i = threadIdx.x; i < TN * TK; i += THREADS) {
        const int r = i / TK, kk = i % TK, n = n0 + r;
        float v = 0.f;
        if (n < p.N) {
          const int64_t g = sg + (int64_t)((k0 + kk) / p.G) * p.N + n;
          const int b = w[(int64_t)n * (p.K / 2) + (k0 + kk) / 2], q = kk & 1 ? b >> 4 : b & 15;
          v = (float)(q - (p.z ? p.z[g] : 8)) * load_scalar(p.s, g, DT);
        }
        ws[kk][r] = v;
      }
      __syncthreads();
      for (int kk = 0; kk < TK; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[kk][ty * 4 + i], ws[kk][tx + 16 * j], acc[i][j]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = ty * 4 + i, n = n0 + tx + 16 * j;
        if (r >= rows || n >= p.N) continue;
        const int64_t row = MOE ? list[r] : next + r;
        const float v = acc[i][j] + (p.bias ? load_scalar(p.bias, n, DT) : 0.f);
        store_scalar(p.out, row * p.ldo + n, p.out_f32 ? B2Q_F32 : DT, v);
      }
    __syncthreads();
    if (!MOE) return;
  }
}

template <bool BF16> __global__ void g4_tile_silu_kernel(const float* gu, void* h, int64_t total, int I) {
  grid_dep_release();
  grid_dep_wait();
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t r = i / I, c = i % I;
    const float g = gu[r * 2 * I + c], u = gu[r * 2 * I + I + c];
    store_scalar(h, i, BF16 ? B2Q_BF16 : B2Q_F16, g / (1.f + expf(-g)) * u);
  }
}
template <bool BF16> __global__ void g4_tile_sum_kernel(const float* y, const float* w, const int32_t* ids, void* out, int64_t total, int H, int k, int E) {
  grid_dep_release();
  grid_dep_wait();
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t t = i / H, c = i % H;
    float acc = 0.f;
    for (int s = 0; s < k; ++s) {
      const int e = ids[t * k + s];
      if (e >= 0 && e < E) acc = fmaf(w[t * k + s], y[(t * k + s) * H + c], acc);
    }
    store_scalar(out, i, BF16 ? B2Q_BF16 : B2Q_F16, acc);
  }
}
}  // namespace g4t

int g4_tile_linear(const G4LinearArgs& a, cudaStream_t st) {
  using namespace g4t;
  Params p{};
  p.x = a.x; p.ldx = a.ldx; p.w = a.w; p.s = a.scale; p.z = a.zero; p.bias = a.bias; p.out = a.out; p.ldo = a.ldo; p.M = a.M; p.N = a.N; p.K = a.K; p.G = a.G;
  const dim3 grid((a.N + TN - 1) / TN, (a.M + TM - 1) / TM);
  launch_overlapped(a.bf16 ? g4_tile_kernel<true, false> : g4_tile_kernel<false, false>, grid, dim3(THREADS), 0, st, tls().overlap_mode > 0, p);
  note_launch("g4_tile");
  return launch_status();
}

size_t g4_tile_moe_bytes(const G4MoeArgs& a) { return (size_t)a.T * a.k * (2 * (size_t)a.I * 4 + (size_t)a.I * 2 + (size_t)a.H * 4) + 1024; }

int g4_tile_moe(const G4MoeArgs& a, void* scratch, cudaStream_t st) {
  using namespace g4t;
  const int64_t pairs = (int64_t)a.T * a.k;
  float* y = reinterpret_cast<float*>(scratch);
  float* gu = y + pairs * a.H;
  void* h = gu + pairs * 2 * a.I;
  const bool ov = tls().overlap_mode > 0;
  Params p{};
  p.x = a.x; p.ldx = a.H; p.w = a.w13; p.s = a.s13; p.z = a.z13; p.out = gu; p.ldo = 2 * a.I; p.out_f32 = 1; p.M = (int)pairs; p.N = 2 * a.I; p.K = a.H; p.G = a.G13;
  p.ids = a.ids; p.E = a.E; p.k = a.k; p.x_div = a.k;
  auto kern = a.bf16 ? g4_tile_kernel<true, true> : g4_tile_kernel<false, true>;
  launch_overlapped(kern, dim3((p.N + TN - 1) / TN, a.E), dim3(THREADS), 0, st, ov, p);
  launch_overlapped(a.bf16 ? g4_tile_silu_kernel<true> : g4_tile_silu_kernel<false>, dim3(592), dim3(256), 0, st, ov, (const float*)gu, h, pairs * a.I, a.I);
  p.x = h; p.ldx = a.I; p.w = a.w2; p.s = a.s2; p.z = a.z2; p.out = y; p.ldo = a.H; p.N = a.H; p.K = a.I; p.G = a.G2; p.x_div = 1;
  launch_overlapped(kern, dim3((p.N + TN - 1) / TN, a.E), dim3(THREADS), 0, st, ov, p);
  launch_overlapped(a.bf16 ? g4_tile_sum_kernel<true> : g4_tile_sum_kernel<false>, dim3(592), dim3(256), 0, st, ov, (const float*)y, a.weights, a.ids, a.out, (int64_t)a.T * a.H,
                    a.H, a.k, a.E);
  note_launch("g4_tile", 4);
  return launch_status();
}
}  // namespace b2q
