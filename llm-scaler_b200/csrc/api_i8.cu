// C ABI of the 8-bit integer operators: argument validation and kernel selection, as in api.cu.
#include "i8.cuh"

namespace b2q {
int sm_count() {
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
}  // namespace b2q

using namespace b2q;

namespace {
bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool known(int dtype) { return dtype >= 0 && dtype <= 2; }
size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
constexpr int64_t MAX_K = 131071;                          // 128 * 128 * K stays below 2^31
constexpr int64_t MAX_ROWS = INT32_MAX - 4096;             // tokens and weight rows of a linear: rounded up to tiles and rounds of tiles, both below this
constexpr int64_t MAX_COLUMNS = INT32_MAX - 512;           // of the quantisers, which count them in steps of 512

int linear_check(const I8LinearArgs& a, int64_t M, int64_t N, int64_t K) {
  if (!a.w || !a.ws || !a.out) return B2Q_ERR_NULL;
  if (!known(a.ws_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || N < 0 || K <= 0 || K % 16 != 0 || a.ldo < N) return B2Q_ERR_SHAPE;
  if (M > MAX_ROWS || N > MAX_ROWS || K > MAX_K) return B2Q_ERR_LIMIT;
  if (!aligned16(a.w) || !aligned_to(a.out, 2) || !aligned_to(a.bias, 2) || !aligned_to(a.ws, dtype_bytes(a.ws_dtype))) return B2Q_ERR_ALIGN;
  return B2Q_OK;
}
// set_force_kernel(2): tcgen05 for everything, no cooperative launch
bool use_stream(const I8LinearArgs& a) { return tls().force_kernel != 2 && i8_stream_preferred(a.M, a.N, a.K); }
bool use_from16(int64_t M, int64_t N, int64_t K) { return tls().force_kernel != 2 && i8_stream_from16(M, N, K); }
bool use_few(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I) { return tls().force_kernel != 2 && moe_i8_few_preferred(T, E, k, H, I); }
}  // namespace

extern "C" {

int b2q_quantize_int8(const void* x, int x_dtype, int64_t ldx, int8_t* q, float* scale, int64_t M, int64_t K, void* stream) {
  if (!x || !q || !scale) return B2Q_ERR_NULL;
  if (!known(x_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || K <= 0 || ldx < K) return B2Q_ERR_SHAPE;
  if (M > INT32_MAX || K > MAX_COLUMNS) return B2Q_ERR_LIMIT;
  if (!aligned_to(x, dtype_bytes(x_dtype)) || !aligned_to(scale, 4)) return B2Q_ERR_ALIGN;
  return quantize_i8(x, x_dtype, ldx, q, scale, M, (int)K, (cudaStream_t)stream);
}

int b2q_silu_mul_quantize_int8(const void* gate_up, int act_dtype, int64_t ldx, int8_t* q, float* scale, int64_t M, int64_t K, void* stream) {
  if (!gate_up || !q || !scale) return B2Q_ERR_NULL;
  if (!is16(act_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || K <= 0 || ldx < 2 * K) return B2Q_ERR_SHAPE;
  if (M > INT32_MAX || K > INT32_MAX / 2) return B2Q_ERR_LIMIT;
  if (!aligned_to(gate_up, 2) || !aligned_to(scale, 4)) return B2Q_ERR_ALIGN;
  return silu_mul_quantize_i8(gate_up, act_dtype == B2Q_BF16, ldx, q, scale, M, (int)K, (cudaStream_t)stream);
}

int b2q_resadd_rmsnorm_quantize_int8(const void* hidden, const void* residual, const void* norm_weight, void* residual_out, int act_dtype,
                                     float eps, int8_t* q, float* scale, int64_t M, int64_t K, void* stream) {
  if (!hidden || !residual || !norm_weight || !residual_out || !q || !scale) return B2Q_ERR_NULL;
  if (!is16(act_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || K <= 0) return B2Q_ERR_SHAPE;
  if (M > INT32_MAX || K > MAX_COLUMNS) return B2Q_ERR_LIMIT;
  if (!aligned_to(hidden, 2) || !aligned_to(residual, 2) || !aligned_to(norm_weight, 2) || !aligned_to(residual_out, 2) || !aligned_to(scale, 4))
    return B2Q_ERR_ALIGN;
  return resadd_rmsnorm_quantize_i8(hidden, residual, norm_weight, residual_out, act_dtype == B2Q_BF16, eps, q, scale, M, (int)K,
                                    (cudaStream_t)stream);
}

int b2q_linear_int8(const int8_t* q, int64_t ldq, const float* scale, const int8_t* w, const void* wscale, int wscale_dtype, const void* bias,
                    void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N, int64_t K, void* stream) {
  if (!q || !scale) return B2Q_ERR_NULL;
  if (!is16(out_dtype)) return B2Q_ERR_DTYPE;
  I8LinearArgs a{};
  a.xq = q; a.ldx = ldq; a.xs = scale; a.w = w; a.ws = wscale; a.ws_dtype = wscale_dtype; a.bias = bias;
  a.out = out; a.ldo = ldo; a.out_bf16 = out_dtype == B2Q_BF16; a.M = (int)M; a.N = (int)N; a.K = (int)K;
  const int rc = linear_check(a, M, N, K);
  if (rc) return rc;
  if (ldq < K) return B2Q_ERR_SHAPE;
  if (!aligned16(q) || ldq % 16 != 0 || !aligned_to(scale, 4)) return B2Q_ERR_ALIGN;
  if (M == 0 || N == 0) return B2Q_OK;
  return use_stream(a) ? i8_stream_linear(a, (cudaStream_t)stream) : umma_i8_linear(a, (cudaStream_t)stream);
}

size_t b2q_linear_int8_dynamic_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (use_from16(M, N, K)) return 0;
  return align_up((size_t)M * (size_t)K, 256) + align_up((size_t)M * 4, 256);
}

int b2q_linear_int8_dynamic(const void* x, int act_dtype, int64_t ldx, const int8_t* w, const void* wscale, int wscale_dtype, const void* bias,
                            void* out, int64_t ldo, int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (!x) return B2Q_ERR_NULL;
  if (!is16(act_dtype)) return B2Q_ERR_DTYPE;
  I8LinearArgs a{};
  a.x16 = x; a.ldx16 = ldx; a.x_bf16 = act_dtype == B2Q_BF16; a.w = w; a.ws = wscale; a.ws_dtype = wscale_dtype; a.bias = bias;
  a.out = out; a.ldo = ldo; a.out_bf16 = a.x_bf16; a.M = (int)M; a.N = (int)N; a.K = (int)K;
  int rc = linear_check(a, M, N, K);
  if (rc) return rc;
  if (ldx < K) return B2Q_ERR_SHAPE;
  if (!aligned_to(x, 2)) return B2Q_ERR_ALIGN;
  if (M == 0 || N == 0) return B2Q_OK;
  if (use_from16(M, N, K)) return i8_stream_linear(a, (cudaStream_t)stream);
  if (!workspace) return B2Q_ERR_NULL;
  if (!aligned16(workspace)) return B2Q_ERR_ALIGN;
  if (workspace_bytes < b2q_linear_int8_dynamic_workspace_bytes(M, N, K)) return B2Q_ERR_WORKSPACE;
  int8_t* q = reinterpret_cast<int8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + align_up((size_t)M * (size_t)K, 256));
  rc = quantize_i8(x, act_dtype, ldx, q, s, M, (int)K, (cudaStream_t)stream);
  if (rc) return rc;
  a.x16 = nullptr; a.xq = q; a.ldx = K; a.xs = s;
  return use_stream(a) ? i8_stream_linear(a, (cudaStream_t)stream) : umma_i8_linear(a, (cudaStream_t)stream);
}

}  // extern "C"

namespace {
// Workspace of an expert layer in its grouped form, part by part.
// Each expert's output for each of its rows: in fp32 for decode batches, where it costs nothing (16 tokens, 128 experts of 2048 x 768, top-8: 85 us either way), so that
// their results are the one-kernel form's, bit for bit; beyond, in 16 bits of act_dtype (256 tokens 127 us, in fp32 137; bf16 error against
// 64 bits 2.3e-3 of the norm, in fp32 1.7e-3), but for outputs that those cannot hold, which the weighted sum makes anew.
bool moe_y_f32(size_t elements) { return elements <= (size_t)1 << 19; }

struct MoeParts {
  uint8_t *weights, *ids, *place, *rows, *base, *offsets, *count, *tiles, *xq, *xs, *h, *hq, *hs, *y;
  size_t total;
};
MoeParts moe_parts(void* ws, int64_t T, int E, int k, int64_t H, int64_t I) {
  MoeParts p{};
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  size_t at = 0;
  auto take = [&](size_t bytes) { uint8_t* q = base + at; at += align_up(bytes, 256); return q; };
  const size_t rows = (size_t)T * k;
  p.weights = take(rows * 4); p.ids = take(rows * 4); p.place = take(rows * 4); p.rows = take(rows * 4);
  p.base = take((size_t)moe_i8_route_ctas(T) * E * 4); p.offsets = take((size_t)(E + 1) * 4); p.count = take(8);
  p.tiles = take(16 + 8 * (rows / 32 + 1 + E));
  p.xq = take(rows * H); p.xs = take(rows * 4); p.h = take(rows * I * 4); p.hq = take(rows * I); p.hs = take(rows * 4); p.y = take(rows * H * (moe_y_f32(rows * H) ? 4 : 2));
  p.total = at;
  return p;
}
}  // namespace

extern "C" {

size_t b2q_moe_forward_int8_workspace_bytes(int64_t T, int64_t E, int64_t top_k, int64_t H, int64_t I) {
  if (T <= 0 || E <= 0 || E > 1024 || top_k <= 0 || top_k > 32 || H <= 0 || I <= 0 || T > INT32_MAX / 32) return 0;
  if (use_few(T, E, top_k, H, I)) return moe_i8_few_bytes(T, top_k, I);
  return moe_parts(nullptr, T, (int)E, (int)top_k, H, I).total;
}

int b2q_moe_forward_int8(const b2q_moe_int8* m, void* workspace, size_t workspace_bytes, void* stream) {
  if (!m) return B2Q_ERR_NULL;
  const b2q_moe_int8& a = *m;
  if (!a.x || !a.logits || !a.w13 || !a.s13 || !a.w2 || !a.s2 || !a.out) return B2Q_ERR_NULL;
  if (!is16(a.act_dtype) || !known(a.logits_dtype) || !known(a.s13_dtype) || !known(a.s2_dtype)) return B2Q_ERR_DTYPE;
  if (a.T < 0 || a.E <= 0 || a.top_k <= 0 || a.top_k > a.E || a.H <= 0 || a.I <= 0 || a.H % 16 != 0 || a.I % 16 != 0) return B2Q_ERR_SHAPE;
  if (a.E > 1024 || a.top_k > 32 || a.H > 32768 || a.I > MAX_K || a.T > INT32_MAX / 32 || 2 * a.E * a.I > INT32_MAX || a.E * a.H > INT32_MAX) return B2Q_ERR_LIMIT;
  if (!aligned16(a.x) || !aligned16(a.w13) || !aligned16(a.w2) || !aligned16(a.out) || !aligned_to(a.logits, dtype_bytes(a.logits_dtype)) ||
      !aligned_to(a.s13, dtype_bytes(a.s13_dtype)) || !aligned_to(a.s2, dtype_bytes(a.s2_dtype)))
    return B2Q_ERR_ALIGN;
  if (a.T == 0) return B2Q_OK;
  if (!workspace) return B2Q_ERR_NULL;
  if (!aligned_to(workspace, 256)) return B2Q_ERR_ALIGN;
  if (workspace_bytes < b2q_moe_forward_int8_workspace_bytes(a.T, a.E, a.top_k, a.H, a.I)) return B2Q_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf16 = a.act_dtype == B2Q_BF16;
  const int E = (int)a.E, k = (int)a.top_k, H = (int)a.H, I = (int)a.I;
  if (use_few(a.T, E, k, H, I)) {
    I8FewArgs f{};
    f.x = a.x; f.bf16 = bf16; f.logits = a.logits; f.logits_dtype = a.logits_dtype;
    f.w13 = a.w13; f.s13 = a.s13; f.s13_dtype = a.s13_dtype; f.w2 = a.w2; f.s2 = a.s2; f.s2_dtype = a.s2_dtype;
    f.out = a.out; f.T = (int)a.T; f.E = E; f.k = k; f.H = H; f.I = I; f.renorm = a.renormalize != 0; f.scratch = workspace;
    return moe_i8_few(f, st);
  }
  const MoeParts p = moe_parts(workspace, a.T, E, k, H, I);
  const int64_t rows = a.T * k;
  int32_t *off = reinterpret_cast<int32_t*>(p.offsets), *tiles = reinterpret_cast<int32_t*>(p.tiles), *out_rows = reinterpret_cast<int32_t*>(p.rows);
  const int tile = i8_grouped_tile(rows, E), ctas = moe_i8_route_ctas(a.T);
  I8Copies to{};
  to.ids = reinterpret_cast<int32_t*>(p.ids); to.place = reinterpret_cast<int32_t*>(p.place); to.base = reinterpret_cast<int32_t*>(p.base);
  to.rows = out_rows; to.k = k; to.E = E; to.run = (int)((a.T + ctas - 1) / ctas);
  int rc = moe_i8_route(a.logits, a.logits_dtype, a.T, E, k, a.renormalize != 0, tile, reinterpret_cast<float*>(p.weights), reinterpret_cast<int32_t*>(p.ids),
                        reinterpret_cast<int32_t*>(p.place), reinterpret_cast<int32_t*>(p.base), off, tiles, p.count, st);
  if (rc) return rc;
  I8GroupedArgs g{};
  g.xq = reinterpret_cast<int8_t*>(p.xq); g.xs = reinterpret_cast<float*>(p.xs); g.w = a.w13; g.ws = a.s13; g.ws_dtype = a.s13_dtype;
  g.offsets = off; g.tiles = tiles; g.tile = tile; g.tile_cap = (int)((rows + tile - 1) / tile + E); g.E = E;
  g.out = p.h; g.out_bf16 = bf16; g.rows = (int)rows; g.N = I; g.K = H; g.gated = true;
  I8GroupedArgs d = g;
  d.xq = reinterpret_cast<int8_t*>(p.hq); d.xs = reinterpret_cast<float*>(p.hs); d.w = a.w2; d.ws = a.s2; d.ws_dtype = a.s2_dtype;
  d.out = p.y; d.out_f32 = moe_y_f32((size_t)rows * H); d.N = H; d.K = I; d.gated = false;
  rc = quantize_i8_copies(a.x, bf16, to, reinterpret_cast<int8_t*>(p.xq), reinterpret_cast<float*>(p.xs), a.T, H, st);
  if (!rc) rc = umma_i8_grouped(g, st);
  if (!rc) rc = quantize_i8_computed(reinterpret_cast<float*>(p.h), off + E, reinterpret_cast<int8_t*>(p.hq), reinterpret_cast<float*>(p.hs), rows, I, st);
  if (!rc) rc = umma_i8_grouped(d, st);
  const I8Outputs of{d.xq, d.xs, d.w, d.ws, d.ws_dtype, to.ids, I};
  if (!rc) rc = moe_i8_sum(p.y, d.out_f32, reinterpret_cast<float*>(p.weights), out_rows, of, a.out, bf16, a.T, k, H, st);
  return rc;
}

}  // extern "C"
