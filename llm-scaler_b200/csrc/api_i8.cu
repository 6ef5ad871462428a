// C ABI of the 8-bit integer operators: argument validation and kernel selection, as in api.cu.
#include "i8.cuh"

using namespace b2q;

namespace {
bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool known(int dtype) { return dtype >= 0 && dtype <= 2; }
size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
constexpr int64_t MAX_K = 131071;                          // 128 * 128 * K stays below 2^31

int linear_check(const I8LinearArgs& a, int64_t M, int64_t N, int64_t K) {
  if (!a.w || !a.ws || !a.out) return B2Q_ERR_NULL;
  if (!known(a.ws_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || N < 0 || K <= 0 || K % 16 != 0 || a.ldo < N) return B2Q_ERR_SHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > MAX_K) return B2Q_ERR_LIMIT;
  if (!aligned16(a.w) || !aligned_to(a.out, 2) || !aligned_to(a.bias, 2) || !aligned_to(a.ws, dtype_bytes(a.ws_dtype))) return B2Q_ERR_ALIGN;
  return B2Q_OK;
}
}  // namespace

extern "C" {

int b2q_quantize_int8(const void* x, int x_dtype, int64_t ldx, int8_t* q, float* scale, int64_t M, int64_t K, void* stream) {
  if (!x || !q || !scale) return B2Q_ERR_NULL;
  if (!known(x_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || K <= 0 || ldx < K) return B2Q_ERR_SHAPE;
  if (M > INT32_MAX || K > INT32_MAX) return B2Q_ERR_LIMIT;
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
  if (M > INT32_MAX || K > INT32_MAX) return B2Q_ERR_LIMIT;
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
  return M <= I8_STREAM_MAX_TOK ? i8_stream_linear(a, (cudaStream_t)stream) : umma_i8_linear(a, (cudaStream_t)stream);
}

size_t b2q_linear_int8_dynamic_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  // also where one launch does without: rows that are not 16-byte aligned go through the quantiser whatever their number
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
  if (i8_stream_supported(a)) return i8_stream_linear(a, (cudaStream_t)stream);
  if (!workspace) return B2Q_ERR_NULL;
  if (!aligned16(workspace)) return B2Q_ERR_ALIGN;
  if (workspace_bytes < b2q_linear_int8_dynamic_workspace_bytes(M, N, K)) return B2Q_ERR_WORKSPACE;
  int8_t* q = reinterpret_cast<int8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + align_up((size_t)M * (size_t)K, 256));
  rc = quantize_i8(x, act_dtype, ldx, q, s, M, (int)K, (cudaStream_t)stream);
  if (rc) return rc;
  a.x16 = nullptr; a.xq = q; a.ldx = K; a.xs = s;
  return M <= I8_STREAM_MAX_TOK ? i8_stream_linear(a, (cudaStream_t)stream) : umma_i8_linear(a, (cudaStream_t)stream);
}

}  // extern "C"
