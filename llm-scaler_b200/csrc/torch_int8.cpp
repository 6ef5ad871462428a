// torch ops of the 8-bit integer operators, straight over the C ABI of include/b2q.h.  They have no counterpart in the reference and so
// a namespace of their own, b2q_int8; the Python package gives them their public names (custom_esimd_kernels_vllm/int8.py).
// Built by build.py into custom_esimd_kernels_vllm/libb2q_int8.so, which links libb2q.so and libtorch.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "b2q.h"

namespace {

using at::Tensor;

int dtype_of(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return B2Q_BF16;
  if (t.scalar_type() == at::kHalf) return B2Q_F16;
  if (t.scalar_type() == at::kFloat) return B2Q_F32;
  TORCH_CHECK(false, "b2q: unsupported dtype ", t.scalar_type());
}
bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
void check(int rc) { TORCH_CHECK(rc == 0, b2q_strerror(rc)); }

// all on one CUDA device, that of the first
void same_device(std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  for (const Tensor* t : ts) {
    TORCH_CHECK(t->is_cuda(), "b2q: tensor must live on a CUDA device (no CPU path exists)");
    TORCH_CHECK(t->device() == first.device(), "b2q: tensors live on different devices");
  }
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void check_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have contiguous rows");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " has rows that overlap");
}
void check_weight(const Tensor& w, const Tensor& s, int64_t K) {
  TORCH_CHECK(w.dim() == 2 && w.scalar_type() == at::kChar && w.is_contiguous(), "weight must be a contiguous int8 [N, K] tensor");
  TORCH_CHECK(w.size(1) == K, "weight has another K than the activations");
  TORCH_CHECK(K % 16 == 0, "K must be a multiple of 16");
  TORCH_CHECK(s.dim() <= 2 && s.numel() == w.size(0) && s.is_contiguous(), "weight_scale must have N contiguous elements");
}
const void* check_bias(const c10::optional<Tensor>& bias, const Tensor& w, at::ScalarType out) {
  if (!bias.has_value()) return nullptr;
  same_device({&w, &*bias});
  TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.size(0) && bias->is_contiguous() && bias->scalar_type() == out,
              "bias must be a contiguous [N] tensor of the output type");
  return bias->data_ptr();
}
// a new tensor on x's device, which is current: without the dispatcher, whose hop is a tenth of what a small call costs
Tensor fresh(const Tensor& x, at::IntArrayRef size, at::ScalarType type) { return at::detail::empty_cuda(size, type, x.device(), c10::nullopt); }
Tensor codes_like(const Tensor& x, int64_t M, int64_t K) { return fresh(x, {M, K}, at::kChar); }
Tensor scales_like(const Tensor& x, int64_t M) { return fresh(x, {M}, at::kFloat); }

std::tuple<Tensor, Tensor> quantize(const Tensor& x) {
  same_device({&x});
  check_rows(x, "x");
  const int dt = dtype_of(x);
  const int64_t M = x.size(0), K = x.size(1);
  TORCH_CHECK(K > 0, "x has no columns");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor q = codes_like(x, M, K), s = scales_like(x, M);
  if (M > 0) check(b2q_quantize_int8(x.data_ptr(), dt, pitch(x), q.data_ptr<int8_t>(), s.data_ptr<float>(), M, K, stream_of(x)));
  return {q, s};
}

std::tuple<Tensor, Tensor> silu_mul_quantize(const Tensor& gate_up) {
  same_device({&gate_up});
  check_rows(gate_up, "gate_up");
  TORCH_CHECK(is16(gate_up.scalar_type()), "gate_up must be bf16 or fp16");
  TORCH_CHECK(gate_up.size(1) > 0 && gate_up.size(1) % 2 == 0, "gate_up must have an even number of columns: gate, then up");
  const int64_t M = gate_up.size(0), K = gate_up.size(1) / 2;
  const c10::cuda::CUDAGuard guard(gate_up.device());
  Tensor q = codes_like(gate_up, M, K), s = scales_like(gate_up, M);
  if (M > 0)
    check(b2q_silu_mul_quantize_int8(gate_up.data_ptr(), dtype_of(gate_up), pitch(gate_up), q.data_ptr<int8_t>(), s.data_ptr<float>(), M, K,
                                     stream_of(gate_up)));
  return {q, s};
}

std::tuple<Tensor, Tensor> resadd_rmsnorm_quantize(const Tensor& hidden, Tensor residual, const Tensor& norm_weight, double eps,
                                                   const c10::optional<Tensor>& residual_out) {
  const Tensor& out = residual_out.has_value() ? *residual_out : residual;
  same_device({&hidden, &residual, &norm_weight, &out});
  TORCH_CHECK(hidden.dim() == 2 && is16(hidden.scalar_type()), "hidden must be 2-D bf16 / fp16");
  const int64_t M = hidden.size(0), K = hidden.size(1);
  TORCH_CHECK(K > 0, "hidden has no columns");
  const Tensor* const same[] = {&hidden, &residual, &out};
  const char* const names[] = {"hidden", "residual", "residual_out"};
  for (int i = 0; i < 3; ++i)
    TORCH_CHECK(same[i]->scalar_type() == hidden.scalar_type() && same[i]->dim() == 2 && same[i]->size(0) == M && same[i]->size(1) == K &&
                    same[i]->is_contiguous(), names[i], " must be a contiguous [M, K] tensor of the activation type");
  TORCH_CHECK(norm_weight.scalar_type() == hidden.scalar_type() && norm_weight.dim() == 1 && norm_weight.size(0) == K && norm_weight.is_contiguous(),
              "norm_weight must be a contiguous [K] tensor of the activation type");
  const c10::cuda::CUDAGuard guard(hidden.device());
  Tensor q = codes_like(hidden, M, K), s = scales_like(hidden, M);
  if (M > 0)
    check(b2q_resadd_rmsnorm_quantize_int8(hidden.data_ptr(), residual.data_ptr(), norm_weight.data_ptr(), out.data_ptr(), dtype_of(hidden), (float)eps,
                                           q.data_ptr<int8_t>(), s.data_ptr<float>(), M, K, stream_of(hidden)));
  return {q, s};
}

Tensor linear(const Tensor& codes, const Tensor& scale, const Tensor& weight, const Tensor& weight_scale, const c10::optional<Tensor>& bias,
              at::ScalarType out_dtype) {
  same_device({&codes, &scale, &weight, &weight_scale});
  check_rows(codes, "codes");
  TORCH_CHECK(codes.scalar_type() == at::kChar, "codes must be int8");
  TORCH_CHECK(is16(out_dtype), "out_dtype must be bf16 or fp16");
  const int64_t M = codes.size(0), K = codes.size(1), N = weight.dim() == 2 ? weight.size(0) : 0;
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.dim() <= 2 && scale.numel() == M && scale.is_contiguous(), "scale must be fp32 with M contiguous elements");
  check_weight(weight, weight_scale, K);
  const void* b = check_bias(bias, weight, out_dtype);
  const c10::cuda::CUDAGuard guard(codes.device());
  Tensor out = fresh(codes, {M, N}, out_dtype);
  if (M > 0 && N > 0)
    check(b2q_linear_int8(codes.data_ptr<int8_t>(), pitch(codes), scale.data_ptr<float>(), weight.data_ptr<int8_t>(), weight_scale.data_ptr(),
                          dtype_of(weight_scale), b, out.data_ptr(), dtype_of(out), N, M, N, K, stream_of(codes)));
  return out;
}

Tensor linear_dynamic(const Tensor& x, const Tensor& weight, const Tensor& weight_scale, const c10::optional<Tensor>& bias) {
  same_device({&x, &weight, &weight_scale});
  check_rows(x, "x");
  TORCH_CHECK(is16(x.scalar_type()), "x must be bf16 or fp16");
  const int64_t M = x.size(0), K = x.size(1), N = weight.dim() == 2 ? weight.size(0) : 0;
  check_weight(weight, weight_scale, K);
  const void* b = check_bias(bias, weight, x.scalar_type());
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = fresh(x, {M, N}, x.scalar_type()), ws;
  if (M > 0 && N > 0) {
    const size_t wsb = b2q_linear_int8_dynamic_workspace_bytes(M, N, K);
    if (wsb) ws = fresh(x, {(int64_t)wsb}, at::kByte);
    check(b2q_linear_int8_dynamic(x.data_ptr(), dtype_of(x), pitch(x), weight.data_ptr<int8_t>(), weight_scale.data_ptr(), dtype_of(weight_scale), b,
                                  out.data_ptr(), N, M, N, K, wsb ? ws.data_ptr() : nullptr, wsb, stream_of(x)));
  }
  return out;
}

Tensor moe_forward(const Tensor& x, const Tensor& logits, const Tensor& w13, const Tensor& s13, const Tensor& w2, const Tensor& s2, int64_t top_k,
                   bool renormalize) {
  same_device({&x, &logits, &w13, &s13, &w2, &s2});
  TORCH_CHECK(x.dim() == 2 && is16(x.scalar_type()) && x.is_contiguous(), "x must be a contiguous bf16 / fp16 [T, H] tensor");
  TORCH_CHECK(logits.dim() == 2 && logits.size(0) == x.size(0) && logits.is_contiguous(), "router_logits must be a contiguous [T, E] tensor");
  const int64_t T = x.size(0), H = x.size(1), E = logits.size(1);
  TORCH_CHECK(w13.dim() == 3 && w13.scalar_type() == at::kChar && w13.is_contiguous() && w13.size(0) == E && w13.size(2) == H && w13.size(1) % 2 == 0,
              "gate_up_weight must be a contiguous int8 [E, 2I, H] tensor");
  const int64_t I = w13.size(1) / 2;
  TORCH_CHECK(w2.dim() == 3 && w2.scalar_type() == at::kChar && w2.is_contiguous() && w2.size(0) == E && w2.size(1) == H && w2.size(2) == I,
              "down_weight must be a contiguous int8 [E, H, I] tensor");
  TORCH_CHECK(s13.numel() == E * 2 * I && s13.is_contiguous(), "gate_up_scale must have E * 2I contiguous elements");
  TORCH_CHECK(s2.numel() == E * H && s2.is_contiguous(), "down_scale must have E * H contiguous elements");
  TORCH_CHECK(top_k > 0 && top_k <= E, "top_k must be between 1 and the number of experts");
  TORCH_CHECK(H > 0 && I > 0 && H % 16 == 0 && I % 16 == 0, "H and I must be multiples of 16");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = fresh(x, {T, H}, x.scalar_type());
  if (T == 0) return out;
  b2q_moe_int8 a{};
  a.x = x.data_ptr(); a.logits = logits.data_ptr(); a.w13 = w13.data_ptr<int8_t>(); a.s13 = s13.data_ptr(); a.w2 = w2.data_ptr<int8_t>(); a.s2 = s2.data_ptr();
  a.out = out.data_ptr(); a.T = T; a.E = E; a.top_k = top_k; a.H = H; a.I = I;
  a.act_dtype = dtype_of(x); a.logits_dtype = dtype_of(logits); a.s13_dtype = dtype_of(s13); a.s2_dtype = dtype_of(s2); a.renormalize = renormalize;
  const size_t wsb = b2q_moe_forward_int8_workspace_bytes(T, E, top_k, H, I);
  const Tensor ws = fresh(x, {(int64_t)wsb}, at::kByte);
  check(b2q_moe_forward_int8(&a, ws.data_ptr(), wsb, stream_of(x)));
  return out;
}

}  // namespace

TORCH_LIBRARY(b2q_int8, m) {
  m.def("quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("silu_mul_quantize(Tensor gate_up) -> (Tensor, Tensor)");
  m.def("resadd_rmsnorm_quantize(Tensor hidden, Tensor(a!) residual, Tensor norm_weight, float eps, Tensor(b!)? residual_out) -> (Tensor, Tensor)");
  m.def("linear(Tensor codes, Tensor scale, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType out_dtype) -> Tensor");
  m.def("linear_dynamic(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias) -> Tensor");
  m.def("moe_forward(Tensor x, Tensor router_logits, Tensor gate_up_weight, Tensor gate_up_scale, Tensor down_weight, Tensor down_scale, "
        "int top_k, bool renormalize) -> Tensor");
}

TORCH_LIBRARY_IMPL(b2q_int8, CUDA, m) {
  m.impl("quantize", &quantize);
  m.impl("silu_mul_quantize", &silu_mul_quantize);
  m.impl("resadd_rmsnorm_quantize", &resadd_rmsnorm_quantize);
  m.impl("linear", &linear);
  m.impl("linear_dynamic", &linear_dynamic);
  m.impl("moe_forward", &moe_forward);
}
