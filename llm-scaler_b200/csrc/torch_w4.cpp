// torch ops of expert routing and the 4-bit group-quantised layers, straight over the C ABI of include/b2q.h.  They have no counterpart in the reference and so
// a namespace of their own, b2q_w4; the Python package gives them their public names (custom_esimd_kernels_vllm/w4.py).
// Built by build.py into custom_esimd_kernels_vllm/libb2q_w4.so, which links libb2q.so and libtorch.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "b2q.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

int dtype_of(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return B2Q_BF16;
  if (t.scalar_type() == at::kHalf) return B2Q_F16;
  if (t.scalar_type() == at::kFloat) return B2Q_F32;
  TORCH_CHECK(false, "b2q: unsupported dtype ", t.scalar_type());
}
bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
// Messages are made of strings alone: see build.py, build_torch_ops.
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
// a new tensor on x's device, which is current: without the dispatcher, whose hop is a tenth of what a small call costs
Tensor fresh(const Tensor& x, at::IntArrayRef size, at::ScalarType type) { return at::detail::empty_cuda(size, type, x.device(), c10::nullopt); }

// A 4-bit weight of [..experts, N, K]: codes as uint8 [.., N, K / 2] or int32 [.., N, K / 8].  Its group, from the scales' [.., K / group, N].
struct Weight { int64_t N, K, group; const uint8_t* w; const void* s; const uint8_t* z; };
Weight weight_of(const char* name, const Tensor& x, const Tensor& w, const Tensor& s, const OptTensor& z, int64_t experts) {
  same_device({&x, &w, &s});
  const int64_t d = experts >= 0 ? 1 : 0;
  TORCH_CHECK(w.scalar_type() == at::kByte || w.scalar_type() == at::kInt, name, " weight must be uint8 (two codes to a byte) or int32 (eight)");
  TORCH_CHECK(w.dim() == 2 + d && w.is_contiguous(), name, " weight must be a contiguous ", d ? "[E, N, K / 2]" : "[N, K / 2]", " tensor (int32: K / 8)");
  Weight r{};
  r.N = w.size(d);
  r.K = w.size(d + 1) * (w.scalar_type() == at::kByte ? 2 : 8);
  TORCH_CHECK(s.scalar_type() == x.scalar_type(), name, " scale must have the activations' type");
  TORCH_CHECK(s.dim() == 2 + d && s.is_contiguous() && s.size(d + 1) == r.N && s.size(d) > 0, name, " scale must be a contiguous ", d ? "[E, K / group, N]" : "[K / group, N]",
              " tensor");
  TORCH_CHECK(r.K > 0 && r.K % s.size(d) == 0, name, " scale has a number of groups that does not divide K");
  r.group = r.K / s.size(d);
  TORCH_CHECK(r.group == 32 || r.group == 64 || r.group == 128, name, " groups must have 32, 64 or 128 values");
  if (d) TORCH_CHECK(w.size(0) == experts && s.size(0) == experts, name, " weight and scale must have the same number of experts");
  if (z.has_value()) {
    same_device({&x, &*z});
    TORCH_CHECK(z->scalar_type() == at::kByte && z->is_contiguous() && z->sizes() == s.sizes(), name, " zero must be contiguous uint8 of the scale's shape");
    r.z = z->data_ptr<uint8_t>();
  }
  r.w = reinterpret_cast<const uint8_t*>(w.data_ptr());
  r.s = s.data_ptr();
  return r;
}

// scoring, group_score: B2Q_SCORE_*, B2Q_GROUP_* (a string takes longer through the dispatcher than a small call)
std::tuple<Tensor, Tensor> route_experts(const Tensor& logits, int64_t top_k, int64_t scoring, const OptTensor& bias, int64_t num_groups, int64_t top_groups,
                                         int64_t group_score, bool renormalize, double scale) {
  same_device({&logits});
  check_rows(logits, "logits");
  const int dt = dtype_of(logits);
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(scoring == B2Q_SCORE_SOFTMAX || scoring == B2Q_SCORE_SIGMOID, "scoring must be 0 (softmax) or 1 (sigmoid)");
  TORCH_CHECK(group_score == B2Q_GROUP_MAX || group_score == B2Q_GROUP_TOP2, "group_score must be 0 (max) or 1 (top2)");
  TORCH_CHECK(E > 0 && num_groups > 0 && E % num_groups == 0, "num_groups must divide the number of experts");
  TORCH_CHECK(top_groups > 0 && top_groups <= num_groups, "top_groups must be between 1 and num_groups");
  TORCH_CHECK(top_k > 0 && top_k <= E / num_groups * top_groups, "top_k must be between 1 and the number of experts in top_groups groups");
  if (bias.has_value()) {
    same_device({&logits, &*bias});
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == E && bias->is_contiguous(), "bias must be a contiguous [E] tensor");
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  Tensor w = fresh(logits, {T, top_k}, at::kFloat), ids = fresh(logits, {T, top_k}, at::kInt);
  if (T > 0)
    check(b2q_route_experts(logits.data_ptr(), dt, pitch(logits), bias.has_value() ? bias->data_ptr() : nullptr, bias.has_value() ? dtype_of(*bias) : 0, w.data_ptr<float>(),
                            ids.data_ptr<int32_t>(), T, E, top_k, (int)scoring, num_groups, top_groups, (int)group_score, renormalize, (float)scale, stream_of(logits)));
  return {w, ids};
}

Tensor linear(const Tensor& x, const Tensor& weight, const Tensor& scale, const OptTensor& zero, const OptTensor& bias) {
  same_device({&x, &weight, &scale});
  check_rows(x, "x");
  TORCH_CHECK(is16(x.scalar_type()), "x must be bf16 or fp16");
  const Weight w = weight_of("the", x, weight, scale, zero, -1);
  const int64_t M = x.size(0);
  TORCH_CHECK(x.size(1) == w.K, "weight has another K than x");
  if (bias.has_value()) {
    same_device({&x, &*bias});
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.N && bias->is_contiguous() && bias->scalar_type() == x.scalar_type(), "bias must be a contiguous [N] tensor of x's type");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = fresh(x, {M, w.N}, x.scalar_type()), ws;
  if (M > 0 && w.N > 0) {
    const size_t wsb = b2q_linear_w4_workspace_bytes(M, w.N, w.K, w.group);
    if (wsb) ws = fresh(x, {(int64_t)wsb}, at::kByte);
    check(b2q_linear_w4(x.data_ptr(), dtype_of(x), pitch(x), w.w, w.s, w.z, bias.has_value() ? bias->data_ptr() : nullptr, out.data_ptr(), w.N, M, w.N, w.K, w.group,
                        wsb ? ws.data_ptr() : nullptr, wsb, stream_of(x)));
  }
  return out;
}

Tensor moe_forward(const Tensor& x, const Tensor& topk_weights, const Tensor& topk_ids, const Tensor& w13, const Tensor& s13, const Tensor& w2, const Tensor& s2,
                   const OptTensor& z13, const OptTensor& z2) {
  same_device({&x, &topk_weights, &topk_ids, &w13, &s13, &w2, &s2});
  TORCH_CHECK(x.dim() == 2 && is16(x.scalar_type()) && x.is_contiguous(), "x must be a contiguous bf16 / fp16 [T, H] tensor");
  const int64_t T = x.size(0), H = x.size(1);
  TORCH_CHECK(topk_ids.dim() == 2 && topk_ids.size(0) == T && topk_ids.size(1) > 0 && topk_ids.scalar_type() == at::kInt && topk_ids.is_contiguous(),
              "topk_ids must be a contiguous int32 [T, top_k] tensor");
  TORCH_CHECK(topk_weights.sizes() == topk_ids.sizes() && topk_weights.scalar_type() == at::kFloat && topk_weights.is_contiguous(),
              "topk_weights must be a contiguous fp32 tensor of the shape of topk_ids");
  TORCH_CHECK(w13.dim() == 3, "the gate_up weight must be a contiguous [E, N, K / 2] tensor (int32: K / 8)");
  const int64_t E = w13.size(0);
  TORCH_CHECK(E > 0, "there are no experts");
  const Weight u = weight_of("the gate_up", x, w13, s13, z13, E), d = weight_of("the down", x, w2, s2, z2, E);
  TORCH_CHECK(u.K == H && u.N % 2 == 0, "the gate_up weight must be of [E, 2I, H]");
  TORCH_CHECK(d.N == H && d.K == u.N / 2, "the down weight must be of [E, H, I]");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = fresh(x, {T, H}, x.scalar_type());
  if (T == 0) return out;
  b2q_moe_w4 a{};
  a.x = x.data_ptr(); a.weights = topk_weights.data_ptr<float>(); a.ids = topk_ids.data_ptr<int32_t>();
  a.w13 = u.w; a.s13 = u.s; a.z13 = u.z; a.w2 = d.w; a.s2 = d.s; a.z2 = d.z; a.out = out.data_ptr();
  a.T = T; a.E = E; a.top_k = topk_ids.size(1); a.H = H; a.I = d.K; a.group13 = u.group; a.group2 = d.group; a.act_dtype = dtype_of(x);
  const size_t wsb = b2q_moe_forward_w4_workspace_bytes(T, E, a.top_k, H, a.I);
  const Tensor ws = fresh(x, {(int64_t)wsb}, at::kByte);
  check(b2q_moe_forward_w4(&a, ws.data_ptr(), wsb, stream_of(x)));
  return out;
}

}  // namespace

TORCH_LIBRARY(b2q_w4, m) {
  m.def("route_experts(Tensor logits, int top_k, int scoring, Tensor? bias, int num_groups, int top_groups, int group_score, bool renormalize, float scale) -> (Tensor, Tensor)");
  m.def("linear(Tensor x, Tensor weight, Tensor scale, Tensor? zero, Tensor? bias) -> Tensor");
  m.def("moe_forward(Tensor x, Tensor topk_weights, Tensor topk_ids, Tensor gate_up_weight, Tensor gate_up_scale, Tensor down_weight, Tensor down_scale, "
        "Tensor? gate_up_zero, Tensor? down_zero) -> Tensor");
}

TORCH_LIBRARY_IMPL(b2q_w4, CUDA, m) {
  m.impl("route_experts", &route_experts);
  m.impl("linear", &linear);
  m.impl("moe_forward", &moe_forward);
}
