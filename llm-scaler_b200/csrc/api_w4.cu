// C ABI of expert routing and the layers of 4-bit group-quantised weights: argument validation and kernel selection, as in api.cu.
#include "g4.cuh"

using namespace b2q;

namespace {
bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool known(int dtype) { return dtype >= 0 && dtype <= 2; }
bool is_group(int64_t g) { return g == 32 || g == 64 || g == 128; }
constexpr int64_t MAX_ROWS = INT32_MAX - 4096;             // tokens and weight rows: rounded up to tiles and rounds of tiles, both below this
constexpr int64_t MAX_K = 1 << 20;
// set_force_kernel(2): tcgen05 for everything
bool use_stream(int64_t M, int64_t N, int64_t K, int64_t group) { return tls().force_kernel != 2 && g4_stream_preferred((int)M, (int)N, (int)K, (int)group); }
bool use_few(const G4MoeArgs& a) { return tls().force_kernel != 2 && moe_g4_few_preferred(a); }
}  // namespace

extern "C" {

int b2q_route_experts(const void* logits, int logits_dtype, int64_t ldl, const void* bias, int bias_dtype, float* weights, int32_t* ids, int64_t T, int64_t E,
                      int64_t top_k, int scoring, int64_t num_groups, int64_t top_groups, int group_score, int renormalize, float scale, void* stream) {
  if (!logits || !weights || !ids) return B2Q_ERR_NULL;
  if (!known(logits_dtype) || (bias && !known(bias_dtype))) return B2Q_ERR_DTYPE;
  if (scoring != B2Q_SCORE_SOFTMAX && scoring != B2Q_SCORE_SIGMOID) return B2Q_ERR_LAYOUT;
  if (group_score != B2Q_GROUP_MAX && group_score != B2Q_GROUP_TOP2) return B2Q_ERR_LAYOUT;
  if (T < 0 || E <= 0 || top_k <= 0 || ldl < E || num_groups <= 0 || top_groups <= 0 || top_groups > num_groups || E % num_groups != 0) return B2Q_ERR_SHAPE;
  if (E > 1024 || top_k > 32 || num_groups > 32 || T > MAX_ROWS) return B2Q_ERR_LIMIT;
  if (top_k > E / num_groups * top_groups) return B2Q_ERR_SHAPE;
  if (!aligned_to(logits, dtype_bytes(logits_dtype)) || (bias && !aligned_to(bias, dtype_bytes(bias_dtype))) || !aligned_to(weights, 4) || !aligned_to(ids, 4)) return B2Q_ERR_ALIGN;
  if (T == 0) return B2Q_OK;
  RouteExpertsArgs a{};
  a.logits = logits; a.dtype = logits_dtype; a.ldl = ldl; a.bias = bias; a.bias_dtype = bias_dtype; a.weights = weights; a.ids = ids;
  a.T = (int)T; a.E = (int)E; a.k = (int)top_k; a.groups = (int)num_groups; a.top_groups = (int)top_groups;
  a.sigmoid = scoring == B2Q_SCORE_SIGMOID; a.top2 = group_score == B2Q_GROUP_TOP2; a.renorm = renormalize != 0; a.scale = scale;
  return route_experts(a, (cudaStream_t)stream);
}

size_t b2q_linear_w4_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t group) {
  if (M <= 0 || N <= 0 || K <= 0 || !is_group(group) || K % group != 0 || M > MAX_ROWS || N > MAX_ROWS || K > MAX_K) return 0;
  if (use_stream(M, N, K, group)) return g4_stream_bytes((int)M, (int)N, (int)K, (int)group);
  return umma_g4_bytes(nullptr, 0, (int)M, (int)N, (int)K, (int)group);
}

int b2q_linear_w4(const void* x, int act_dtype, int64_t ldx, const uint8_t* w, const void* scale, const uint8_t* zero, const void* bias, void* out, int64_t ldo, int64_t M,
                  int64_t N, int64_t K, int64_t group, void* workspace, size_t workspace_bytes, void* stream) {
  if (!x || !w || !scale || !out) return B2Q_ERR_NULL;
  if (!is16(act_dtype)) return B2Q_ERR_DTYPE;
  if (M < 0 || N < 0 || K <= 0 || !is_group(group) || K % group != 0 || ldx < K || ldo < N) return B2Q_ERR_SHAPE;
  if (M > MAX_ROWS || N > MAX_ROWS || K > MAX_K || N > INT32_MAX / (K / group)) return B2Q_ERR_LIMIT;
  if (!aligned16(w) || !aligned_to(x, 2) || !aligned_to(scale, 2) || !aligned_to(bias, 2) || !aligned_to(out, 2)) return B2Q_ERR_ALIGN;
  if (M == 0 || N == 0) return B2Q_OK;
  const size_t need = b2q_linear_w4_workspace_bytes(M, N, K, group);
  if (need) {
    if (!workspace) return B2Q_ERR_NULL;
    if (!aligned_to(workspace, 256)) return B2Q_ERR_ALIGN;
    if (workspace_bytes < need) return B2Q_ERR_WORKSPACE;
  }
  G4LinearArgs a{};
  a.x = x; a.ldx = ldx; a.bf16 = act_dtype == B2Q_BF16; a.w = w; a.scale = scale; a.zero = zero; a.bias = bias; a.out = out; a.ldo = ldo;
  a.M = (int)M; a.N = (int)N; a.K = (int)K; a.G = (int)group;
  if (use_stream(M, N, K, group)) return g4_stream_linear(a, workspace, (cudaStream_t)stream);
  return umma_g4_linear(a, workspace, (cudaStream_t)stream);
}

size_t b2q_moe_forward_w4_workspace_bytes(int64_t T, int64_t E, int64_t top_k, int64_t H, int64_t I) {
  if (T <= 0 || E <= 0 || E > 1024 || top_k <= 0 || top_k > 32 || H <= 0 || I <= 0 || H > MAX_K || I > MAX_K || T > INT32_MAX / 32) return 0;
  G4MoeArgs g{};
  g.T = (int)T; g.E = (int)E; g.k = (int)top_k; g.H = (int)H; g.I = (int)I;
  const size_t few = moe_g4_few_bytes(g), many = moe_g4_many_bytes(g);      // which form a few tokens get depends on the groups too
  return few > many ? few : many;
}

int b2q_moe_forward_w4(const b2q_moe_w4* m, void* workspace, size_t workspace_bytes, void* stream) {
  if (!m) return B2Q_ERR_NULL;
  const b2q_moe_w4& a = *m;
  if (!a.x || !a.weights || !a.ids || !a.w13 || !a.s13 || !a.w2 || !a.s2 || !a.out) return B2Q_ERR_NULL;
  if (!is16(a.act_dtype)) return B2Q_ERR_DTYPE;
  if (a.T < 0 || a.E <= 0 || a.top_k <= 0 || a.H <= 0 || a.I <= 0 || !is_group(a.group13) || !is_group(a.group2) || a.H % a.group13 != 0 || a.I % a.group2 != 0) return B2Q_ERR_SHAPE;
  if (a.E > 1024 || a.top_k > 32 || a.H > MAX_K || a.I > MAX_K || a.T > INT32_MAX / 32 || 2 * a.E * a.I > INT32_MAX || a.E * a.H > INT32_MAX ||
      2 * a.I > INT32_MAX / (a.H / a.group13) || a.H > INT32_MAX / (a.I / a.group2) || !moe_g4_many_fits(a.T, a.E, a.top_k, a.H, a.I))
    return B2Q_ERR_LIMIT;
  if (!aligned16(a.x) || !aligned16(a.w13) || !aligned16(a.w2) || !aligned16(a.out) || !aligned_to(a.s13, 2) || !aligned_to(a.s2, 2) || !aligned_to(a.weights, 4) ||
      !aligned_to(a.ids, 4))
    return B2Q_ERR_ALIGN;
  if (a.T == 0) return B2Q_OK;
  if (!workspace) return B2Q_ERR_NULL;
  if (!aligned_to(workspace, 256)) return B2Q_ERR_ALIGN;
  if (workspace_bytes < b2q_moe_forward_w4_workspace_bytes(a.T, a.E, a.top_k, a.H, a.I)) return B2Q_ERR_WORKSPACE;
  G4MoeArgs g{};
  g.x = a.x; g.bf16 = a.act_dtype == B2Q_BF16; g.weights = a.weights; g.ids = a.ids; g.w13 = a.w13; g.s13 = a.s13; g.z13 = a.z13; g.w2 = a.w2; g.s2 = a.s2; g.z2 = a.z2;
  g.out = a.out; g.T = (int)a.T; g.E = (int)a.E; g.k = (int)a.top_k; g.H = (int)a.H; g.I = (int)a.I; g.G13 = (int)a.group13; g.G2 = (int)a.group2;
  if (use_few(g)) return moe_g4_few(g, workspace, (cudaStream_t)stream);
  return moe_g4_many(g, workspace, (cudaStream_t)stream);
}

}  // extern "C"
