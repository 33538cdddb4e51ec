// The gated feed-forward block with 16-bit weights (a shared expert): forward and backward.
//
//   ab = x . W13^T   a = ab[:, :I], b = ab[:, I:]       h = silu(a) * b       y = h . W2^T (+ add)
//   dh = dy . W2     da = dh b s (1 + a (1 - s)), db = dh a s   with s = 1 / (1 + exp(-a))
//   dx = [da db] . W13      dW13 = [da db]^T . x      dW2 = dy^T . h
//
// Roundings to 16 bits besides the results': h (the second product's operand), da and db (the
// operands of dx and dW13), each once from fp32. The pre-activations are kept in fp32 for the
// backward pass, 8 T I bytes: kept in 16 bits their rounding would enter da, db and h a second
// time. h is recomputed from them rather than kept.
#include "few_tokens.cuh"
#include "kernels.cuh"

namespace muse {
namespace {

constexpr size_t kAlign = 256;

int check_ffn(int tokens, int hidden, int inter) {
  if (tokens < 0 || hidden <= 0 || inter <= 0) return MUSE_ERR_INVALID_ARGUMENT;
  if (hidden % 8 || inter % 8 || hidden > (1 << 24) || inter > (1 << 24) || tokens > kMaxRows)
    return MUSE_ERR_UNSUPPORTED_SHAPE;
  return MUSE_OK;
}

// How a forward product runs: few tokens stream the weights; else the cheaper side for the weights by
// the sizes' estimates (64 x 7168 x 2048 block: 25 us with the weights as the MMA's rows, 38 as its
// columns). It depends on the sizes alone, so a forward pass has the same bits whether it keeps its
// pre-activations or not.
int (*forward_product(int t, int n, int k, int mode))(const DenseGemm&, cudaStream_t) {
  if (streams_dense(t, n, k)) return launch_few_dense;
  return swap_dense_cost(t, n, k) < dense_cost(t, n, k, mode, true) ? launch_swap_dense : launch_dense_gemm;
}
size_t forward_scratch(int t, int n, int k, int mode) {
  if (forward_product(t, n, k, mode) != launch_dense_gemm) return 0;
  return dense_scratch_bytes(t, n, k, mode, true);
}

PlanInfo forward_plan(int t, int n, int k, int mode) {
  const auto product = forward_product(t, n, k, mode);
  if (product == launch_few_dense) return {};
  return product == launch_swap_dense ? swap_dense_plan(t, n, k) : dense_plan(t, n, k, mode, true);
}

size_t up(size_t v) { return align_up(v, kAlign); }
size_t most(size_t a, size_t b) { return a > b ? a : b; }

// Workspace: h [T, I] 16-bit, (backward) [da db] [T, 2I] 16-bit, partial sums of the split products.
struct FfnLayout {
  size_t h, dab, partials, total;
};
FfnLayout ffn_layout(int t, int hidden, int inter, bool backward) {
  FfnLayout l;
  size_t part;
  if (backward)
    part = most(most(dense_scratch_bytes(t, inter, hidden, kDGate, false),
                     dense_scratch_bytes(t, hidden, 2 * inter, kStore, false)),
                most(dense_scratch_bytes(2 * inter, hidden, t, kStore, false),
                     dense_scratch_bytes(hidden, inter, t, kStore, false)));
  else
    part = most(forward_scratch(t, 2 * inter, hidden, kGate), forward_scratch(t, hidden, inter, kStore));
  l.h = 0;
  l.dab = up((size_t)2 * t * inter);
  l.partials = l.dab + (backward ? up((size_t)4 * t * inter) : 0);
  l.total = l.partials + up(part);
  return l;
}

bool bad_matrix(const void* p, long long ld, long long width) {
  return !p || reinterpret_cast<uintptr_t>(p) % 16 || ld % 8 || ld < width;
}

}  // namespace
}  // namespace muse

using namespace muse;

extern "C" int muse_moe_ffn_workspace_size(int tokens, int hidden, int inter, int backward, size_t* bytes) {
  if (!bytes) return MUSE_ERR_INVALID_ARGUMENT;
  const int rc = check_ffn(tokens, hidden, inter);
  if (rc) return rc;
  *bytes = tokens == 0 ? 0 : ffn_layout(tokens, hidden, inter, backward != 0).total;
  return MUSE_OK;
}

extern "C" int muse_moe_ffn_plan(int product, int tokens, int hidden, int inter, int* plan) {
  const int rc = check_ffn(tokens, hidden, inter);
  if (rc) return rc;
  if (!plan || tokens == 0) return MUSE_ERR_INVALID_ARGUMENT;
  switch (product) {
    case 0: return put_plan(forward_plan(tokens, 2 * inter, hidden, kGate), plan);
    case 1: return put_plan(forward_plan(tokens, hidden, inter, kStore), plan);
    case 2: return put_plan(dense_plan(tokens, inter, hidden, kDGate, false), plan);
    case 3: return put_plan(dense_plan(tokens, hidden, 2 * inter, kStore, false), plan);
    case 4: return put_plan(dense_plan(2 * inter, hidden, tokens, kStore, false), plan);
    case 5: return put_plan(dense_plan(hidden, inter, tokens, kStore, false), plan);
    default: return MUSE_ERR_INVALID_ARGUMENT;
  }
}

extern "C" int muse_moe_ffn_forward(const void* x, long long ldx, int dtype, int tokens, int hidden, int inter,
                                    const void* w13, long long ld13, const void* w2, long long ld2, const void* add,
                                    long long ld_add, void* out, float* ab, void* workspace, size_t workspace_bytes,
                                    muse_stream_t stream) {
  int rc = check_ffn(tokens, hidden, inter);
  if (rc) return rc;
  if (dtype != kBf16 && dtype != kFp16) return MUSE_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return MUSE_OK;
  if (bad_matrix(x, ldx, hidden) || bad_matrix(w13, ld13, hidden) || bad_matrix(w2, ld2, inter) ||
      bad_matrix(out, hidden, hidden) || (add && bad_matrix(add, ld_add, hidden)) || !workspace ||
      reinterpret_cast<uintptr_t>(ab) % 16 || reinterpret_cast<uintptr_t>(workspace) % kAlign)
    return MUSE_ERR_INVALID_ARGUMENT;
  const FfnLayout l = ffn_layout(tokens, hidden, inter, false);
  if (workspace_bytes < l.total) return MUSE_ERR_WORKSPACE_TOO_SMALL;
  char* ws = static_cast<char*>(workspace);
  int* flag = nullptr;
  if ((rc = device_status_ptr(&flag))) return rc;
  DenseGemm g{};
  g.dtype = dtype;
  g.error_flag = flag;
  g.partials = reinterpret_cast<float*>(ws + l.partials);
  g.a = {x, ldx, true};
  g.b = {w13, ld13, true};
  g.m = tokens, g.n = 2 * inter, g.k = hidden;
  g.mode = kGate;
  g.out = ws + l.h, g.ldo = inter;
  g.ab = ab;
  const cudaStream_t st = (cudaStream_t)stream;
  if ((rc = forward_product(g.m, g.n, g.k, g.mode)(g, st))) return rc;
  g.a = {ws + l.h, inter, true};
  g.b = {w2, ld2, true};
  g.n = hidden, g.k = inter;
  g.mode = kStore;
  g.out = out, g.ldo = hidden;
  g.ab = nullptr;
  g.add = add, g.ld_add = ld_add;
  return forward_product(g.m, g.n, g.k, g.mode)(g, st);
}

extern "C" int muse_moe_ffn_backward(const void* dy, long long ldy, const void* x, long long ldx, int dtype, int tokens,
                                     int hidden, int inter, const void* w13, long long ld13, const void* w2,
                                     long long ld2, const float* ab, void* dx, void* dw13, void* dw2, void* workspace,
                                     size_t workspace_bytes, muse_stream_t stream) {
  int rc = check_ffn(tokens, hidden, inter);
  if (rc) return rc;
  if (tokens == 0 || (dtype != kBf16 && dtype != kFp16)) return MUSE_ERR_INVALID_ARGUMENT;
  if (!dx && !dw13 && !dw2) return MUSE_OK;
  if (bad_matrix(dy, ldy, hidden) || bad_matrix(w2, ld2, inter) || !ab || reinterpret_cast<uintptr_t>(ab) % 16 ||
      (dx && (bad_matrix(w13, ld13, hidden) || bad_matrix(dx, hidden, hidden))) ||
      (dw13 && (bad_matrix(x, ldx, hidden) || bad_matrix(dw13, hidden, hidden))) ||
      (dw2 && bad_matrix(dw2, inter, inter)) || !workspace || reinterpret_cast<uintptr_t>(workspace) % kAlign)
    return MUSE_ERR_INVALID_ARGUMENT;
  const FfnLayout l = ffn_layout(tokens, hidden, inter, true);
  if (workspace_bytes < l.total) return MUSE_ERR_WORKSPACE_TOO_SMALL;
  char* ws = static_cast<char*>(workspace);
  int* flag = nullptr;
  if ((rc = device_status_ptr(&flag))) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  const void* dab = ws + l.dab;
  DenseGemm base{};
  base.dtype = dtype;
  base.error_flag = flag;
  base.partials = reinterpret_cast<float*>(ws + l.partials);
  base.mode = kStore;

  DenseGemm g = base;  // dh = dy . W2 -> [da db], h
  g.a = {dy, ldy, true};
  g.b = {w2, ld2, false};
  g.m = tokens, g.n = inter, g.k = hidden;
  g.mode = kDGate;
  g.out = ws + l.dab, g.ldo = 2LL * inter;
  g.ab = const_cast<float*>(ab);
  g.h_out = ws + l.h;
  if ((rc = launch_dense_gemm(g, st))) return rc;
  if (dx) {
    g = base;
    g.a = {dab, 2LL * inter, true};
    g.b = {w13, ld13, false};
    g.m = tokens, g.n = hidden, g.k = 2 * inter;
    g.out = dx, g.ldo = hidden;
    if ((rc = launch_dense_gemm(g, st))) return rc;
  }
  if (dw13) {
    g = base;
    g.a = {dab, 2LL * inter, false};
    g.b = {x, ldx, false};
    g.m = 2 * inter, g.n = hidden, g.k = tokens;
    g.out = dw13, g.ldo = hidden;
    if ((rc = launch_dense_gemm(g, st))) return rc;
  }
  if (dw2) {
    g = base;
    g.a = {dy, ldy, false};
    g.b = {ws + l.h, inter, false};
    g.m = hidden, g.n = inter, g.k = tokens;
    g.out = dw2, g.ldo = inter;
    rc = launch_dense_gemm(g, st);
  }
  return rc;
}
