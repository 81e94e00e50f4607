// extern "C" entry points of the sorted routes and of the low-rank adapters (declared in include/awq_w4a16.h): argument
// checks and dispatch.  No function throws, allocates device memory or leaves a pending HIP error behind.
#include "awq_launch.h"

using namespace awq;
using namespace awq_host;

namespace {
bool dtype_16(int d) { return d == AWQ_DTYPE_F16 || d == AWQ_DTYPE_BF16; }
bool dtype_float(int d) { return dtype_16(d) || d == AWQ_DTYPE_F32; }
bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
constexpr int64_t kMaxRoutes = (int64_t)1 << 30;  // 32 bits number them, a block's behind the last too
constexpr int64_t kMaxTokens = (int64_t)1 << 23;  // a launch's threads in 32 bits, with 256 a token,
constexpr int64_t kMaxRows = (int64_t)1 << 24;    // or 128 a row
constexpr int64_t kMaxWidth = (int64_t)1 << 24;   // a row's pieces, and blocks over them, in 32 and 16 bits
constexpr int64_t kMaxRank = 256;

bool routes_fit(int64_t T, int64_t H, int32_t top_k) { return T <= kMaxTokens && T * top_k <= kMaxRoutes && H <= kMaxWidth; }
bool lora_fits(int64_t M, int64_t N, int64_t K, int64_t R) {
  return M <= kMaxRows && N <= kMaxWidth && K <= kMaxWidth && R <= kMaxRank;
}
}  // namespace

extern "C" {

size_t awq_w4a16_moe_sort_workspace_bytes(int64_t T, int32_t E, int32_t top_k) {
  return T <= 0 || E <= 0 || E > 1024 || top_k <= 0 || top_k > 1024 || !routes_fit(T, 0, top_k) ? 0 : moe_sort_workspace_bytes(T, E, top_k);
}

int awq_w4a16_moe_sort(const void* x, int64_t ldx, const void* topk_ids, int32_t ids_bits, void* rows, int32_t* offsets,
                       int32_t* experts, int32_t* places, int64_t T, int64_t H, int32_t E, int32_t top_k, int32_t dtype,
                       void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || H < 0 || E <= 0 || top_k <= 0) return AWQ_ERR_SHAPE;
  if (!offsets || (T > 0 && (!topk_ids || !experts || !places || (H > 0 && (!x || !rows))))) return AWQ_ERR_NULL;
  if (!dtype_float(dtype) || (ids_bits != 32 && ids_bits != 64)) return AWQ_ERR_UNSUPPORTED;
  if (E > 1024 || top_k > 1024 || !routes_fit(T, H, top_k)) return AWQ_ERR_UNSUPPORTED;
  const int size = dtype == AWQ_DTYPE_F32 ? 4 : 2;
  if ((T > 1 && ldx < H) || !aligned(x, size) || !aligned(rows, size)) return AWQ_ERR_STRIDE;
  const size_t need = awq_w4a16_moe_sort_workspace_bytes(T, E, top_k);
  if (need && (!workspace || workspace_bytes < need)) return AWQ_ERR_WORKSPACE;
  if (need && !aligned(workspace, 16)) return AWQ_ERR_STRIDE;
  MoeSortCall c{};
  c.x = x, c.ldx = ldx, c.ids = topk_ids, c.id64 = ids_bits == 64, c.rows = rows, c.offsets = offsets, c.experts = experts;
  c.places = places, c.T = T, c.H = H, c.E = E, c.topk = top_k, c.elem_bytes = size, c.workspace = workspace;
  return launch_moe_sort(c, (hipStream_t)stream);
}

int awq_w4a16_moe_unsort(const void* rows, const int32_t* places, const void* topk_weights, int32_t weights_dtype, void* out,
                         int64_t ldo, int64_t T, int64_t H, int32_t top_k, int32_t dtype, void* stream) {
  if (T < 0 || H < 0 || top_k <= 0) return AWQ_ERR_SHAPE;
  if (T == 0 || H == 0) return AWQ_OK;
  if (!rows || !places || !out) return AWQ_ERR_NULL;
  if (!dtype_float(dtype) || (topk_weights ? !dtype_float(weights_dtype) : weights_dtype != AWQ_DTYPE_NONE)) return AWQ_ERR_UNSUPPORTED;
  if (!routes_fit(T, H, top_k)) return AWQ_ERR_UNSUPPORTED;
  const int size = dtype == AWQ_DTYPE_F32 ? 4 : 2;
  if ((T > 1 && ldo < H) || !aligned(rows, size) || !aligned(out, size)) return AWQ_ERR_STRIDE;
  MoeUnsortCall c{};
  c.rows = rows, c.places = places, c.weights = topk_weights, c.w_dtype = weights_dtype, c.out = out, c.ldo = ldo;
  c.T = T, c.H = H, c.topk = top_k, c.dtype = dtype;
  return launch_moe_unsort(c, (hipStream_t)stream);
}

int awq_w4a16_moe_unsort_grad(const void* upstream, int64_t ldu, const void* rows, const int32_t* places, const int32_t* total,
                              const void* topk_weights, int32_t weights_dtype, void* grad_rows, void* grad_weights, int64_t T,
                              int64_t H, int32_t top_k, int32_t dtype, void* stream) {
  if (T < 0 || H < 0 || top_k <= 0) return AWQ_ERR_SHAPE;
  if (T == 0 || (!grad_rows && !grad_weights)) return AWQ_OK;
  if (!places || (H > 0 && !upstream) || (grad_rows && !total) || (grad_weights && H > 0 && !rows)) return AWQ_ERR_NULL;
  if (!dtype_float(dtype) || (topk_weights || grad_weights ? !dtype_float(weights_dtype) : weights_dtype != AWQ_DTYPE_NONE))
    return AWQ_ERR_UNSUPPORTED;
  if (!routes_fit(T, H, top_k)) return AWQ_ERR_UNSUPPORTED;
  const int size = dtype == AWQ_DTYPE_F32 ? 4 : 2;
  if ((T > 1 && ldu < H) || !aligned(rows, size) || !aligned(upstream, size) || !aligned(grad_rows, size)) return AWQ_ERR_STRIDE;
  MoeUnsortCall c{};
  c.upstream = upstream, c.ldu = ldu, c.rows = rows, c.places = places, c.total = total, c.weights = topk_weights;
  c.w_dtype = weights_dtype, c.grad_rows = grad_rows, c.grad_weights = grad_weights;
  c.T = T, c.H = H, c.topk = top_k, c.dtype = dtype;
  return launch_moe_unsort_grad(c, (hipStream_t)stream);
}

size_t awq_w4a16_lora_workspace_bytes(int64_t M, int64_t K, int64_t R) {
  return M <= 0 || K <= 0 || R <= 0 || !lora_fits(M, 0, K, R) ? 0 : lora_workspace_bytes(M, K, R);
}

int awq_w4a16_lora_add(const void* base, int64_t ldb, const void* x, int64_t ldx, const void* lora_a, int64_t a_stride,
                       const void* lora_b, int64_t b_stride, const void* ids, int32_t ids_bits, const float* scales, void* out,
                       int64_t ldo, int64_t M, int64_t N, int64_t K, int64_t R, int32_t L, int32_t dtype, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || R <= 0 || L <= 0) return AWQ_ERR_SHAPE;
  if (M == 0 || N == 0) return AWQ_OK;
  if (!x || !lora_a || !lora_b || !ids || !out) return AWQ_ERR_NULL;
  if (!dtype_16(dtype) || (ids_bits != 32 && ids_bits != 64) || !lora_fits(M, N, K, R)) return AWQ_ERR_UNSUPPORTED;
  if (M > 1 && (ldx < K || ldo < N || (base && ldb < N))) return AWQ_ERR_STRIDE;
  if (L > 1 && (a_stride < R * K || b_stride < N * R)) return AWQ_ERR_STRIDE;
  if (!aligned(x, 2) || !aligned(lora_a, 2) || !aligned(lora_b, 2) || !aligned(base, 2) || !aligned(out, 2)) return AWQ_ERR_STRIDE;
  const size_t need = lora_workspace_bytes(M, K, R);
  if (need && (!workspace || workspace_bytes < need)) return AWQ_ERR_WORKSPACE;
  if (need && !aligned(workspace, 16)) return AWQ_ERR_STRIDE;
  LoraCall c{};
  c.base = base, c.ldb = ldb, c.x = x, c.ldx = ldx, c.a = lora_a, c.a_stride = a_stride, c.b = lora_b, c.b_stride = b_stride;
  c.ids = ids, c.id64 = ids_bits == 64, c.scales = scales, c.out = out, c.ldo = ldo;
  c.M = M, c.N = N, c.K = K, c.R = R, c.L = L, c.dtype = dtype, c.workspace = workspace;
  return launch_lora(c, (hipStream_t)stream);
}

}  // extern "C"
