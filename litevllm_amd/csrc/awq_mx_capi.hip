// extern "C" entry points of the microscaled fp4 products and of the router's balance loss (declared in
// include/awq_w4a16.h): argument checks and dispatch.  No function throws, allocates device memory or
// leaves a pending HIP error behind.
#include "awq_launch.h"
#include "awq_mx_common.h"

using namespace awq;
using namespace awq_host;

namespace {
bool dtype_16(int d) { return d == AWQ_DTYPE_F16 || d == AWQ_DTYPE_BF16; }
bool dtype_float(int d) { return dtype_16(d) || d == AWQ_DTYPE_F32; }
bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
constexpr int64_t kIntMax = 0x7FFFFFFFLL;
constexpr int64_t kMaxBalance = (int64_t)1 << 30;  // tokens and routes: 32 bits number them, a block's behind the last too
constexpr int64_t kMaxN = kIntMax - 255;       // columns of a block, those behind the last too, in 32 bits
constexpr int64_t kMaxK = (int64_t)1 << 24;   // 256 rows of codes are addressed in 32 bits,
constexpr int64_t kBytes = 0xFFFF0000LL;      // and so are all of the tokens' and all of an expert's gate and up

// What the calls take; their workspace queries answer 0 for the rest.
bool gemm_fits(int64_t M, int64_t N, int64_t K) { return M <= kIntMax && N <= kMaxN && K <= kMaxK; }
bool moe_fits(int64_t T, int64_t H, int64_t I, int32_t E, int32_t top_k) {
  return E <= 1024 && H <= kMaxK && I <= kMaxK && T <= kIntMax && T * top_k <= kIntMax && T * (H / 2) <= kBytes && I * H <= kBytes;
}
bool balance_fits(int64_t T, int32_t E) { return E <= 1024 && T <= kMaxBalance; }
}  // namespace

extern "C" {

int awq_w4a16_mxfp4_quantize(const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t M, int64_t K, int32_t dtype,
                             void* stream) {
  if (M < 0 || K < 0 || (K % 32) != 0) return AWQ_ERR_SHAPE;
  if (M == 0 || K == 0) return AWQ_OK;
  if (!x || !codes || !scales) return AWQ_ERR_NULL;
  if (!dtype_float(dtype) || K > kIntMax) return AWQ_ERR_UNSUPPORTED;
  if ((M > 1 && (ldx < K || (ldx % 8) != 0)) || !aligned(x, 16) || !aligned(codes, 16)) return AWQ_ERR_STRIDE;
  return launch_mx_quantize(x, ldx, codes, scales, K / 32, M, K, dtype, (hipStream_t)stream);
}

int awq_w4a16_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int64_t M, int64_t K, int32_t out_dtype,
                               void* stream) {
  if (M < 0 || K < 0 || (K % 32) != 0) return AWQ_ERR_SHAPE;
  if (M == 0 || K == 0) return AWQ_OK;
  if (!codes || !scales || !out) return AWQ_ERR_NULL;
  if (!dtype_float(out_dtype) || K > kIntMax) return AWQ_ERR_UNSUPPORTED;
  if (!aligned(codes, 16) || !aligned(out, 16)) return AWQ_ERR_STRIDE;
  return launch_mx_dequantize(codes, scales, out, M, K, out_dtype, (hipStream_t)stream);
}

size_t awq_w4a16_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || !gemm_fits(M, N, K) || mx_quantizes_itself(M, K)) return 0;
  return align256((size_t)M * (size_t)(K / 2)) + (size_t)M * (size_t)(K / 32);
}

int awq_w4a16_mxfp4_gemm(const void* a, int64_t lda, const uint8_t* a_scales, const uint8_t* w, const uint8_t* w_scales,
                         const void* bias, void* c, int64_t ldc, int64_t M, int64_t N, int64_t K, int32_t act_dtype,
                         int32_t bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || (K % 32) != 0) return AWQ_ERR_SHAPE;
  if (M == 0 || N == 0) return AWQ_OK;
  if (!a || !w || !w_scales || !c) return AWQ_ERR_NULL;
  if (!dtype_16(act_dtype) || !gemm_fits(M, N, K)) return AWQ_ERR_UNSUPPORTED;
  if (bias ? !dtype_float(bias_dtype) : bias_dtype != AWQ_DTYPE_NONE) return AWQ_ERR_UNSUPPORTED;
  if (!aligned(a, 16) || !aligned(w, 16) || !aligned(c, 2) || ldc < N) return AWQ_ERR_STRIDE;
  MxArgs p{};
  if (a_scales) {
    p.a = (const uint8_t*)a;
    p.as = a_scales;
  } else {
    if (M > 1 && (lda < K || (lda % 8) != 0)) return AWQ_ERR_STRIDE;
    const size_t need = awq_w4a16_mxfp4_gemm_workspace_bytes(M, N, K);
    if (need == 0) {
      p.x = (const uint16_t*)a;
      p.ldx = lda;
      p.xrows = (int)M;
    } else {
      if (!workspace || workspace_bytes < need) return AWQ_ERR_WORKSPACE;
      if (!aligned(workspace, 256)) return AWQ_ERR_STRIDE;
      uint8_t* codes = (uint8_t*)workspace;
      uint8_t* scales = codes + align256((size_t)M * (size_t)(K / 2));
      const int rc = launch_mx_quantize(a, lda, codes, scales, K / 32, M, K, act_dtype, (hipStream_t)stream);
      if (rc != AWQ_OK) return rc;
      p.a = codes;
      p.as = scales;
    }
  }
  p.w = w;
  p.ws = w_scales;
  p.K = (int)K;
  p.N = (int)N;
  p.M = (int)M;
  p.wrows = N;
  p.a_rows = M;
  p.as_ld = (int)(K / 32);
  p.c = (uint16_t*)c;
  p.ldc = ldc;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.out_bf16 = act_dtype == AWQ_DTYPE_BF16;
  return mx_takes_rows(M, N, K) ? launch_mx_rows_gemm(p, (hipStream_t)stream) : launch_mx_tile_gemm(p, (hipStream_t)stream);
}

size_t awq_w4a16_mxfp4_moe_workspace_bytes(int64_t T, int64_t H, int64_t I, int32_t E, int32_t top_k) {
  if (T <= 0 || H <= 0 || I <= 0 || E <= 0 || top_k <= 0 || !moe_fits(T, H, I, E, top_k)) return 0;
  return (size_t)mx_moe_workspace(T, H, I, E, top_k).total;
}

int awq_w4a16_mxfp4_moe(const void* x, int64_t ldx, const void* topk_ids, int32_t ids_bits, const void* topk_weights,
                        int32_t weights_dtype, const uint8_t* gate_up, const uint8_t* gate_up_scales, const uint8_t* down,
                        const uint8_t* down_scales, void* out, int64_t ldo, int64_t T, int64_t H, int64_t I, int32_t E,
                        int32_t top_k, int32_t activation, int32_t act_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || H <= 0 || I <= 0 || E <= 0 || top_k <= 0 || (H % 32) != 0 || (I % 32) != 0) return AWQ_ERR_SHAPE;
  if (T == 0) return AWQ_OK;
  if (!x || !topk_ids || !topk_weights || !gate_up || !gate_up_scales || !down || !down_scales || !out) return AWQ_ERR_NULL;
  if (!dtype_16(act_dtype) || !dtype_float(weights_dtype) || (ids_bits != 32 && ids_bits != 64)) return AWQ_ERR_UNSUPPORTED;
  if (activation != AWQ_MOE_ACT_SILU && activation != AWQ_MOE_ACT_GELU_TANH) return AWQ_ERR_UNSUPPORTED;
  if (!moe_fits(T, H, I, E, top_k)) return AWQ_ERR_UNSUPPORTED;
  if ((T > 1 && (ldx < H || (ldx % 8) != 0 || ldo < H)) || !aligned(x, 16) || !aligned(out, 2)) return AWQ_ERR_STRIDE;
  if (!aligned(gate_up, 16) || !aligned(down, 16)) return AWQ_ERR_STRIDE;
  if (!workspace || workspace_bytes < awq_w4a16_mxfp4_moe_workspace_bytes(T, H, I, E, top_k)) return AWQ_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return AWQ_ERR_STRIDE;
  MxMoeCall c{};
  c.x = x, c.ldx = ldx, c.ids = topk_ids, c.id64 = ids_bits == 64, c.weights = topk_weights, c.weights_dtype = weights_dtype;
  c.gate_up = gate_up, c.gate_up_scales = gate_up_scales, c.down = down, c.down_scales = down_scales;
  c.out = out, c.ldo = ldo, c.T = T, c.H = H, c.I = I, c.E = E, c.topk = top_k;
  c.act_kind = activation, c.act_dtype = act_dtype, c.workspace = workspace;
  return launch_mx_moe(c, (hipStream_t)stream);
}

size_t awq_w4a16_moe_balance_workspace_bytes(int64_t T, int32_t E) {
  return T < 0 || E <= 0 || !balance_fits(T, E) ? 0 : balance_workspace_bytes(T, E);
}

int awq_w4a16_moe_balance(const void* logits, int64_t ld, int32_t logits_dtype, const void* topk_ids, int32_t ids_bits,
                          const uint8_t* mask, int64_t T, int32_t E, int32_t top_k, float* loss, int32_t* counts, float* factor,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || E <= 0 || top_k <= 0) return AWQ_ERR_SHAPE;
  if (!loss || !counts || !factor || (T > 0 && (!logits || !topk_ids))) return AWQ_ERR_NULL;
  if (!dtype_float(logits_dtype) || (ids_bits != 32 && ids_bits != 64)) return AWQ_ERR_UNSUPPORTED;
  if (!balance_fits(T, E) || T * top_k > kMaxBalance) return AWQ_ERR_UNSUPPORTED;
  if (T > 1 && ld < E) return AWQ_ERR_STRIDE;
  if (!workspace || workspace_bytes < balance_workspace_bytes(T, E)) return AWQ_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return AWQ_ERR_STRIDE;
  return launch_moe_balance(logits, ld, logits_dtype, topk_ids, ids_bits == 64, mask, T, E, top_k, loss, counts, factor, workspace,
                            (hipStream_t)stream);
}

int awq_w4a16_moe_balance_grad(const void* logits, int64_t ld, int32_t logits_dtype, const uint8_t* mask, const float* factor,
                               const float* upstream, void* grad, int64_t T, int32_t E, void* stream) {
  if (T < 0 || E <= 0) return AWQ_ERR_SHAPE;
  if (T == 0) return AWQ_OK;
  if (!logits || !factor || !upstream || !grad) return AWQ_ERR_NULL;
  if (!dtype_float(logits_dtype) || !balance_fits(T, E)) return AWQ_ERR_UNSUPPORTED;
  if (T > 1 && ld < E) return AWQ_ERR_STRIDE;
  return launch_moe_balance_grad(logits, ld, logits_dtype, mask, factor, upstream, grad, T, E, (hipStream_t)stream);
}

}  // extern "C"
