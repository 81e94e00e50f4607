// Load-balancing loss of a router, the routes per expert, and the logits' gradient.
//
//   n = kept tokens (mask; all without one);  counts_e = kept routes to e;  p_t = softmax(logits_t)
//   loss = E sum_e f_e P_e,  f_e = counts_e / (n top_k),  P_e = sum over kept t of p_te / n
//   d loss / d logits_te = p_te (F_e - sum_j F_j p_tj),  F_e = E f_e / n  (f is piecewise constant)
// A row of nothing but -inf has no probabilities: p = 0.  No kept token: loss 0, gradient 0.
// Both passes read the logits once; the gradient computes the softmax again instead of keeping it.
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kBalWaves = 4, kBalThreads = kBalWaves * 64;

__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}
template <typename T>
__device__ __forceinline__ float logit(const void* z, int64_t i) {
  if constexpr (std::is_same<T, float>::value) return ((const float*)z)[i];
  else return from_bits<T>(((const uint16_t*)z)[i]);
}

// Softmax of a row by the hardware's exp2 (a value below 2^-126 becomes 0); value v of a lane is expert 64 v + lane (0 past E).
template <typename T, int V>
__device__ __forceinline__ void row_softmax(const void* z, int64_t at, int E, int lane, float* p) {
  float top = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = 64 * v + lane;
    p[v] = e < E ? logit<T>(z, at + e) : -__builtin_inff();
    top = fmaxf(top, p[v]);
  }
  top = wave_max_f32(top);
  if (top == -__builtin_inff()) top = 0.f;  // exp(-inf) = 0 for the whole row
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p[v] = __expf(p[v] - top);
    s += p[v];
  }
  s = wave_sum_f32(s);
  const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] *= inv;
}

struct BalanceArgs {
  const void *logits, *ids;
  int64_t ld;
  const uint8_t* mask;
  int T, E, topk, id64;
  // partial sums of `blocks` blocks: probabilities [blocks][E] fp32, routes [blocks][E], kept [blocks]
  float* part_p;
  int *part_c, *part_n;
  float *loss, *factor;
  int* counts;
  int blocks;
};

template <typename T, int V>
__global__ void __launch_bounds__(kBalThreads) balance_rows_kernel(BalanceArgs a) {
  extern __shared__ int hist[];  // [E], then the waves' sums [kBalWaves][64 V]
  float* sums = (float*)(hist + a.E);
  __shared__ int kept_all;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int e = t; e < a.E; e += kBalThreads) hist[e] = 0;
  if (t == 0) kept_all = 0;
  __syncthreads();
  float acc[V] = {};
  int kept = 0;
  for (int row = blockIdx.x * kBalWaves + wave; row < a.T; row += a.blocks * kBalWaves) {
    if (a.mask && !a.mask[row]) continue;
    ++kept;
    float p[V];
    row_softmax<T, V>(a.logits, (int64_t)row * a.ld, a.E, lane, p);
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] += p[v];
    for (int j = lane; j < a.topk; j += 64) {
      const int64_t r = (int64_t)row * a.topk + j;
      const int64_t e = a.id64 ? ((const int64_t*)a.ids)[r] : (int64_t)((const int32_t*)a.ids)[r];
      if (e >= 0 && e < a.E) atomicAdd(&hist[e], 1);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sums[wave * 64 * V + 64 * v + lane] = acc[v];
  if (lane == 0 && kept) atomicAdd(&kept_all, kept);
  __syncthreads();
  for (int e = t; e < a.E; e += kBalThreads) {
    float s = sums[e];
    for (int w = 1; w < kBalWaves; ++w) s += sums[w * 64 * V + e];
    a.part_p[(int64_t)blockIdx.x * a.E + e] = s;
    a.part_c[(int64_t)blockIdx.x * a.E + e] = hist[e];
  }
  if (t == 0) a.part_n[blockIdx.x] = kept_all;
}

// One block joins the blocks' sums, in block order, in fp64.
__global__ void __launch_bounds__(1024) balance_join_kernel(BalanceArgs a) {
  __shared__ double part[16];
  __shared__ int kept_all;
  const int t = threadIdx.x;
  if (t == 0) kept_all = 0;
  __syncthreads();
  int kept = 0;
  for (int b = t; b < a.blocks; b += 1024) kept += a.part_n[b];
  if (kept) atomicAdd(&kept_all, kept);
  __syncthreads();
  const double n = kept_all > 0 ? (double)kept_all : 1.0;
  double mine = 0.0;
  if (t < a.E) {
    double s = 0.0;
    int c = 0;
    for (int b = 0; b < a.blocks; ++b) {
      s += (double)a.part_p[(int64_t)b * a.E + t];
      c += a.part_c[(int64_t)b * a.E + t];
    }
    const double f = (double)c / (n * a.topk);
    a.counts[t] = c;
    a.factor[t] = (float)(a.E * f / n);
    mine = a.E * f * (s / n);
  }
  mine = wave_sum_f64(mine);
  if ((t & 63) == 0) part[t >> 6] = mine;
  __syncthreads();
  if (t == 0) {
    double loss = 0.0;
    for (int w = 0; w < 16; ++w) loss += part[w];
    a.loss[0] = (float)loss;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kBalThreads) balance_grad_kernel(const void* __restrict__ logits, int64_t ld,
                                                                   const uint8_t* __restrict__ mask, const float* __restrict__ factor,
                                                                   const float* __restrict__ upstream, void* __restrict__ grad, int rows,
                                                                   int E) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = 64 * v + lane < E ? factor[64 * v + lane] : 0.f;
  const float g = upstream[0];
  for (int row = blockIdx.x * kBalWaves + wave; row < rows; row += gridDim.x * kBalWaves) {
    float p[V];
    const bool in = !mask || mask[row];
    if (in) {
      row_softmax<T, V>(logits, (int64_t)row * ld, E, lane, p);
      float dot = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) dot = fmaf(f[v], p[v], dot);
      dot = wave_sum_f32(dot);
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = g * (p[v] * (f[v] - dot));
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = 64 * v + lane;
      if (e >= E) continue;
      const int64_t at = (int64_t)row * E + e;
      if constexpr (std::is_same<T, float>::value) ((float*)grad)[at] = p[v];
      else ((uint16_t*)grad)[at] = to_bits<T>(p[v]);
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

// Blocks of the forward pass: 16 rows for each of a block's waves, at most two blocks per CU.
static int balance_blocks(int64_t T) { return (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(T, kBalWaves * 16), 512)); }

size_t balance_workspace_bytes(int64_t T, int E) { return (size_t)balance_blocks(T) * (size_t)(2 * E + 1) * 4; }

template <typename T>
static void rows_by_width(const BalanceArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.blocks), block(kBalThreads);
  const auto lds = [&](int V) { return (size_t)(a.E + kBalWaves * 64 * V) * 4; };
  if (a.E <= 64) balance_rows_kernel<T, 1><<<grid, block, lds(1), st>>>(a);
  else if (a.E <= 128) balance_rows_kernel<T, 2><<<grid, block, lds(2), st>>>(a);
  else if (a.E <= 256) balance_rows_kernel<T, 4><<<grid, block, lds(4), st>>>(a);
  else if (a.E <= 512) balance_rows_kernel<T, 8><<<grid, block, lds(8), st>>>(a);
  else balance_rows_kernel<T, 16><<<grid, block, lds(16), st>>>(a);
}

int launch_moe_balance(const void* logits, int64_t ld, int dtype, const void* ids, int id64, const uint8_t* mask, int64_t T, int E,
                       int topk, float* loss, int32_t* counts, float* factor, void* workspace, hipStream_t st) {
  BalanceArgs a{};
  a.logits = logits, a.ids = ids, a.ld = ld, a.mask = mask;
  a.T = (int)T, a.E = E, a.topk = topk, a.id64 = id64;
  a.blocks = balance_blocks(T);
  a.part_p = (float*)workspace;
  a.part_c = (int*)(a.part_p + (size_t)a.blocks * E);
  a.part_n = a.part_c + (size_t)a.blocks * E;
  a.loss = loss, a.factor = factor, a.counts = counts;
  if (dtype == AWQ_DTYPE_F16) rows_by_width<f16>(a, st);
  else if (dtype == AWQ_DTYPE_BF16) rows_by_width<bf16>(a, st);
  else rows_by_width<float>(a, st);
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  balance_join_kernel<<<1, 1024, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

template <typename T>
static void grad_by_width(const void* logits, int64_t ld, const uint8_t* mask, const float* factor, const float* upstream, void* grad,
                          int T_, int E, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(T_, kBalWaves), 2048)), block(kBalThreads);
  if (E <= 64) balance_grad_kernel<T, 1><<<grid, block, 0, st>>>(logits, ld, mask, factor, upstream, grad, T_, E);
  else if (E <= 128) balance_grad_kernel<T, 2><<<grid, block, 0, st>>>(logits, ld, mask, factor, upstream, grad, T_, E);
  else if (E <= 256) balance_grad_kernel<T, 4><<<grid, block, 0, st>>>(logits, ld, mask, factor, upstream, grad, T_, E);
  else if (E <= 512) balance_grad_kernel<T, 8><<<grid, block, 0, st>>>(logits, ld, mask, factor, upstream, grad, T_, E);
  else balance_grad_kernel<T, 16><<<grid, block, 0, st>>>(logits, ld, mask, factor, upstream, grad, T_, E);
}

int launch_moe_balance_grad(const void* logits, int64_t ld, int dtype, const uint8_t* mask, const float* factor, const float* upstream,
                            void* grad, int64_t T, int E, hipStream_t st) {
  if (dtype == AWQ_DTYPE_F16) grad_by_width<f16>(logits, ld, mask, factor, upstream, grad, (int)T, E, st);
  else if (dtype == AWQ_DTYPE_BF16) grad_by_width<bf16>(logits, ld, mask, factor, upstream, grad, (int)T, E, st);
  else grad_by_width<float>(logits, ld, mask, factor, upstream, grad, (int)T, E, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
