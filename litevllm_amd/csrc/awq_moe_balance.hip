// Load-balancing loss of a router, the routes per expert, and the logits' gradient.
//
//   n = kept tokens (mask; all without one);  counts_e = kept routes to e;  p_t = softmax(logits_t)
//   loss = E sum_e f_e P_e,  f_e = counts_e / (n top_k),  P_e = sum over kept t of p_te / n
//   d loss / d logits_te = p_te (F_e - sum_j F_j p_tj),  F_e = E f_e / n  (f is piecewise constant)
// A row of nothing but -inf has no probabilities: p = 0.  No kept token: loss 0, gradient 0.
// Both passes read the logits once; the gradient computes the softmax again instead of keeping it (65536 tokens, 160
// experts, fp32: 42 MB; forward 10.6 us and 7.1 for the join, gradient 13.9 us, which reads and writes at 6.2 TB/s, partly
// from the caches).  Shorter calls are latencies and the launches; with a gradient the host is slower than the kernels
// from a call of 16384 tokens, 64 experts on down (10.5 us of kernels).
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kBalThreads = 1024, kBalWaves = kBalThreads / 64, kBalChain = 512;

// Steps of a reduction over G = 16, 32 or 64 neighbouring lanes: DPP inside rows of 16, then across rows.
template <int G, class Op>
__device__ __forceinline__ float group_reduce(float v, Op op) {
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = op(v, dpp(v, std::integral_constant<int, 0xB1>{}));   // quad_perm [1, 0, 3, 2]
  v = op(v, dpp(v, std::integral_constant<int, 0x4E>{}));   // quad_perm [2, 3, 0, 1]
  v = op(v, dpp(v, std::integral_constant<int, 0x141>{}));  // row_half_mirror
  v = op(v, dpp(v, std::integral_constant<int, 0x140>{}));  // row_mirror
  if constexpr (G >= 32) v = op(v, __shfl_xor(v, 16));
  if constexpr (G >= 64) v = op(v, __shfl_xor(v, 32));
  return v;
}
template <typename T>
__device__ __forceinline__ float logit(const void* z, int64_t i) {
  if constexpr (std::is_same<T, float>::value) return ((const float*)z)[i];
  else return from_bits<T>(((const uint16_t*)z)[i]);
}

// G lanes share a row, lane l of them the experts G v + l: a wave works on 64 / G rows at once, which keeps
// the reductions short and the loads of several rows under way.
template <typename T, int G, int V>
__device__ __forceinline__ void load_row(const void* z, int64_t at, int E, int l, float* p) {
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = G * v + l < E ? logit<T>(z, at + G * v + l) : -__builtin_inff();
}
// Softmax by the hardware's exp2 (a value below 2^-126 becomes 0); 0 past E.
template <int G, int V>
__device__ __forceinline__ void row_softmax(float* p) {
  float top = p[0];
#pragma unroll
  for (int v = 1; v < V; ++v) top = fmaxf(top, p[v]);
  top = group_reduce<G>(top, [](float a, float b) { return fmaxf(a, b); });
  if (top == -__builtin_inff()) top = 0.f;  // exp(-inf) = 0 for the whole row
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p[v] = __expf(p[v] - top);
    s += p[v];
  }
  s = group_reduce<G>(s, [](float a, float b) { return a + b; });
  const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] *= inv;
}

struct BalanceArgs {
  const void *logits, *ids;
  int64_t ld;
  const uint8_t* mask;
  int T, E, topk, id64;
  // sums of each of `blocks` blocks, of `rows` rows: probabilities [blocks][E] fp32, routes [blocks][E], kept [blocks]
  float* part_p;
  int *part_c, *part_n;
  float *loss, *factor;
  int* counts;
  int blocks, rows;
};

// Loss, counts and factors from every expert's sums (thread e has expert e's), by one block.
__device__ __forceinline__ void balance_finish(const BalanceArgs& a, int kept, double p, int c) {
  __shared__ double part[kBalWaves];
  const int t = threadIdx.x;
  const double n = kept > 0 ? (double)kept : 1.0;
  double mine = 0.0;
  if (t < a.E) {
    const double f = (double)c / (n * a.topk);
    a.counts[t] = c;
    a.factor[t] = (float)(a.E * f / n);
    mine = a.E * f * (p / n);
  }
  mine = wave_sum_f64(mine);
  if ((t & 63) == 0) part[t >> 6] = mine;
  __syncthreads();
  if (t == 0) {
    double loss = 0.0;
    for (int w = 0; w < kBalWaves; ++w) loss += part[w];
    a.loss[0] = (float)loss;
  }
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(kBalThreads) balance_rows_kernel(BalanceArgs a) {
  constexpr int COLS = G * V, PER = 64 / G;
  __shared__ float sums[kBalWaves][COLS];
  __shared__ int hist[COLS], kept_all;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l = lane % G;
  for (int e = t; e < COLS; e += kBalThreads) hist[e] = 0;
  if (t == 0) kept_all = 0;
  __syncthreads();
  const int first = blockIdx.x * a.rows, end = min(first + a.rows, a.T);
  for (int64_t i = (int64_t)first * a.topk + t; i < (int64_t)end * a.topk; i += kBalThreads) {
    if (a.mask && !a.mask[i / a.topk]) continue;
    const int64_t e = a.id64 ? ((const int64_t*)a.ids)[i] : (int64_t)((const int32_t*)a.ids)[i];
    if (e >= 0 && e < a.E) atomicAdd(&hist[e], 1);
  }
  // Sums in chains of at most kBalChain rows, and a chain of those, at most as many up to 2^30 tokens: 2 * 512 roundings, where
  // one chain would have up to 262144 (2^27 equal rows of p = 0.25: off by 3e-6, by 1.2e-4 in one chain).
  float acc[V] = {}, all[V] = {};
  int kept = 0;
  for (int base = first + wave * PER; base < end;) {
    const int stop = min(base + kBalChain * kBalWaves * PER, end);
    for (; base < stop; base += kBalWaves * PER) {
      const int row = base + lane / G;
      if (row >= end || (a.mask && !a.mask[row])) continue;
      ++kept;
      float p[V];
      load_row<T, G, V>(a.logits, (int64_t)row * a.ld, a.E, l, p);
      row_softmax<G, V>(p);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += p[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) all[v] += acc[v], acc[v] = 0.f;
  }
  if (l == 0 && kept) atomicAdd(&kept_all, kept);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (G <= 16) all[v] += __shfl_xor(all[v], 16);
    if constexpr (G <= 32) all[v] += __shfl_xor(all[v], 32);
    if (lane < G) sums[wave][G * v + l] = all[v];
  }
  __syncthreads();
  float s = 0.f;
  if (t < a.E)
    for (int w = 0; w < kBalWaves; ++w) s += sums[w][t];
  if (a.blocks == 1) {
    balance_finish(a, kept_all, s, t < a.E ? hist[t] : 0);
    return;
  }
  if (t < a.E) {
    a.part_p[(int64_t)blockIdx.x * a.E + t] = s;
    a.part_c[(int64_t)blockIdx.x * a.E + t] = hist[t];
  }
  if (t == 0) a.part_n[blockIdx.x] = kept_all;
}

// One block joins the blocks' sums: threads of a column take shares of the blocks, added in order in fp64.
__global__ void __launch_bounds__(kBalThreads) balance_join_kernel(BalanceArgs a) {
  __shared__ double sp[kBalThreads];
  __shared__ int sc[kBalThreads], kept_all;
  const int t = threadIdx.x, shares = kBalThreads / a.E, share = t / a.E, e = t - share * a.E;
  if (t == 0) kept_all = 0;
  __syncthreads();
  int kept = 0;
  for (int b = t; b < a.blocks; b += kBalThreads) kept += a.part_n[b];
  if (kept) atomicAdd(&kept_all, kept);
  double s = 0.0;
  int c = 0;
  if (share < shares) {
#pragma unroll 8
    for (int b = share; b < a.blocks; b += shares) {
      s += (double)a.part_p[(int64_t)b * a.E + e];
      c += a.part_c[(int64_t)b * a.E + e];
    }
  }
  sp[t] = s;
  sc[t] = c;
  __syncthreads();
  if (t < a.E)
    for (int i = 1; i < shares; ++i) s += sp[i * a.E + t], c += sc[i * a.E + t];
  balance_finish(a, kept_all, s, c);
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(256) balance_grad_kernel(const void* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask,
                                                           const float* __restrict__ factor, const float* __restrict__ upstream,
                                                           void* __restrict__ grad, int rows, int E) {
  constexpr int PER = 64 / G;
  const int lane = threadIdx.x & 63, l = lane % G;
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = G * v + l < E ? factor[G * v + l] : 0.f;
  const float g = upstream[0];
  for (int64_t row = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * PER + lane / G; row < rows; row += (int64_t)gridDim.x * 4 * PER) {
    float p[V];
    if (!mask || mask[row]) {
      load_row<T, G, V>(logits, row * ld, E, l, p);
      row_softmax<G, V>(p);
      float dot = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) dot = fmaf(f[v], p[v], dot);
      dot = group_reduce<G>(dot, [](float a, float b) { return a + b; });
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = g * (p[v] * (f[v] - dot));
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = G * v + l;
      if (e >= E) continue;
      if constexpr (std::is_same<T, float>::value) ((float*)grad)[row * E + e] = p[v];
      else ((uint16_t*)grad)[row * E + e] = to_bits<T>(p[v]);
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

// Up to 256 rows one block does everything (one launch); else at most a block per CU, so that the join, whose one block
// reads every block's sums, stays small (256 blocks of 160 experts: 7.1 us, of 64: 5.8).
static int balance_rows(int64_t T) { return T <= 256 ? 256 : (int)cdiv(T, std::min<int64_t>(256, cdiv(T, 64))); }
static int balance_blocks(int64_t T) { return (int)std::max<int64_t>(1, cdiv(T, balance_rows(T))); }

size_t balance_workspace_bytes(int64_t T, int E) { return (size_t)balance_blocks(T) * (size_t)(2 * E + 1) * 4; }

// Lanes to a row and values to a lane by the number of experts.
template <class F>
static void by_width(int E, F f) {
  using std::integral_constant;
  if (E <= 64) f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  else if (E <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  else if (E <= 192) f(integral_constant<int, 16>{}, integral_constant<int, 12>{});
  else if (E <= 256) f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  else if (E <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  else f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

template <typename T>
static void rows_by_width(const BalanceArgs& a, hipStream_t st) {
  by_width(a.E, [&](auto g, auto v) {
    balance_rows_kernel<T, decltype(g)::value, decltype(v)::value><<<dim3((unsigned)a.blocks), dim3(kBalThreads), 0, st>>>(a);
  });
}

int launch_moe_balance(const void* logits, int64_t ld, int dtype, const void* ids, int id64, const uint8_t* mask, int64_t T, int E,
                       int topk, float* loss, int32_t* counts, float* factor, void* workspace, hipStream_t st) {
  BalanceArgs a{};
  a.logits = logits, a.ids = ids, a.ld = ld, a.mask = mask;
  a.T = (int)T, a.E = E, a.topk = topk, a.id64 = id64;
  a.blocks = balance_blocks(T);
  a.rows = balance_rows(T);
  a.part_p = (float*)workspace;
  a.part_c = (int*)(a.part_p + (size_t)a.blocks * E);
  a.part_n = a.part_c + (size_t)a.blocks * E;
  a.loss = loss, a.factor = factor, a.counts = counts;
  if (dtype == AWQ_DTYPE_F16) rows_by_width<f16>(a, st);
  else if (dtype == AWQ_DTYPE_BF16) rows_by_width<bf16>(a, st);
  else rows_by_width<float>(a, st);
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  if (a.blocks == 1) return AWQ_OK;
  balance_join_kernel<<<1, kBalThreads, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

template <typename T>
static void grad_by_width(const void* logits, int64_t ld, const uint8_t* mask, const float* factor, const float* upstream, void* grad,
                          int T_, int E, hipStream_t st) {
  by_width(E, [&](auto g, auto v) {
    constexpr int G = decltype(g)::value, V = decltype(v)::value;
    const dim3 grid((unsigned)std::min<int64_t>(cdiv(T_, 4 * (64 / G)), 2048));
    balance_grad_kernel<T, G, V><<<grid, dim3(256), 0, st>>>(logits, ld, mask, factor, upstream, grad, T_, E);
  });
}

int launch_moe_balance_grad(const void* logits, int64_t ld, int dtype, const uint8_t* mask, const float* factor, const float* upstream,
                            void* grad, int64_t T, int E, hipStream_t st) {
  if (dtype == AWQ_DTYPE_F16) grad_by_width<f16>(logits, ld, mask, factor, upstream, grad, (int)T, E, st);
  else if (dtype == AWQ_DTYPE_BF16) grad_by_width<bf16>(logits, ld, mask, factor, upstream, grad, (int)T, E, st);
  else grad_by_width<float>(logits, ld, mask, factor, upstream, grad, (int)T, E, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
