// Products of microscaled fp4 matrices on the scaled MFMA (format, modes and operand order:
// awq_mx_common.h).
#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kMxWaves = 4;

// h of one value: act(gate) * up in fp32.
__device__ __forceinline__ float mx_gated(float g, float u, int act) {
  return (act == AWQ_MOE_ACT_GELU_TANH ? gated_act_fast<1>(g) : gated_act_fast<0>(g)) * u;
}

// Block: 16 MT rows of a by 16 NT rows of w; its waves take the steps of 128 along K in turn and their
// sums meet in LDS.  Operands go straight from memory to registers: each weight byte is used by one
// block of the row tile only.
// Grid x: column blocks, y: row tiles.  Gate_up blocks hold 32 gate rows and the same 32 up rows.
template <int MODE, int MT, int NT>
__global__ void __launch_bounds__(kMxWaves * 64) mx_rows_kernel(MxArgs p) {
  __shared__ float red[kMxWaves][MT * NT][256];
  const int tile = blockIdx.y;
  if (MODE != kMxDense && tile >= p.tile_count[0]) return;
  const MxRows t = mx_rows<MODE, 16 * MT>(p, tile);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  constexpr int COLS = MODE == kMxGateUp ? 8 * NT : 16 * NT;
  const int n0 = (int)blockIdx.x * COLS;
  const int KB = p.K / 32, steps = (KB + 3) / 4;

  const uint8_t *wc[NT], *wsc[NT], *ac[MT], *asc[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    int64_t row;
    if constexpr (MODE == kMxGateUp) row = (j < NT / 2 ? n0 + 16 * j : p.N + n0 + 16 * (j - NT / 2)) + r;
    else row = n0 + 16 * j + r < p.N ? n0 + 16 * j + r : p.N - 1;
    row += (int64_t)t.expert * p.wrows;
    wc[j] = p.w + row * (p.K / 2) + q * 16;
    wsc[j] = p.ws + row * KB + q;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = mx_a_row<MODE>(p, t, 16 * i + r);
    ac[i] = p.a + row * (p.K / 2) + q * 16;
    asc[i] = p.as + row * p.as_ld + q;
  }

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll 2
  for (int s = wave; s < steps; s += kMxWaves) {
    const bool in = 4 * s + q < KB;  // the last step may end inside
    u32x4 a[MT], b[NT];
    uint32_t sa[MT], sb[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      b[j] = in ? *(const u32x4*)(wc[j] + (int64_t)s * 64) : u32x4{0u, 0u, 0u, 0u};
      sb[j] = in ? wsc[j][s * 4] : 127u;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      a[i] = in ? *(const u32x4*)(ac[i] + (int64_t)s * 64) : u32x4{0u, 0u, 0u, 0u};
      sa[i] = in ? asc[i][s * 4] : 127u;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mx_mfma<0, 0>(a[i], b[j], acc[i][j], sa[i], sb[j]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) red[wave][i * NT + j][(4 * q + u) * 16 + r] = acc[i][j][u];
  __syncthreads();

  auto sum = [&](int tile16, int at) {
    float v = red[0][tile16][at];
#pragma unroll
    for (int w = 1; w < kMxWaves; ++w) v += red[w][tile16][at];
    return v;
  };
  if constexpr (MODE == kMxGateUp) {
    // 32 lanes hold a row's 32 columns: their largest magnitude, then the codes, two to a byte
    static_assert(NT == 4, "32 gate and 32 up rows");
    const int n = threadIdx.x & 31;
    for (int m = threadIdx.x >> 5; m < t.rows; m += kMxWaves * 2) {
      const int at = (m & 15) * 16 + (n & 15), tg = (m >> 4) * NT + (n >> 4);
      const float v = mx_gated(sum(tg, at), sum(tg + 2, at), p.act);
      uint32_t top = mx_abs_bits(v);
#pragma unroll
      for (int d = 1; d < 32; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
      const uint32_t byte = mx_scale_byte(top);
      const float other = __shfl_xor(v, 1);
      if ((n & 1) == 0) {
        const uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, v, other, mx_scale_value(byte == 255u ? 0u : byte), 0);
        p.h[(int64_t)(t.first + m) * (p.N / 2) + (n0 + n) / 2] = byte == 255u ? (uint8_t)0 : (uint8_t)code;
      }
      if (n == 0) p.hs[(int64_t)(t.first + m) * (p.N / 32) + n0 / 32] = (uint8_t)byte;
    }
  } else {
    for (int i = threadIdx.x; i < MT * NT * 256; i += kMxWaves * 64) {
      const int t16 = i >> 8, at = i & 255, m = (t16 / NT) * 16 + (at >> 4), n = n0 + (t16 % NT) * 16 + (at & 15);
      if (m >= t.rows || n >= p.N) continue;
      float v = sum(t16, at);
      if constexpr (MODE == kMxDense) {
        v += load_bias(p.bias, p.bias_dtype, n);
        p.c[(int64_t)(t.first + m) * p.ldc + n] = p.out_bf16 ? f2bf_bits(v) : f2h_bits(v);
      } else {
        p.y[(int64_t)p.order[t.first + m] * p.N + n] = v;
      }
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

template <int MODE, int MT, int NT>
static void launch_rows(const MxArgs& p, int64_t row_tiles, hipStream_t st) {
  constexpr int COLS = MODE == kMxGateUp ? 8 * NT : 16 * NT;
  const dim3 grid((unsigned)cdiv(p.N, COLS), (unsigned)row_tiles);
  mx_rows_kernel<MODE, MT, NT><<<grid, dim3(kMxWaves * 64), 0, st>>>(p);
}

int launch_mx_gemm(const MxArgs& p, hipStream_t st) {
  if (p.M > 64) return launch_mx_tile_gemm(p, st);
  if (p.M <= 16) launch_rows<kMxDense, 1, 1>(p, 1, st);
  else if (p.M <= 32) launch_rows<kMxDense, 2, 1>(p, 1, st);
  else launch_rows<kMxDense, 4, 2>(p, 1, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

int launch_mx_grouped(const MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st) {
  if (rows > 16) return launch_mx_tile_grouped(p, gate_up, rows, row_tiles, st);
  if (row_tiles > 65535) return AWQ_ERR_UNSUPPORTED;
  if (gate_up) launch_rows<kMxGateUp, 1, 4>(p, row_tiles, st);
  else launch_rows<kMxDown, 1, 2>(p, row_tiles, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
