// Products of microscaled fp4 matrices, many rows: tiles of both operands in LDS (format, modes and operand
// order: awq_mx_common.h).
#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kStageK = 256;  // K of a stage: 128 bytes of codes and 8 scale bytes per row

// Loads 16 bytes per lane straight into LDS, lane l to base + 16 l.
__device__ __forceinline__ void lds_load16(const uint8_t* src, void* base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)base, 16, 0, 0);
}

// Block: BM rows of a by BN rows of w, WM x WN waves of (BM / WM) x (BN / WN); the stages along K are double
// buffered, one barrier each.
//
// LDS: 16-byte chunk c of a tile's row sits at place c ^ (row & 7) of its 128 bytes, so that the 16 rows a
// fragment reads lie in different banks; the direct loads write lanes in order, so it is their sources that are
// permuted, inside the row's line.  Quarter q of a wave takes chunks 2 q and 2 q + 1 in its two steps of 128:
// the order along K is free as long as both operands share it, and its two scale bytes are neighbours.
// The operands enter the MFMA swapped, so that a lane holds four consecutive columns of one row of c.
//
// K past the end: chunks repeat the row's last one (codes are finite) and both scales are 2^-127, which makes
// their products 0 in fp32.
template <int MODE, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) mx_tile_kernel(MxArgs p, int row_tiles, int col_tiles) {
  constexpr int THREADS = WM * WN * 64, WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int ROWS = BM + BN, STAGE = ROWS * 136;
  static_assert(ROWS % (8 * WAVES) == 0, "whole loads");
  extern __shared__ __align__(16) uint8_t lds[];  // per stage: codes [ROWS][128], scales [ROWS][8]

  // blocks go to the 8 XCDs in turn: each takes a run of tiles, in groups of 8 row tiles, column by column, so
  // that the tiles it runs at once share rows of a and of w in its L2
  const int tiles = row_tiles * col_tiles, per = (tiles + 7) / 8;
  const int id = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (((int)blockIdx.x >> 3) >= per || id >= tiles) return;
  const int group = id / (8 * col_tiles), in_group = id - group * 8 * col_tiles;
  const int group_rows = min(8, row_tiles - 8 * group);
  const int tm = 8 * group + in_group % group_rows, tn = in_group / group_rows;
  if (MODE != kMxDense && tm >= p.tile_count[0]) return;
  const MxRows t = mx_rows<MODE, BM>(p, tm);
  constexpr int COLS = MODE == kMxGateUp ? BN / 2 : BN;
  const int n0 = tn * COLS;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int KB = p.K / 32, stages = (KB + 7) / 8;
  const uint8_t* w = p.w + (int64_t)t.expert * p.wrows * (p.K / 2);
  const uint8_t* ws = p.ws + (int64_t)t.expert * p.wrows * KB;

  // Row i of the stage (a's rows, then w's) times KB: its scales' offset in bytes, its codes' in 16 bytes.
  // 32 bits hold it (checked on the host).
  auto row_offset = [&](int i) -> uint32_t {
    if (i < BM) return (uint32_t)mx_a_row<MODE>(p, t, i) * (uint32_t)KB;
    const int j = i - BM;
    uint32_t row;
    if constexpr (MODE == kMxGateUp) row = (uint32_t)(min(n0 + (j < COLS ? j : j - COLS), p.N - 1) + (j < COLS ? 0 : p.N));
    else row = (uint32_t)min(n0 + j, p.N - 1);
    return row * (uint32_t)KB;
  };
  // this thread's loads: LOADS chunks of codes, A_LOADS of them a's, and the scales of SROWS rows
  constexpr int LOADS = ROWS / (8 * WAVES), A_LOADS = BM / (8 * WAVES), SROWS = (ROWS + THREADS - 1) / THREADS;
  static_assert(BM % (8 * WAVES) == 0, "whole loads");
  uint32_t src[LOADS], ssrc[SROWS];
  const int place = (lane & 7) ^ (lane >> 3);  // row & 7 is lane >> 3
#pragma unroll
  for (int u = 0; u < LOADS; ++u) src[u] = row_offset((u * WAVES + wave) * 8 + (lane >> 3));
#pragma unroll
  for (int u = 0; u < SROWS; ++u) ssrc[u] = row_offset(min(tid + u * THREADS, ROWS - 1));
  u32x2 sv[SROWS];
  auto fetch = [&](int s) {
    uint8_t* base = lds + (s & 1) * STAGE;
    const int chunk = min(8 * s + place, KB - 1);
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
      lds_load16((u < A_LOADS ? p.a : w) + (uint64_t)(src[u] + (uint32_t)chunk) * 16, base + (u * WAVES + wave) * 1024);
    if (8 * s + 8 <= KB) {
#pragma unroll
      for (int u = 0; u < SROWS; ++u) __builtin_memcpy(&sv[u], (tid + u * THREADS < BM ? p.as : ws) + ssrc[u] + 8 * s, 8);
    } else {
#pragma unroll
      for (int u = 0; u < SROWS; ++u) {
        sv[u] = u32x2{0u, 0u};
        const uint8_t* from = (tid + u * THREADS < BM ? p.as : ws) + ssrc[u] + 8 * s;
#pragma unroll
        for (int b = 0; b < 7; ++b)
          if (b < KB - 8 * s) sv[u][b >> 2] |= (uint32_t)from[b] << (8 * (b & 3));
      }
    }
  };
  auto put_scales = [&](int s) {
    uint8_t* base = lds + (s & 1) * STAGE + ROWS * 128;
#pragma unroll
    for (int u = 0; u < SROWS; ++u)
      if (tid + u * THREADS < ROWS) *(u32x2*)(base + (tid + u * THREADS) * 8) = sv[u];
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int m0 = (wave / WN) * TM * 16, c0 = BM + (wave % WN) * TN * 16;
  fetch(0);
  put_scales(0);
  __syncthreads();
  for (int s = 0; s < stages; ++s) {
    if (s + 1 < stages) fetch(s + 1);
    const uint8_t* base = lds + (s & 1) * STAGE;
    uint32_t sa[TM], sb[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = *(const uint16_t*)(base + ROWS * 128 + (m0 + 16 * i + r) * 8 + 2 * q);
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] = *(const uint16_t*)(base + ROWS * 128 + (c0 + 16 * j + r) * 8 + 2 * q);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      u32x4 a[TM], b[TN];
      const int at = ((2 * q + k) ^ (r & 7)) * 16;
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = *(const u32x4*)(base + (m0 + 16 * i + r) * 128 + at);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = *(const u32x4*)(base + (c0 + 16 * j + r) * 128 + at);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = k == 0 ? mx_mfma<0, 0>(b[j], a[i], acc[i][j], sb[j], sa[i]) : mx_mfma<1, 1>(b[j], a[i], acc[i][j], sb[j], sa[i]);
    }
    if (s + 1 < stages) put_scales(s + 1);
    __syncthreads();
  }

  // lane: row m0 + 16 i + r, columns 16 j + 4 q .. + 3
  if constexpr (MODE == kMxGateUp) {
    // the waves of the gate half and of the up half hold the same places of different columns: up goes through
    // LDS, [BM][COLS] fp32, then each wave of the gate half forms h
    float* up = (float*)lds;
    const int cw = (wave % WN) * TN * 16;
    constexpr int LD = COLS + 4;
    if (cw >= COLS) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) *(f32x4*)(up + (m0 + 16 * i + r) * LD + cw - COLS + 16 * j + 4 * q) = acc[i][j];
    }
    __syncthreads();
    if (cw < COLS) {
      static_assert(TN % 2 == 0 && WN % 2 == 0, "blocks of 32 columns in a wave");
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = m0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
          float v[8];
          uint32_t top = 0;
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const f32x4 u = *(const f32x4*)(up + m * LD + cw + 16 * (j + d) + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float g = acc[i][j + d][e];
              v[4 * d + e] = (p.act == AWQ_MOE_ACT_GELU_TANH ? gated_act_fast<1>(g) : gated_act_fast<0>(g)) * u[e];
              top = max(top, mx_abs_bits(v[4 * d + e]));
            }
          }
          top = max(top, (uint32_t)__shfl_xor((int)top, 16));
          top = max(top, (uint32_t)__shfl_xor((int)top, 32));
          const uint32_t byte = mx_scale_byte(top);
          const uint32_t codes = byte == 255u ? 0u : mx_codes8(v, mx_scale_value(byte));
          const int c = n0 + cw + 16 * j;
          if (m < t.rows && c < p.N) {
            uint8_t* o = p.h + (int64_t)(t.first + m) * (p.N / 2) + c / 2 + 2 * q;
            *(uint16_t*)o = (uint16_t)codes;
            *(uint16_t*)(o + 8) = (uint16_t)(codes >> 16);
            if (q == 0) p.hs[(int64_t)(t.first + m) * (p.N / 32) + c / 32] = (uint8_t)byte;
          }
        }
      }
    }
  } else if constexpr (MODE == kMxDown) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = m0 + 16 * i + r;
      if (m >= t.rows) continue;
      float* y = p.y + (int64_t)p.order[t.first + m] * p.N;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + c0 - BM + 16 * j + 4 * q;
        if (n < p.N) *(f32x4*)(y + n) = acc[i][j];
      }
    }
  } else {
    const bool whole = (p.ldc & 3) == 0 && ((uintptr_t)p.c & 7) == 0;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + c0 - BM + 16 * j + 4 * q;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = n + e < p.N ? load_bias(p.bias, p.bias_dtype, n + e) : 0.f;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = m0 + 16 * i + r;
        if (m >= t.rows) continue;
        uint16_t* at = p.c + (int64_t)(t.first + m) * p.ldc + n;
        uint16_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = p.out_bf16 ? f2bf_bits(acc[i][j][e] + bias[e]) : f2h_bits(acc[i][j][e] + bias[e]);
        if (whole && n + 4 <= p.N) {
          *(u32x2*)at = u32x2{(uint32_t)o[0] | ((uint32_t)o[1] << 16), (uint32_t)o[2] | ((uint32_t)o[3] << 16)};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.N) at[e] = o[e];
        }
      }
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

template <int MODE, int BM, int BN, int WM, int WN>
static int launch_tile(const MxArgs& p, int64_t row_tiles, hipStream_t st) {
  constexpr int COLS = MODE == kMxGateUp ? BN / 2 : BN;
  const int64_t col_tiles = cdiv(p.N, COLS);
  if (row_tiles * col_tiles > 0x7FFFFFF0LL) return AWQ_ERR_UNSUPPORTED;
  constexpr int lds = 2 * (BM + BN) * 136;
  static_assert(MODE != kMxGateUp || BM * (BN / 2 + 4) * 4 <= lds, "the up half");
  auto kernel = mx_tile_kernel<MODE, BM, BN, WM, WN>;
  if (lds > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    (void)hipGetLastError();
    return AWQ_ERR_LAUNCH;
  }
  kernel<<<dim3((unsigned)(cdiv(row_tiles * col_tiles, 8) * 8)), dim3(WM * WN * 64), lds, st>>>(p, (int)row_tiles, (int)col_tiles);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

int launch_mx_tile_gemm(const MxArgs& p, hipStream_t st) {
  const int64_t big = cdiv(p.M, 256) * cdiv(p.N, 256), mid = cdiv(p.M, 128) * cdiv(p.N, 128);
  if (big >= 256) return launch_tile<kMxDense, 256, 256, 2, 4>(p, cdiv(p.M, 256), st);
  if (mid >= 256) return launch_tile<kMxDense, 128, 128, 2, 2>(p, cdiv(p.M, 128), st);
  return launch_tile<kMxDense, 64, 64, 2, 2>(p, cdiv(p.M, 64), st);
}

int launch_mx_tile_grouped(const MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st) {
  if (rows == 128)
    return gate_up ? launch_tile<kMxGateUp, 128, 128, 2, 2>(p, row_tiles, st) : launch_tile<kMxDown, 128, 128, 2, 2>(p, row_tiles, st);
  return gate_up ? launch_tile<kMxGateUp, 64, 128, 2, 2>(p, row_tiles, st) : launch_tile<kMxDown, 64, 128, 2, 2>(p, row_tiles, st);
}

}  // namespace awq_host
