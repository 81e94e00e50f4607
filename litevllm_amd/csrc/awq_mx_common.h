// Device helpers of the microscaled fp4 (MXFP4) kernels.
//
// Format (OCP Microscaling Formats, version 1.0): 32 consecutive values along K share a scale
// 2^(byte - 127) (byte 255: the block stands for NaN); a value is an e2m1 code -- sign, two exponent
// bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A [rows, K] matrix is codes [rows, K/2] bytes
// (the even index in the low nibble) and scales [rows, K/32] bytes, as checkpoints hold it.
//
// The scaled MFMA of gfx950 takes 16 x 128 and 128 x 16 operands in this order: lane l = 16 q + r
// holds the 16 bytes of codes of row r, block q of the step's four, and that block's scale byte; the
// four results of a lane are rows 4 q .. 4 q + 3 of column r.  The raw matrices therefore serve as they
// are.  Its sums hold to a few 1e-7 of the sum of magnitudes (scales 2^50 apart measured 3e-8), a scale
// byte of 255 gives NaN, and 0 and 254 are exact.
#pragma once

#include "awq_common.h"

namespace awq {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// c += a . b^T over 128 values of K.  sa / sb: scale bytes in the low eight bits.
__device__ __forceinline__ f32x4 mx_mfma(const u32x4& a, const u32x4& b, const f32x4& c, uint32_t sa, uint32_t sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// Scale byte of a block whose largest magnitude has these bits (sign clear; they order like the
// values, NaN above Inf): floor(log2) - 2 puts it in [4, 8), what passes 6 saturates.  Subnormal and
// zero: the smallest scale.  Inf or NaN: 255.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {  // 2^(byte - 127), byte < 255
  return __builtin_bit_cast(float, byte == 0u ? 0x00400000u : byte << 23);
}
// Codes of eight values (value i in nibble i), each x / scale rounded to nearest even, saturated.
__device__ __forceinline__ uint32_t mx_codes8(const float* x, float scale) {
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[0], x[1], scale, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[2], x[3], scale, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[4], x[5], scale, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[6], x[7], scale, 3);
  return o;
}
__device__ __forceinline__ uint32_t mx_abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// Eight consecutive values as fp32.
template <typename T>
__device__ __forceinline__ void load8(const void* p, float* v) {
  if constexpr (std::is_same<T, float>::value) {
    const f32x4 a = ((const f32x4*)p)[0], b = ((const f32x4*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
    const u32x4 a = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = from_bits<T>((uint16_t)(a[i] & 0xFFFF));
      v[2 * i + 1] = from_bits<T>((uint16_t)(a[i] >> 16));
    }
  }
}

// Eight values of a row, number `piece`, by a lane; the four lanes of a block of 32 share its largest magnitude by two
// DPP steps inside their quad.
template <typename T, typename Piece>
__device__ __forceinline__ void mx_quantize8(const void* x, uint8_t* codes, uint8_t* scales, Piece piece) {
  float v[8];
  load8<T>((const char*)x + piece * (Piece)(8 * sizeof(T)), v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, mx_abs_bits(v[j]));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));
  const uint32_t byte = mx_scale_byte(top);
  *(uint32_t*)(codes + piece * 4) = byte == 255u ? 0u : mx_codes8(v, mx_scale_value(byte));
  if ((piece & 3) == 0) scales[piece >> 2] = (uint8_t)byte;
}

// h of one value: act(gate) * up in fp32.
__device__ __forceinline__ float mx_gated(float g, float u, int act) {
  return (act == AWQ_MOE_ACT_GELU_TANH ? gated_act_fast<1>(g) : gated_act_fast<0>(g)) * u;
}

// One product of MXFP4 matrices: rows of `a` by rows of `w`.  Which rows, and where the sums go:
//   kMxDense: c[m, n] = sum (+ bias), one rounding to 16 bits.
//   kMxGateUp: a tile table row {expert, first, rows} names `rows` consecutive places of `order`; the
//     row at place p is token order[p] / topk of a; gate and up rows of the expert are n and I + n;
//     h = act(gate) * up, quantised per 32 columns, goes to row p of h / hs.
//   kMxDown: the same places; a's rows are the places themselves (the h above), the fp32 sum goes to
//     row order[p] of y.
enum MxMode { kMxDense = 0, kMxGateUp = 1, kMxDown = 2 };

struct MxArgs {
  const uint8_t *a, *as;  // codes [rows, K/2], scales [rows, as_ld]
  const uint8_t *w, *ws;  // codes [experts][wrows, K/2], scales [experts][wrows, K/32]
  int K, N, M;            // N: output columns (gate_up: I)
  int as_ld;              // bytes between rows of a's scales; a multiple of 4 for gate_up
  int64_t wrows, a_rows;  // rows of w per expert; rows of a
  // dense
  uint16_t* c;
  int64_t ldc;
  const void* bias;
  int bias_dtype, out_bf16;
  // grouped
  const int *tiles, *tile_count, *order;
  int topk, act;
  uint8_t *h, *hs;
  float* y;
  // a in 16 bits, quantised by the blocks themselves: at most xrows rows a block
  const uint16_t* x;
  int64_t ldx;
  int xrows;
  // few routes, without a table
  const void* ids;
  int id64, routes, experts;
};
constexpr int kMxScanRoutes = 64;  // of a call without a table

__device__ __forceinline__ int64_t mx_route_id(const void* ids, int id64, int64_t r) {
  return id64 ? ((const int64_t*)ids)[r] : (int64_t)((const int32_t*)ids)[r];
}
__device__ __forceinline__ float mx_route_weight(const void* w, int dtype, int64_t r) {
  if (dtype == AWQ_DTYPE_F32) return ((const float*)w)[r];
  const uint16_t b = ((const uint16_t*)w)[r];
  return dtype == AWQ_DTYPE_F16 ? h_bits2f(b) : bf_bits2f(b);
}

// The rows that a block works on.
struct MxRows {
  int expert, first, rows;
};
template <int MODE, int ROWS>
__device__ __forceinline__ MxRows mx_rows(const MxArgs& p, int tile) {
  if constexpr (MODE == kMxDense) {
    const int first = tile * ROWS;
    return {0, first, p.M - first < ROWS ? p.M - first : ROWS};
  } else {
    const auto* row = (const __attribute__((address_space(4))) int*)p.tiles + 3 * tile;  // constant here: scalar loads
    return {row[0], row[1], row[2]};
  }
}
// Row of a for row r of the block of a table's or a dense tile (rows past the end repeat the last: their results are dropped).
template <int MODE>
__device__ __forceinline__ int64_t mx_a_row(const MxArgs& p, const MxRows& t, int r) {
  const int at = t.first + (r < t.rows ? r : t.rows - 1);
  if constexpr (MODE == kMxGateUp) return p.order[at] / p.topk;
  return at;
}

}  // namespace awq

namespace awq_host {
int launch_mx_tile_gemm(const awq::MxArgs& p, hipStream_t st);
int launch_mx_rows_gemm(const awq::MxArgs& p, hipStream_t st);
bool mx_quantizes_itself(int64_t M, int64_t K);  // whether launch_mx_rows_gemm takes a in 16 bits (p.x)
bool mx_takes_rows(int64_t M, int64_t N, int64_t K);  // whether launch_mx_rows_gemm is the kernel of the size
// gate_up or down product of the grouped routes in `row_tiles` (at most) row tiles of `rows` rows
int launch_mx_grouped(const awq::MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st);
int launch_mx_tile_grouped(const awq::MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st);
// the same for at most kMxScanRoutes routes, without a table; down with the weighted sum
int launch_mx_scan_gate_up(const awq::MxArgs& p, hipStream_t st);
int launch_mx_down_combine(const awq::MxArgs& p, const void* weights, int w_dtype, void* out, int64_t ldo, hipStream_t st);
}  // namespace awq_host
