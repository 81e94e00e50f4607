// Quantisation to microscaled fp4 and back (the format: awq_mx_common.h).
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kQuantThreads = 256;

// Eight values per lane: the four lanes of a block of 32 share its largest magnitude by two DPP steps
// inside their quad.  One pass: what it reads and writes bounds it.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint32_t* __restrict__ codes,
                                                                    uint8_t* __restrict__ scales, int64_t lds, int64_t pieces, uint32_t per_row) {
  const int64_t i = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  if (i >= pieces) return;  // whole blocks: pieces % 4 == 0
  const T* at = x + i * 8;
  int64_t block = i >> 2;
  if (per_row) {  // rows apart, here or there
    const int64_t row = i / per_row;
    at = x + row * ldx + (i - row * per_row) * 8;
    block = row * lds + ((i - row * per_row) >> 2);
  }
  float v[8];
  if constexpr (std::is_same<T, float>::value) load8<float>(at, v);
  else load8<T>(at, v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, mx_abs_bits(v[j]));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));
  const uint32_t byte = mx_scale_byte(top);
  codes[i] = byte == 255u ? 0u : mx_codes8(v, mx_scale_value(byte));
  if ((i & 3) == 0) scales[block] = (uint8_t)byte;
}

// Eight values per lane.  An e2m1 value has two significant bits: times the scale it is exact in fp32
// (and below fp32's range or above it as the multiplication rounds), then rounded once to the output.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                                      const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                                      int64_t pieces) {
  const int64_t i = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  if (i >= pieces) return;
  const uint32_t c = codes[i], byte = scales[i >> 2];
  const float s = byte == 255u ? __builtin_nanf("") : mx_scale_value(byte);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t n = (c >> (4 * j)) & 15u;
    // e2m1 bits moved into an fp32: exponent field 1 .. 3 is 2^0 .. 2^2; field 0 is mantissa / 2
    const uint32_t e = (n >> 1) & 3u, m = n & 1u;
    const float size = e ? __builtin_bit_cast(float, ((e + 126u) << 23) | (m << 22)) : 0.5f * (float)m;
    v[j] = (n & 8u ? -size : size) * s;
  }
  if constexpr (std::is_same<T, float>::value) {
    f32x4* o = (f32x4*)(out + i * 8);
    o[0] = f32x4{v[0], v[1], v[2], v[3]};
    o[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
    *(u32x4*)(out + i * 8) = o;
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

int launch_mx_quantize(const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t lds, int64_t M, int64_t K, int dtype,
                       hipStream_t st) {
  const int64_t pieces = M * (K / 8);
  if (pieces <= 0) return AWQ_OK;
  if (cdiv(pieces, kQuantThreads) > 0x7FFFFFFFLL) return AWQ_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)cdiv(pieces, kQuantThreads)), block(kQuantThreads);
  const uint32_t per_row = ((ldx == K && lds == K / 32) || M == 1) ? 0u : (uint32_t)(K / 8);
  auto* o = (uint32_t*)codes;
  if (dtype == AWQ_DTYPE_F16) mx_quantize_kernel<f16><<<grid, block, 0, st>>>((const f16*)x, ldx, o, scales, lds, pieces, per_row);
  else if (dtype == AWQ_DTYPE_BF16) mx_quantize_kernel<bf16><<<grid, block, 0, st>>>((const bf16*)x, ldx, o, scales, lds, pieces, per_row);
  else mx_quantize_kernel<float><<<grid, block, 0, st>>>((const float*)x, ldx, o, scales, lds, pieces, per_row);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

int launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int64_t M, int64_t K, int dtype, hipStream_t st) {
  const int64_t pieces = M * (K / 8);
  if (pieces <= 0) return AWQ_OK;
  if (cdiv(pieces, kQuantThreads) > 0x7FFFFFFFLL) return AWQ_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)cdiv(pieces, kQuantThreads)), block(kQuantThreads);
  const auto* c = (const uint32_t*)codes;
  if (dtype == AWQ_DTYPE_F16) mx_dequantize_kernel<f16><<<grid, block, 0, st>>>(c, scales, (f16*)out, pieces);
  else if (dtype == AWQ_DTYPE_BF16) mx_dequantize_kernel<bf16><<<grid, block, 0, st>>>(c, scales, (bf16*)out, pieces);
  else mx_dequantize_kernel<float><<<grid, block, 0, st>>>(c, scales, (float*)out, pieces);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
