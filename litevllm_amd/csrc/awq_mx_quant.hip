// Quantisation to microscaled fp4 and back (the format: awq_mx_common.h).
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kQuantThreads = 256;

// Eight values per lane, consecutive lanes consecutive pieces, nothing kept.  One pass: what it reads and writes bounds it
// ([2048, 12288] bf16 11 us, 5.8 TB/s, partly from the caches; [11008, 4128] fp32 46.7 us, 4.4 TB/s).
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes,
                                                                    uint8_t* __restrict__ scales, int64_t lds, int64_t pieces, uint32_t per_row) {
  const int64_t i = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  if (i >= pieces) return;  // whole blocks of 32: pieces % 4 == 0
  const int64_t row = per_row ? i / per_row : 0;  // 0: all one row, as the rows follow each other here and there
  mx_quantize8<T>(x + row * ldx, codes + row * per_row * 4, scales + row * lds, i - row * per_row);
}

// Eight values per lane.  An e2m1 value has two significant bits: times the scale it is exact in fp32
// (and below fp32's range or above it as the multiplication rounds), then rounded once to the output.  Bound by what it
// writes ([2048, 12288] to bf16 13 us, 4.9 TB/s; [11008, 4128] to fp32 34 us, 6.1 TB/s).
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
  if (dtype == AWQ_DTYPE_F16) mx_quantize_kernel<f16><<<grid, block, 0, st>>>((const f16*)x, ldx, codes, scales, lds, pieces, per_row);
  else if (dtype == AWQ_DTYPE_BF16) mx_quantize_kernel<bf16><<<grid, block, 0, st>>>((const bf16*)x, ldx, codes, scales, lds, pieces, per_row);
  else mx_quantize_kernel<float><<<grid, block, 0, st>>>((const float*)x, ldx, codes, scales, lds, pieces, per_row);
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
