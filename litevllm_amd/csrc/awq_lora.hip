// Low-rank adapters of many requests, added to what a shared projection gave:
//
//   l = ids[m];  v[m] = s_l x[m] A_l^T  (rank values);  out[m] = base[m] + v[m] B_l^T;  out[m] = base[m] without an adapter
//
// Two launches: the ranks (x and A once, fp32 sums, K in shares that the second launch adds in order) and the columns (base and
// B once).  Rows go in tiles of 16 (columns: 16 MT) that the matrix cores take; a tile looks up which adapters its rows have and
// runs once for each: once where the rows of a request lie together, as in prompts, up to 16 times in a batch of single
// tokens, where blocks (`slots`) share these.  A product's rows do not mix, so the other rows of a tile only cost idle lanes.
//
// v enters the second product as two 16-bit numbers of sum v 2^-e (the row's own e puts its largest value at 2^13 .. 2^14,
// so nothing passes fp16's range): 16 bits of mantissa at least for bf16, 21 for fp16, and one rounding for the output.  Both
// halves meet the same B in one instruction of depth 32: 16 ranks, high parts then low parts.
#include <algorithm>

#include "awq_launch.h"

namespace awq {

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any address of a 16-bit element

struct LoraArgs {
  const uint16_t *base, *x, *a, *b;
  const void* ids;
  const float* scales;
  uint16_t* out;
  float* v;  // [splits][M][ranks]
  int64_t ldb, ldx, ldo, a_stride, b_stride;
  int64_t M;
  int N, K, R, L, id64;
  int ranks;        // R in whole tiles of 16
  int slots;        // blocks that share a row tile's adapters
  int splits, per;  // shares of K, each of `per` units of 64
  int cols;         // columns of a block, a multiple of 256
};

__device__ __forceinline__ int lora_id(const LoraArgs& p, int64_t m) {
  const int64_t l = p.id64 ? ((const int64_t*)p.ids)[m] : (int64_t)((const int32_t*)p.ids)[m];
  return l >= 0 && l < p.L ? (int)l : -1;
}
// Eight elements of which the first n exist, zeros behind them.
__device__ __forceinline__ u32x4 load8_to(const uint16_t* at, int n) {
  if (n >= 8) return *(const u32x4_any*)at;
  u32x4 v = {0, 0, 0, 0};
  for (int i = 0; i < n; ++i) v[i >> 1] |= (uint32_t)at[i] << (16 * (i & 1));
  return v;
}

// ------------------------------------------------------------------ ranks
constexpr int kUnit = 64;  // values of K that a wave takes at once: whole lines of both operands

// RT tiles of 16 ranks by a tile of 16 rows and a share of K.  Waves take units in turn; lane (q, i) holds values
// 16 q .. 16 q + 15 of a unit for rank i and for row i, the results are ranks 4 q .. 4 q + 3 of row i.
template <typename T, int RT>
__global__ void __launch_bounds__(256) lora_ranks_kernel(LoraArgs p) {
  __shared__ f32x4 part[4][RT][64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15;
  const int tile = blockIdx.x / p.slots, slot = blockIdx.x - tile * p.slots, split = blockIdx.y, r0 = blockIdx.z * RT * 16;
  const int64_t m = (int64_t)tile * 16 + i;
  const bool exists = m < p.M;
  const int id = exists ? lora_id(p, m) : -1;
  const uint16_t* const x = p.x + (exists ? m : p.M - 1) * p.ldx;
  uint64_t left = __ballot(lane < 16 && id >= 0);
  for (int n = 0; left; ++n) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    left &= ~__ballot(lane < 16 && id == cur);
    if (n % p.slots != slot) continue;
    const uint16_t* a[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) a[r] = p.a + cur * p.a_stride + (int64_t)min(r0 + 16 * r + i, p.R - 1) * p.K;
    f32x4 acc[RT] = {};
    const int first = split * p.per, units = min(first + p.per, (p.K + kUnit - 1) / kUnit), whole = min(units, p.K / kUnit);
#pragma unroll 2
    for (int u = first + wave; u < whole; u += 4) {
      const int k = u * kUnit + 16 * q;
      const u32x4 x0 = *(const u32x4_any*)(x + k), x1 = *(const u32x4_any*)(x + k + 8);
      u32x4 a0[RT], a1[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) a0[r] = *(const u32x4_any*)(a[r] + k), a1[r] = *(const u32x4_any*)(a[r] + k + 8);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        acc[r] = MfmaOp<T>::run(a0[r], x0, acc[r]);
        acc[r] = MfmaOp<T>::run(a1[r], x1, acc[r]);
      }
    }
    if (whole < units && (whole - first) % 4 == wave) {
      const int k = whole * kUnit + 16 * q, n8 = p.K - k;
      const u32x4 x0 = load8_to(x + k, n8), x1 = load8_to(x + k + 8, n8 - 8);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        acc[r] = MfmaOp<T>::run(load8_to(a[r] + k, n8), x0, acc[r]);
        acc[r] = MfmaOp<T>::run(load8_to(a[r] + k + 8, n8 - 8), x1, acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) part[wave][r][lane] = acc[r];
    __syncthreads();
    if (id == cur) {
      for (int r = wave; r < RT; r += 4) {
        const f32x4 s = (part[0][r][lane] + part[1][r][lane]) + (part[2][r][lane] + part[3][r][lane]);
        const int at = r0 + 16 * r + 4 * q;
        if (at < p.ranks) *(f32x4*)(p.v + ((int64_t)split * p.M + m) * p.ranks + at) = s;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ columns
__device__ __forceinline__ float row_max16(float v) {  // over the 16 lanes of a row
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0xB1>{}));
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x4E>{}));
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x141>{}));
  return fmaxf(v, dpp(v, std::integral_constant<int, 0x140>{}));
}

// Sixteen columns of a row, of which `n` exist.
template <typename T>
__device__ __forceinline__ void finish16(const LoraArgs& p, int64_t m, int col, int n, const float (&delta)[16]) {
  const uint16_t* const from = p.base ? p.base + m * p.ldb + col : nullptr;
  uint16_t* const to = p.out + m * p.ldo + col;
  if (n >= 16) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 o, b = {0, 0, 0, 0};
      if (from) b = *(const u32x4_any*)(from + 8 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = pack2<T>(delta[8 * h + 2 * j] + from_bits<T>((uint16_t)(b[j] & 0xFFFF)),
                        delta[8 * h + 2 * j + 1] + from_bits<T>((uint16_t)(b[j] >> 16)));
      *(u32x4_any*)(to + 8 * h) = o;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) to[j] = to_bits<T>(delta[j] + (from ? from_bits<T>(from[j]) : 0.f));
  }
}

// 16 MT rows by p.cols columns.  A wave takes 64 columns at a time as four tiles of 16, tile c of them the columns
// 16 (i / 4) + 4 c + i % 4, so that lane (q, i) ends with the sixteen columns 16 q .. 16 q + 15 of row i.  RT tiles of 16 ranks
// at a time.
template <typename T, int RT, int MT>
__global__ void __launch_bounds__(256) lora_columns_kernel(LoraArgs p) {
  constexpr int ROWS = 16 * MT;
  // [ROWS][ld]: of each tile of ranks its high parts, then its low parts; rows lie 16 bytes apart from whole banks
  extern __shared__ u32x4 dynamic_lds[];
  __shared__ int exponent[ROWS];
  uint16_t* const v = (uint16_t*)dynamic_lds;
  const int chunks = (p.ranks / 16 + RT - 1) / RT, ld = 32 * RT * chunks + 8;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15;
  const int tile = blockIdx.x / p.slots, slot = blockIdx.x - tile * p.slots;
  const int64_t m0 = (int64_t)tile * ROWS;
  const bool exists = lane < ROWS && m0 + lane < p.M;
  const int id = exists ? lora_id(p, m0 + lane) : -1;
  const int end = min((int)(blockIdx.y + 1) * p.cols, p.N);
  uint64_t left = __ballot(exists);
  for (int n = 0; left; ++n) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t rows = __ballot(exists && id == cur);
    left &= ~rows;
    if (n % p.slots != slot) continue;
    if (cur < 0) {
      if (p.out == p.base && p.ldo == p.ldb) continue;  // in place already
      const float zero[16] = {};
      for (int c0 = blockIdx.y * p.cols + wave * 64; c0 < end; c0 += 256)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          if (rows >> (16 * mt + i) & 1) finish16<T>(p, m0 + 16 * mt + i, c0 + 16 * q, end - c0 - 16 * q, zero);
      continue;
    }
    const float scale = p.scales ? p.scales[cur] : 1.f;
    __syncthreads();  // v of the adapter before is read
    for (int row = t >> 4; row < ROWS; row += 16) {
      const bool mine = rows >> row & 1;
      float f[RT], top = 0.f;
      auto load = [&](int chunk) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int at = 16 * (chunk * RT + r) + i;
          f[r] = 0.f;
          if (!mine || at >= p.R) continue;
          for (int s = 0; s < p.splits; ++s) f[r] += p.v[((int64_t)s * p.M + m0 + row) * p.ranks + at];
          f[r] *= scale;
        }
      };
      for (int chunk = chunks - 1; chunk >= 0; --chunk) {
        load(chunk);
#pragma unroll
        for (int r = 0; r < RT; ++r) top = fmaxf(top, fabsf(f[r]));
      }
      top = row_max16(top);
      const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 13;
      if (i == 0) exponent[row] = e;
      for (int chunk = 0; chunk < chunks; ++chunk) {
        if (chunk) load(chunk);  // the first is there
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float s = ldexpf(f[r], -e);
          const uint16_t hi = to_bits<T>(s);
          uint16_t* const to = v + row * ld + 32 * (chunk * RT + r) + i;
          to[0] = hi;
          to[16] = fabsf(s) < __builtin_inff() ? to_bits<T>(s - from_bits<T>(hi)) : (uint16_t)0;
        }
      }
    }
    __syncthreads();
    int ex[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) ex[mt] = exponent[16 * mt + i];
    const uint16_t* const b = p.b + cur * p.b_stride;
    for (int c0 = blockIdx.y * p.cols + wave * 64; c0 < end; c0 += 256) {
      f32x4 acc[MT][4] = {};
      for (int chunk = 0; chunk < chunks; ++chunk) {
        u32x4 bv[4][RT];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint16_t* const row = b + (int64_t)min(c0 + 16 * (i >> 2) + 4 * c + (i & 3), p.N - 1) * p.R;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const int at = 16 * (chunk * RT + r) + 8 * (q & 1);
            bv[c][r] = load8_to(row + at, p.R - at);
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const u32x4 low = *(const u32x4*)(v + (16 * mt + i) * ld + 32 * (chunk * RT + r) + 8 * q);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[mt][c] = MfmaOp<T>::run(bv[c][r], low, acc[mt][c]);
          }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float delta[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) delta[j] = ldexpf(acc[mt][j >> 2][j & 3], ex[mt]);
        if (rows >> (16 * mt + i) & 1) finish16<T>(p, m0 + 16 * mt + i, c0 + 16 * q, end - c0 - 16 * q, delta);
      }
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

struct LoraPlan {
  int tiles, slots, splits, per, ranks;
};
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t R) {
  LoraPlan l{};
  l.tiles = (int)cdiv(M, 16);
  l.ranks = (int)cdiv(R, 16) * 16;
  // a batch of single tokens has many adapters in a tile, prompts one or two
  l.slots = M <= 128 ? (int)std::min<int64_t>(16, M) : 1;
  const int64_t units = cdiv(K, kUnit), want = std::max<int64_t>(1, 512 / ((int64_t)l.tiles * l.slots));
  l.per = (int)std::max<int64_t>(4, cdiv(cdiv(units, std::min<int64_t>(want, 16)), 4) * 4);
  l.splits = (int)cdiv(units, l.per);
  return l;
}
size_t lora_workspace_bytes(int64_t M, int64_t K, int64_t R) {
  const LoraPlan l = lora_plan(M, K, R);
  return (size_t)l.splits * (size_t)M * (size_t)l.ranks * 4;
}

template <typename T>
static int lora_typed(LoraArgs p, const LoraPlan& l, hipStream_t st) {
  const int rt = l.ranks / 16;
  auto ranks = [&](auto n) {
    constexpr int RT = decltype(n)::value;
    lora_ranks_kernel<T, RT><<<dim3((unsigned)(l.tiles * l.slots), (unsigned)l.splits, (unsigned)cdiv(rt, RT)), 256, 0, st>>>(p);
  };
  using std::integral_constant;
  if (rt == 1) ranks(integral_constant<int, 1>{});
  else if (rt == 2) ranks(integral_constant<int, 2>{});
  else ranks(integral_constant<int, 4>{});
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  auto columns = [&](auto n, auto mt) {
    constexpr int RT = decltype(n)::value, MT = decltype(mt)::value;
    const int64_t tiles = cdiv(p.M, 16 * MT), want = std::max<int64_t>(1, 1024 / (tiles * p.slots));
    p.cols = (int)(cdiv(cdiv(p.N, 256), std::min<int64_t>(want, cdiv(p.N, 256))) * 256);
    const size_t lds = (size_t)16 * MT * (32 * cdiv(rt, RT) * RT + 8) * 2;
    lora_columns_kernel<T, RT, MT><<<dim3((unsigned)(tiles * p.slots), (unsigned)cdiv(p.N, p.cols)), 256, lds, st>>>(p);
  };
  auto by_rank = [&](auto mt) {
    if (rt == 1) columns(integral_constant<int, 1>{}, mt);
    else if (rt == 2) columns(integral_constant<int, 2>{}, mt);
    else columns(integral_constant<int, 4>{}, mt);
  };
  if (p.M <= 512) by_rank(integral_constant<int, 1>{});
  else by_rank(integral_constant<int, 4>{});
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

int launch_lora(const LoraCall& c, hipStream_t st) {
  const LoraPlan l = lora_plan(c.M, c.K, c.R);
  LoraArgs p{};
  p.base = (const uint16_t*)c.base, p.x = (const uint16_t*)c.x, p.a = (const uint16_t*)c.a, p.b = (const uint16_t*)c.b;
  p.ids = c.ids, p.scales = c.scales, p.out = (uint16_t*)c.out, p.v = (float*)c.workspace;
  p.ldb = c.ldb, p.ldx = c.ldx, p.ldo = c.ldo, p.a_stride = c.a_stride, p.b_stride = c.b_stride;
  p.M = c.M, p.N = (int)c.N, p.K = (int)c.K, p.R = (int)c.R, p.L = c.L, p.id64 = c.id64;
  p.ranks = l.ranks, p.slots = l.slots, p.splits = l.splits, p.per = l.per;
  return c.dtype == AWQ_DTYPE_F16 ? lora_typed<f16>(p, l, st) : lora_typed<bf16>(p, l, st);
}

}  // namespace awq_host
