// Low-rank adapters of many requests, added to what a shared projection gave:
//
//   l = ids[m];  v[m] = s_l x[m] A_l^T  (rank values);  out[m] = base[m] + v[m] B_l^T;  out[m] = base[m] without an adapter
//
// Two launches: the ranks (x and A once, sums in fp32) and the columns (base and B once).  Rows go in tiles that the matrix cores
// take; a tile looks up which adapters its rows have and runs once for each: once where the rows of a request lie together,
// as in prompts, up to 16 times in a batch of single tokens, where blocks (`slots`) share these.  The matrix cores do not mix
// rows, so the other rows of a tile only cost idle lanes.
//
// v enters the second product as two 16-bit numbers, v = high + low: 16 bits of mantissa at least for bf16, 21 for fp16, and
// one rounding for the output.  Both halves meet the same B in one instruction of depth 32: 16 ranks, high parts then low
// parts.  fp16 takes v / 2^e instead, with an e of its own for 16 ranks of a row that puts the largest of them at 2^13 .. 2^14:
// v may pass fp16's range.
#include <algorithm>

#include "awq_launch.h"

namespace awq {

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any address of a 16-bit element

struct LoraArgs {
  const uint16_t *base, *x, *a, *b;
  const void* ids;
  const float* scales;
  uint16_t* out;
  float* partial;  // few rows: [splits][M][ranks], s_l not in it yet
  uint16_t* v;     // many rows: [M][2 ranks], of each 16 ranks the high parts, then the low parts
  float* powers;   // and [M][ranks / 16]: 2^e (fp16)
  int64_t ldb, ldx, ldo, a_stride, b_stride;
  int64_t M;
  int N, K, R, L, id64;
  int ranks;  // R in whole tiles of 16
  int slots;  // blocks that share a row tile's adapters
  int splits, per;  // shares of K, each of `per` units
  int cols;   // columns of a block
  int whole;  // columns that go by eight, see lora_whole
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
// The neighbouring lane's value (lanes 0 and 1 swap, 2 and 3, ...), and the largest of 16 lanes.
__device__ __forceinline__ u32x4 from_neighbour(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[i], 0xB1, 0xF, 0xF, true);
  return v;
}
__device__ __forceinline__ float row_max16(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0xB1>{}));
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x4E>{}));
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x141>{}));
  return fmaxf(v, dpp(v, std::integral_constant<int, 0x140>{}));
}

// v of a rank as its two parts, and 2^e; all 16 ranks of a row's tile in 16 neighbouring lanes.
struct Halves {
  uint16_t high, low;
  float power;
};
template <typename T>
__device__ __forceinline__ Halves halves_of(float f) {
  Halves h;
  h.power = 1.f;
  if constexpr (std::is_same<T, f16>::value) {
    const int e = (int)(__builtin_bit_cast(uint32_t, row_max16(fabsf(f))) >> 23) - 127 - 13;
    f = ldexpf(f, -e);
    h.power = ldexpf(1.f, e);
  }
  h.high = to_bits<T>(f);
  h.low = fabsf(f) < __builtin_inff() ? to_bits<T>(f - from_bits<T>(h.high)) : (uint16_t)0;  // no Inf - Inf
  return h;
}

// ------------------------------------------------------------------ ranks
constexpr int kUnit = 64;  // values of K that a wave takes at once: whole lines of both operands

// RT tiles of 16 ranks by a tile of 16 rows and a share of K, whose units the waves take in turn, D of them at a time; the
// waves' sums meet in LDS.  Loads cover whole lines, eight lanes each; a wave passes them through LDS of its own into the
// matrix cores' order, where lane (q, i) holds values 8 q .. 8 q + 7 and 32 + 8 q .. of rank i and of row i.  (Straight from
// memory in that order a load's neighbouring lanes are in different lines: 4096 rows, K = 4096, rank 64 42 us.)
// FINAL: the share is all of K, the parts of v go out; else the sums.
template <typename T, int RT, int WAVES, int D, bool FINAL>
__global__ void __launch_bounds__(64 * WAVES) lora_ranks_kernel(LoraArgs p) {
  constexpr int TILES = 1 + RT, LD = kUnit + 8;  // rows 16 bytes apart from whole banks
  union Lds {
    uint16_t stage[WAVES][D][TILES * 16][LD];
    f32x4 part[WAVES][RT][64];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15, r8 = lane >> 3, c8 = 8 * (lane & 7);
  const int tile = blockIdx.x / p.slots, slot = blockIdx.x - tile * p.slots, tile0 = blockIdx.y * RT;
  const int64_t m0 = (int64_t)tile * 16;
  const int id = m0 + i < p.M ? lora_id(p, m0 + i) : -1;
  const int begin = blockIdx.z * p.per, units = min(begin + p.per, (p.K + kUnit - 1) / kUnit);
  uint32_t left = (uint32_t)(__ballot(id >= 0) & 0xFFFF);
  for (int n = 0; left; ++n) {
    const int first = __builtin_ctz(left), cur = __builtin_amdgcn_readlane(id, first);
    const uint32_t rows = (uint32_t)(__ballot(id == cur) & 0xFFFF);
    left &= ~rows;
    if (n % p.slots != slot) continue;
    // two rows of each tile a lane; for rows of other adapters a row that is read anyway
    const uint16_t* from[TILES][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      from[0][h] = p.x + (m0 + (rows >> (r8 + 8 * h) & 1 ? r8 + 8 * h : first)) * p.ldx + c8;
#pragma unroll
      for (int r = 0; r < RT; ++r) from[1 + r][h] = p.a + cur * p.a_stride + (int64_t)min(16 * (tile0 + r) + r8 + 8 * h, p.R - 1) * p.K + c8;
    }
    u32x4 piece[D][TILES][2];
    auto load = [&](int u0) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int u = u0 + d * WAVES;
        if (u >= units) continue;
        const bool whole = u * kUnit + kUnit <= p.K;
#pragma unroll
        for (int j = 0; j < TILES; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint16_t* const at = from[j][h] + u * kUnit;
            piece[d][j][h] = whole ? *(const u32x4_any*)at : load8_to(at, p.K - u * kUnit - c8);
          }
      }
    };
    f32x4 acc[RT] = {};
    load(begin + wave);
    for (int u0 = begin + wave; u0 < units; u0 += D * WAVES) {
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int j = 0; j < TILES; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) *(u32x4*)&lds.stage[wave][d][16 * j + r8 + 8 * h][c8] = piece[d][j][h];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      load(u0 + D * WAVES);
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (u0 + d * WAVES >= units) continue;
#pragma unroll
        for (int k = 0; k < kUnit; k += 32) {
          const u32x4 x = *(const u32x4*)&lds.stage[wave][d][i][k + 8 * q];
#pragma unroll
          for (int r = 0; r < RT; ++r)
            acc[r] = MfmaOp<T>::run(*(const u32x4*)&lds.stage[wave][d][16 * (1 + r) + i][k + 8 * q], x, acc[r]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();  // all waves are done with their stages
    // ranks 4 q .. 4 q + 3 of row i
#pragma unroll
    for (int r = 0; r < RT; ++r) lds.part[wave][r][lane] = acc[r];
    __syncthreads();
    for (int at = t; at < RT * 256; at += 64 * WAVES) {
      const int r = at >> 8, row = at >> 4 & 15, rank = 16 * (tile0 + r) + i;  // i == at % 16
      float f = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) f += ((const float*)&lds.part[w][r][16 * (i >> 2) + row])[i & 3];
      if (rank >= p.ranks) continue;  // for the whole row
      const int64_t m = m0 + row;
      if constexpr (FINAL) {
        const Halves h = halves_of<T>(rank < p.R ? f * (p.scales ? p.scales[cur] : 1.f) : 0.f);
        if (rows >> row & 1) {
          uint16_t* const to = p.v + m * 2 * p.ranks + 32 * (tile0 + r) + i;
          to[0] = h.high, to[16] = h.low;
          if (std::is_same<T, f16>::value && i == 0) p.powers[m * (p.ranks / 16) + tile0 + r] = h.power;
        }
      } else if (rows >> row & 1) {
        p.partial[((int64_t)blockIdx.z * p.M + m) * p.ranks + rank] = f;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ columns
// Columns behind p.whole, one by one, of the rows `rows` of `count`; parts(row) and power(row, tile) give a row's v.
template <typename T, class Parts, class Power>
__device__ __forceinline__ void odd_columns(const LoraArgs& p, const uint16_t* b, int64_t m0, int count, uint64_t rows, bool adapter,
                                            Parts parts, Power power) {
  const int odd = p.N - p.whole;
  for (int at = threadIdx.x; at < count * odd; at += 256) {
    const int row = at / odd, col = p.whole + at - row * odd;
    if (!(rows >> row & 1)) continue;
    const int64_t m = m0 + row;
    float s = 0.f;
    if (adapter) {
      const uint16_t* const v = parts(row);
      for (int r0 = 0; r0 < p.R; r0 += 16) {
        float c = 0.f;
#pragma unroll 4
        for (int r = r0; r < min(r0 + 16, p.R); ++r) {
          const float f = from_bits<T>(b[(int64_t)col * p.R + r]);
          c = fmaf(from_bits<T>(v[r0 + r + 16]), f, fmaf(from_bits<T>(v[r0 + r]), f, c));
        }
        s = fmaf(c, power(row, r0 >> 4), s);
      }
    }
    if (p.base) s += from_bits<T>(p.base[m * p.ldb + col]);
    p.out[m * p.ldo + col] = to_bits<T>(s);
  }
}

// Of the last tile's eight ranks 8 (q % 2) .. that a lane holds those that exist, as a mask of their bits.
__device__ __forceinline__ u32x4 last_mask(const LoraArgs& p, int q) {
  const int there = p.R - (p.ranks - 16) - 8 * (q & 1);
  u32x4 mask;
#pragma unroll
  for (int j = 0; j < 4; ++j) mask[j] = (2 * j < there ? 0xFFFFu : 0u) | (2 * j + 1 < there ? 0xFFFF0000u : 0u);
  return mask;
}
template <typename T>
__device__ __forceinline__ u32x4 added(const u32x4& base, const f32x4& d0, const f32x4& d1) {
  u32x4 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x4& d = j < 2 ? d0 : d1;
    o[j] = pack2<T>(d[2 * (j & 1)] + from_bits<T>((uint16_t)(base[j] & 0xFFFF)), d[2 * (j & 1) + 1] + from_bits<T>((uint16_t)(base[j] >> 16)));
  }
  return o;
}

// Few rows: 16 by p.cols columns, B straight from memory.  A wave takes 32 columns at a time as two tiles of 16, tile c of them
// the columns 8 (i / 4) + 4 c + i % 4, so that lane (q, i) ends with the eight columns 8 q .. 8 q + 7 of row i.  RT tiles of 16
// ranks at a time.  Base and B of the first columns are on their way while the shares of v are added up.
template <typename T, int RT>
__global__ void __launch_bounds__(256) lora_columns_few_kernel(LoraArgs p) {
  extern __shared__ u32x4 dynamic_lds[];  // v: [16][ld], of each 16 ranks the high parts, then the low parts
  __shared__ float power[16][16];
  uint16_t* const v = (uint16_t*)dynamic_lds;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15, tiles = p.ranks / 16, ld = 2 * p.ranks + 8;
  const int tile = blockIdx.x / p.slots, slot = blockIdx.x - tile * p.slots;
  const int64_t m0 = (int64_t)tile * 16, m = m0 + i;
  const int id = m < p.M ? lora_id(p, m) : -2;
  const int begin = blockIdx.y * p.cols + wave * 32, end = min((int)(blockIdx.y + 1) * p.cols, p.whole);
  const u32x4 mask = last_mask(p, q);
  uint32_t left = (uint32_t)(__ballot(id >= -1) & 0xFFFF);
  for (int n = 0; left; ++n) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    const uint32_t rows = (uint32_t)(__ballot(id == cur) & 0xFFFF);
    left &= ~rows;
    if (n % p.slots != slot) continue;
    if (cur < 0 && p.out == p.base && p.ldo == p.ldb) continue;  // in place already
    const uint16_t* const b = p.b + max(cur, 0) * p.b_stride;
    const bool mine = id == cur;
    u32x4 bv[2][RT], from;
    auto load_b = [&](int c0, int r0) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r0 + r >= tiles) continue;
        const int at = 16 * (r0 + r) + 8 * (q & 1);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          bv[c][r] = *(const u32x4_any*)(b + (int64_t)min(c0 + 8 * (i >> 2) + 4 * c + (i & 3), p.whole - 1) * p.R + (at < p.R ? at : 0));
      }
    };
    auto load_base = [&](int c0) {
      from = u32x4{0, 0, 0, 0};
      if (p.base && mine && c0 + 8 * q < end) from = *(const u32x4_any*)(p.base + m * p.ldb + c0 + 8 * q);
    };
    if (begin < end) {
      load_base(begin);
      if (cur >= 0) load_b(begin, 0);
    }
    if (cur >= 0) {
      const float scale = p.scales ? p.scales[cur] : 1.f;
      __syncthreads();  // v of the adapter before is read
      // a wave has a row's 16 ranks, lane (q, i) the shares q, q + 4, ... of rank i
      for (int j = wave; j < 16 * tiles; j += 4) {
        const int row = j & 15, r = j >> 4;
        if (!(rows >> row & 1)) continue;
        const float* const at = p.partial + (m0 + row) * p.ranks + 16 * r + i;
        float f = 0.f, part[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) part[s] = q + 4 * s < p.splits ? at[(q + 4 * s) * p.M * p.ranks] : 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s) f += part[s];
        f += __shfl_xor(f, 16);
        f += __shfl_xor(f, 32);
        const Halves h = halves_of<T>(16 * r + i < p.R ? f * scale : 0.f);
        if (q < 2) v[row * ld + 32 * r + 16 * q + i] = q ? h.low : h.high;
        if (lane == 0) power[row][r] = h.power;
      }
      __syncthreads();
    }
    for (int c0 = begin; c0 < end; c0 += 4 * 32) {
      f32x4 sum[2] = {};
      for (int r0 = 0; r0 < tiles && cur >= 0; r0 += RT) {
        if (r0) load_b(c0, r0);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if (r0 + r >= tiles) continue;
          const u32x4 low = *(const u32x4*)(v + i * ld + 32 * (r0 + r) + 8 * q);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (r0 + r == tiles - 1) bv[c][r] &= mask;
            if constexpr (std::is_same<T, f16>::value) {
              const f32x4 one = MfmaOp<T>::run(bv[c][r], low, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int j = 0; j < 4; ++j) sum[c][j] = fmaf(one[j], power[i][r0 + r], sum[c][j]);
            } else {
              sum[c] = MfmaOp<T>::run(bv[c][r], low, sum[c]);
            }
          }
        }
      }
      const u32x4 now = from;
      if (c0 + 4 * 32 < end) {
        load_base(c0 + 4 * 32);
        if (cur >= 0) load_b(c0 + 4 * 32, 0);
      }
      if (mine && c0 + 8 * q < end) *(u32x4_any*)(p.out + m * p.ldo + c0 + 8 * q) = added<T>(now, sum[0], sum[1]);
    }
    if (blockIdx.y + 1 == gridDim.y)
      odd_columns<T>(p, b, m0, 16, rows, cur >= 0, [&](int row) { return v + row * ld; }, [&](int row, int r) { return power[row][r]; });
  }
}

// Many rows: 128 by p.cols columns, 64 of them at a time: their B goes through LDS once for the four waves, which have 32 rows
// each, and the next 64 columns' is on its way meanwhile.  Tile c of the four holds the columns 16 (i / 4) + 4 c + i % 4, so
// that lane (q, i) ends with the sixteen columns 16 q .. 16 q + 15 of row i.  Neighbouring lanes swap halves of theirs, so that each
// load and store of base and out covers whole lines of 128 bytes.
template <typename T, int RT>
__global__ void __launch_bounds__(256) lora_columns_kernel(LoraArgs p) {
  constexpr int MT = 2, ROWS = 64 * MT, LD = 16 * RT + 8, PIECES = 64 * 2 * RT, EACH = (PIECES + 255) / 256;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][64][LD];  // [column][rank]
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15, tiles = p.ranks / 16, chunks = (tiles + RT - 1) / RT;
  // a row tile's blocks go to all XCDs, so that tiles of several adapters, which take longer, do not meet on one
  const int64_t m0 = (int64_t)((blockIdx.x + blockIdx.y) % gridDim.x) * ROWS;
  int id[2];
  uint64_t left[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t m = m0 + 64 * h + lane;
    id[h] = m < p.M ? lora_id(p, m) : -2;
    left[h] = __ballot(id[h] >= -1);
  }
  const int begin = blockIdx.y * p.cols, end = min((int)(blockIdx.y + 1) * p.cols, p.whole), odd = i & 1;
  while (left[0] | left[1]) {
    const int cur = left[0] ? __builtin_amdgcn_readlane(id[0], __builtin_ctzll(left[0])) : __builtin_amdgcn_readlane(id[1], __builtin_ctzll(left[1]));
    const uint64_t rows[2] = {__ballot(id[0] == cur), __ballot(id[1] == cur)};
    left[0] &= ~rows[0], left[1] &= ~rows[1];
    if (cur < 0 && p.out == p.base && p.ldo == p.ldb) continue;  // in place already
    const uint16_t* const b = p.b + max(cur, 0) * p.b_stride;
    const uint32_t mine = (uint32_t)(rows[wave >> 1] >> (32 * (wave & 1)));  // the wave's 32 rows
    const int64_t mw = m0 + 32 * wave;
    u32x4 stage[EACH], bs[MT][2];
    auto load_b = [&](int c0, int chunk) {
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int piece = t + 256 * e, col = piece / (2 * RT), at = 16 * RT * chunk + 8 * (piece % (2 * RT));
        if (PIECES % 256 && piece >= PIECES) continue;
        stage[e] = u32x4{0, 0, 0, 0};
        if (at < p.R) stage[e] = *(const u32x4_any*)(b + (int64_t)min(c0 + col, p.whole - 1) * p.R + at);
        if (at < p.R && at + 8 > p.R) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            stage[e][j] &= (at + 2 * j < p.R ? 0xFFFFu : 0u) | (at + 2 * j + 1 < p.R ? 0xFFFF0000u : 0u);
        }
      }
    };
    // the rows and columns of a lane's loads and stores: both rows of a pair, the even or the odd half of their sixteen columns
    auto row_of = [&](int mt, int k) { return 16 * mt + (i & ~1) + k; };
    auto load_base = [&](int c0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          bs[mt][k] = u32x4{0, 0, 0, 0};
          if (p.base && (mine >> row_of(mt, k) & 1) && c0 + 16 * q + 8 * odd < end)
            bs[mt][k] = *(const u32x4_any*)(p.base + (mw + row_of(mt, k)) * p.ldb + c0 + 16 * q + 8 * odd);
        }
    };
    u32x4 low[MT][RT];
    float power[MT][RT];
    auto load_low = [&](int chunk) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int64_t m = min(mw + 16 * mt + i, p.M - 1);
          if (chunk * RT + r >= tiles) continue;
          low[mt][r] = *(const u32x4*)(p.v + m * 2 * p.ranks + 32 * (chunk * RT + r) + 8 * q);
          if constexpr (std::is_same<T, f16>::value) power[mt][r] = p.powers[m * tiles + chunk * RT + r];
        }
    };
    if (cur >= 0) {
      load_b(begin, 0);
      load_low(0);
    }
    load_base(begin);
    __syncthreads();  // the adapter before is done with the LDS
    int buf = 0;
    for (int c0 = begin; c0 < end; c0 += 64) {
      f32x4 sum[MT][4] = {};
      if (cur >= 0) {
        for (int chunk = 0; chunk < chunks; ++chunk, buf ^= 1) {
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            const int piece = t + 256 * e;
            if (PIECES % 256 && piece >= PIECES) continue;
            *(u32x4*)&lds[buf][piece / (2 * RT)][8 * (piece % (2 * RT))] = stage[e];
          }
          __syncthreads();
          if (chunk + 1 < chunks) load_b(c0, chunk + 1);
          else if (c0 + 64 < end) load_b(c0 + 64, 0);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            if (chunk * RT + r >= tiles || !mine) continue;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const u32x4 bv = *(const u32x4*)&lds[buf][16 * (i >> 2) + 4 * c + (i & 3)][16 * r + 8 * (q & 1)];
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                if constexpr (std::is_same<T, f16>::value) {
                  const f32x4 one = MfmaOp<T>::run(bv, low[mt][r], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                  for (int j = 0; j < 4; ++j) sum[mt][c][j] = fmaf(one[j], power[mt][r], sum[mt][c][j]);
                } else {
                  sum[mt][c] = MfmaOp<T>::run(bv, low[mt][r], sum[mt][c]);
                }
              }
            }
          }
          if (chunks > 1) load_low(chunk + 1 < chunks ? chunk + 1 : 0);
        }
      }
      u32x4 now[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) now[mt][0] = bs[mt][0], now[mt][1] = bs[mt][1];
      if (c0 + 64 < end) load_base(c0 + 64);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const u32x4 got = from_neighbour(odd ? now[mt][0] : now[mt][1]);
        const u32x4 o0 = added<T>(odd ? got : now[mt][0], sum[mt][0], sum[mt][1]);
        const u32x4 o1 = added<T>(odd ? now[mt][1] : got, sum[mt][2], sum[mt][3]);
        const u32x4 other = from_neighbour(odd ? o0 : o1);
        const u32x4 o[2] = {odd ? other : o0, odd ? o1 : other};
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if ((mine >> row_of(mt, k) & 1) && c0 + 16 * q + 8 * odd < end)
            *(u32x4_any*)(p.out + (mw + row_of(mt, k)) * p.ldo + c0 + 16 * q + 8 * odd) = o[k];
      }
    }
    if (blockIdx.y + 1 == gridDim.y) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        odd_columns<T>(p, b, m0 + 64 * h, 64, rows[h], cur >= 0, [&](int row) { return p.v + (m0 + 64 * h + row) * 2 * p.ranks; },
                       [&](int row, int r) { return std::is_same<T, f16>::value ? p.powers[(m0 + 64 * h + row) * tiles + r] : 1.f; });
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

static int64_t lora_ranks(int64_t R) { return cdiv(R, 16) * 16; }

// Columns that go by eight: whole pieces of out, and B's pieces of eight ranks, of which a row's last may reach into the next
// row, end with B.
static int64_t lora_whole(int64_t N, int64_t R) {
  const int64_t past = cdiv(R, 8) * 8 - R;
  return std::max<int64_t>(0, N - cdiv(past, R)) / 8 * 8;
}

struct LoraPlan {
  bool many;
  int slots, rt, splits, per;  // rt: tiles of 16 ranks of a block of the first launch
};
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t R) {
  LoraPlan l{};
  const int64_t tiles = cdiv(M, 16), ranks = lora_ranks(R) / 16, units = cdiv(K, kUnit);
  l.many = M > 512;
  // a batch of single tokens has many adapters in a tile, prompts one or two
  l.slots = M <= 128 ? (int)std::min<int64_t>(16, M) : 1;
  l.rt = ranks >= 3 ? 4 : (int)ranks;
  l.splits = 1, l.per = (int)units;
  if (!l.many) {
    const int64_t want = std::max<int64_t>(1, 256 / (tiles * l.slots * cdiv(ranks, l.rt)));
    l.per = (int)std::max<int64_t>(4, cdiv(units, std::min<int64_t>(want, 16)));
    l.splits = (int)cdiv(units, l.per);
  }
  return l;
}
size_t lora_workspace_bytes(int64_t M, int64_t K, int64_t R) {
  const LoraPlan l = lora_plan(M, K, R);
  const size_t values = (size_t)M * (size_t)lora_ranks(R);
  return l.many ? values * 4 + values / 16 * 4 : (size_t)l.splits * values * 4;
}

template <typename T>
static int lora_typed(LoraArgs p, const LoraPlan& l, hipStream_t st) {
  using std::integral_constant;
  const int tiles = p.ranks / 16;
  auto by_rank = [&](auto f) {
    if (tiles == 1) f(integral_constant<int, 1>{});
    else if (tiles == 2) f(integral_constant<int, 2>{});
    else f(integral_constant<int, 4>{});
  };
  const int64_t row_tiles = cdiv(p.M, 16);
  by_rank([&](auto n) {
    constexpr int RT = decltype(n)::value, D = RT == 4 ? 1 : RT == 2 ? 2 : 4;
    const dim3 grid((unsigned)(row_tiles * p.slots), (unsigned)cdiv(tiles, RT), (unsigned)l.splits);
    if (l.many) lora_ranks_kernel<T, RT, 8, D == 4 ? 2 : D, true><<<grid, 512, 0, st>>>(p);
    else lora_ranks_kernel<T, RT, 4, D, false><<<grid, 256, 0, st>>>(p);
  });
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  const int64_t x = l.many ? cdiv(p.M, 128) : row_tiles * p.slots, step = l.many ? 64 : 128;
  const int64_t steps = std::max<int64_t>(1, cdiv(p.whole, step)), want = std::max<int64_t>(1, 2048 / x);
  p.cols = (int)(cdiv(steps, std::min(want, steps)) * step);
  const dim3 grid((unsigned)x, (unsigned)std::max<int64_t>(1, cdiv(p.whole, p.cols)));
  by_rank([&](auto n) {
    constexpr int RT = decltype(n)::value;
    if (l.many) lora_columns_kernel<T, RT><<<grid, 256, 0, st>>>(p);
    else lora_columns_few_kernel<T, RT><<<grid, 256, (size_t)16 * (2 * p.ranks + 8) * 2, st>>>(p);
  });
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

int launch_lora(const LoraCall& c, hipStream_t st) {
  LoraArgs p{};
  p.base = (const uint16_t*)c.base, p.x = (const uint16_t*)c.x, p.a = (const uint16_t*)c.a, p.b = (const uint16_t*)c.b;
  p.ids = c.ids, p.scales = c.scales, p.out = (uint16_t*)c.out;
  p.ldb = c.ldb, p.ldx = c.ldx, p.ldo = c.ldo, p.a_stride = c.a_stride, p.b_stride = c.b_stride;
  p.M = c.M, p.N = (int)c.N, p.K = (int)c.K, p.R = (int)c.R, p.L = c.L, p.id64 = c.id64;
  p.ranks = (int)lora_ranks(c.R), p.whole = (int)lora_whole(c.N, c.R);
  const LoraPlan l = lora_plan(c.M, c.K, c.R);
  p.slots = l.slots, p.splits = l.splits, p.per = l.per;
  p.partial = (float*)c.workspace;
  p.v = (uint16_t*)c.workspace, p.powers = (float*)(p.v + (size_t)c.M * 2 * p.ranks);
  return c.dtype == AWQ_DTYPE_F16 ? lora_typed<f16>(p, l, st) : lora_typed<bf16>(p, l, st);
}

}  // namespace awq_host
