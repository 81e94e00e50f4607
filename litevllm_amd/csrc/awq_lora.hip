// Low-rank adapters of many requests, added to what a shared projection gave:
//
//   l = ids[m];  v[m] = s_l x[m] A_l^T  (rank values);  out[m] = base[m] + v[m] B_l^T;  out[m] = base[m] without an adapter
//
// Two launches: the ranks (x and A once, sums in fp32) and the columns (base and B once); one for few rows whose adapters are
// small, where the blocks of columns compute their v themselves (lora_plan).  Rows go in tiles of 16 that the matrix cores take; a
// tile looks up which adapters its rows have and is worked on once for each: once where the rows of a request lie together,
// as in prompts, up to 16 times in a batch of single tokens, whose rows are put together by adapter from 65 to 512 rows
// (group_of).  Its blocks (`slots`) share these and, where it has fewer adapters than blocks, an adapter's columns or K.
// The matrix cores do not mix rows, so the other rows of a tile only cost idle lanes.
//
// v enters the second product as two 16-bit numbers, v = high + low, and the output is rounded once.  Both halves meet the same B:
// ranks go in tiles of W = 32, an instruction for the high parts and one for the low parts, or of 16 (rank 16 and less), high and
// low parts in one instruction of depth 32.  fp16 takes v / 2^e instead, with an e of its own for a row's tile that puts the
// largest value at 2^13 .. 2^14: v may pass fp16's range.
// high + low is off from v by at most 2^-17 of v in bf16 (two times eight bits and low's sign; for v above 2^-109, where low is a
// normal number).  In fp16 that is 2^-22 of v down to 2^-16 of the tile's largest value; below, low ends with fp16's smallest
// step, 2^-24 in units of 2^e, and the error stays at 2^-38 of that largest value: a rank 2^26 below it still has 12 bits.
#include <algorithm>

#include "awq_launch.h"

namespace awq {

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any address of a 16-bit element

// A block's group of few rows as the first launch found it, for the second (see Group).
struct GroupRecord {
  int adapter, rows, part, parts, row[16];
};
struct LoraArgs {
  const uint16_t *base, *x, *a, *b;
  const void* ids;
  const float* scales;
  uint16_t* out;
  float* partial;  // few rows: [shares][M][ranks], s_l not in it yet
  uint16_t* v;     // many rows: [M][2 ranks], of each W ranks the high parts, then the low parts
  float* powers;   // and [M][ranks / W]: 2^e (fp16)
  GroupRecord* records;  // NULL where there is no first launch that finds them
  int64_t ldb, ldx, ldo, a_stride, b_stride;
  int64_t M;
  int N, K, R, L, id64;
  int ranks;  // R in whole tiles of W
  int tiles;  // of 16 rows
  int slots;  // blocks that share a tile's adapters, for few rows as many as it may have: block tile + tiles * slot, so that
              // each slot's are on all XCDs
  int splits, shares;  // few rows: shares of K, and how many there may be with sub-shares
  int cols;   // many rows: columns of a block
  int whole;  // columns that go by eight, see lora_whole
  int ranges;   // many rows: blocks over the columns
};

__device__ __forceinline__ int lora_id(const LoraArgs& p, int64_t m) {
  const int64_t l = p.id64 ? ((const int64_t*)p.ids)[m] : (int64_t)((const int32_t*)p.ids)[m];
  return l >= 0 && l < p.L ? (int)l : -1;
}
// Few rows go in groups of up to 16 of the same adapter, the rows without one as if they had the same.  A block has the group of its
// number or, where there are fewer groups than blocks, shares one with others as number `part` of `parts`.
constexpr int kFewRows = 512, kTogether = 64, kMostCounted = 1024;
struct Group {
  int adapter;     // -1: none
  uint32_t rows;   // which of the 16 exist
  int part, parts;
  int row;         // that of lanes i, i + 16, ..., or one that exists
};
struct GroupLds {
  int seen[kMostCounted + 1];  // an adapter's rows so far
  int key[kFewRows], rank[kFewRows];  // a row's adapter (-1), and its number among the adapter's rows
  GroupRecord found;
};
__device__ __forceinline__ Group recorded(const GroupRecord& r) {
  return {__builtin_amdgcn_readfirstlane(r.adapter), (uint32_t)__builtin_amdgcn_readfirstlane(r.rows),
          __builtin_amdgcn_readfirstlane(r.part), __builtin_amdgcn_readfirstlane(r.parts), r.row[threadIdx.x & 15]};
}
// By one wave.
__device__ __forceinline__ void record(const Group& g, GroupRecord& r) {
  if (threadIdx.x < 16) r.row[threadIdx.x] = g.row;
  if (threadIdx.x == 0) r.adapter = g.adapter, r.rows = (int)g.rows, r.part = g.part, r.parts = g.parts;
}
// Groups of 16 neighbouring rows and of one adapter; id: that of lane i's, -2 for no row.
__device__ __forceinline__ Group group_of_neighbours(const LoraArgs& p, int row0, int id, int slot) {
  const int i = threadIdx.x & 15;
  const uint32_t all = (uint32_t)(__ballot(id >= -1) & 0xFFFF);
  int count = 0;
  for (uint32_t left = all; left; ++count) left &= ~(uint32_t)__ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctz(left)));
  Group g{};
  int mine = slot % count;
  g.part = slot / count, g.parts = (p.slots - 1 - mine) / count + 1;
  for (uint32_t left = all; mine >= 0; --mine) {
    g.adapter = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    g.rows = (uint32_t)__ballot(id == g.adapter) & left;
    left &= ~g.rows;
  }
  g.row = row0 + (g.rows >> i & 1 ? i : __builtin_ctz(g.rows));
  return g;
}
// Groups of the adapter's rows wherever they are, in their order, by one wave and 64 rows at a time: lanes with the same adapter find
// each other by its bits.
__device__ __forceinline__ Group group_of_all(const LoraArgs& p, GroupLds& lds, int number) {
  const int t = threadIdx.x, rows = (int)p.M;
  for (int e = t; e <= p.L; e += 64) lds.seen[e] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  int groups = 0;
#pragma unroll 1
  for (int m = t; m - t < rows; m += 64) {
    const bool has = m < rows;
    const int id = has ? lds.key[m] : -1, e = id < 0 ? p.L : id;
    uint64_t same = __ballot(has);
    for (int bit = 1; bit <= p.L; bit <<= 1) {
      const uint64_t set = __ballot(e & bit);
      same &= e & bit ? set : ~set;
    }
    const int ahead = __popcll(same & ((1ull << t) - 1)), before = lds.seen[e], rank = before + ahead;
    __builtin_amdgcn_wave_barrier();
    if (has) lds.rank[m] = rank;
    if (has && ahead == 0) lds.seen[e] = before + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    groups += __popcll(__ballot(has && (rank & 15) == 0));
  }
  const int mine = number % groups;
  int left = mine, adapter = 0, rank0 = -1, count = 0;
#pragma unroll 1
  for (int m = t; m - t < rows; m += 64) {
    const bool has = m < rows;
    const int id = has ? lds.key[m] : -2, rank = has ? lds.rank[m] : 0;
    if (rank0 < 0) {
      const uint64_t first = __ballot(has && (rank & 15) == 0);
      const int n = __popcll(first);
      if (left >= n) {
        left -= n;
        continue;
      }
      const int lane = __builtin_ctzll(__ballot((first >> t & 1) && __popcll(first & ((1ull << t) - 1)) == left));
      adapter = __builtin_amdgcn_readlane(id, lane), rank0 = __builtin_amdgcn_readlane(rank, lane);
      if (t < 16) lds.found.row[t] = m - t + lane;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    const bool in = id == adapter && rank >= rank0 && rank < rank0 + 16;
    if (in) lds.found.row[rank - rank0] = m;
    count += __popcll(__ballot(in));
  }
  Group g{};
  g.adapter = adapter, g.rows = (1u << count) - 1, g.part = number / groups, g.parts = (p.tiles * p.slots - 1 - mine) / groups + 1;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  g.row = lds.found.row[t & 15];
  return g;
}
// Neighbours where most have the same adapter, as in prompts, or the rows are few: the search costs a prompt about 1 us (128 rows, rank
// 16 7.4, 6.9 without it, rank 64 12.7 and 12.3, 200 rows 9.1 and 8.2) and saves single tokens the passes over the same adapter in other
// tiles (64 adapters: 128 rows, rank 16 11.0 and 12.3, rank 64 21.9 and 28.1, 256 rows, rank 64 25.9 and 51, 500 rows, N = 24576, rank
// 16 34 and 84; 64 rows, rank 32 13.1 and 13.4, their prompts 9.6 and 9.2).
__device__ __forceinline__ Group group_of(const LoraArgs& p, GroupLds& lds, int number) {
  const int t = threadIdx.x, i = t & 15, row0 = number % p.tiles * 16, slot = number / p.tiles, m = row0 + i, rows = (int)p.M;
  if (rows <= kTogether || p.L > kMostCounted) {
    const Group g = group_of_neighbours(p, row0, m < rows ? lora_id(p, m) : -2, slot);
    record(g, lds.found);
    return g;
  }
  for (int at = t; at < rows; at += (int)blockDim.x) lds.key[at] = lora_id(p, at);
  __syncthreads();
  if (t < 64) {
    int runs = 1;
    for (int at = t + 1; at - t < rows; at += 64) runs += __popcll(__ballot(at < rows && lds.key[at] != lds.key[at - 1]));
    record(runs > 2 * p.tiles ? group_of_all(p, lds, number) : group_of_neighbours(p, row0, m < rows ? lds.key[m] : -2, slot), lds.found);
  }
  __syncthreads();
  return recorded(lds.found);
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

// v of a rank as its two parts, in units of `power`.
struct Parts {
  uint16_t high, low;
  float power;
};
template <typename T>
__device__ __forceinline__ Parts parts_of(float f, int e) {
  if constexpr (std::is_same<T, f16>::value) f = ldexpf(f, -e);
  uint16_t high = to_bits<T>(f);
  if (std::is_same<T, bf16>::value && fabsf(f) < __builtin_inff() && (high & 0x7FFF) == 0x7F80) --high;  // the rest fits into low
  return {high, fabsf(f) < __builtin_inff() ? to_bits<T>(f - from_bits<T>(high)) : (uint16_t)0,  // no Inf - Inf
          std::is_same<T, f16>::value ? ldexpf(1.f, e) : 1.f};
}
// e of a row's tile from its largest value (0, Inf and NaN included).
__device__ __forceinline__ int tile_exponent(float top) { return (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 13; }
// The same for W neighbouring lanes that hold a row's tile.
template <typename T, int W>
__device__ __forceinline__ Parts tile_parts(float f) {
  if constexpr (!std::is_same<T, f16>::value) return parts_of<T>(f, 0);
  float top = row_max16(fabsf(f));
  if constexpr (W == 32) top = fmaxf(top, __shfl_xor(top, 16));
  return parts_of<T>(f, tile_exponent(top));
}

// ------------------------------------------------------------------ ranks
constexpr int kUnit = 64;  // values of K that a wave takes at once: whole lines of both operands

template <int RT, int WAVES>
union RankLds {
  uint16_t stage[WAVES][(1 + RT) * 16][kUnit + 8];  // rows 16 bytes apart from whole banks
  f32x4 part[WAVES][RT][64];
};
// RT tiles of 16 ranks, from tile0 on, of adapter `cur` by the rows row(0 .. 15) and a share of K, whose units the waves take in
// turn; the waves' sums come to lie in LDS.  A wave's next unit is on its way in registers (more of them made every size slower:
// one row, K = N = 4096, rank 16 6.6 us with two, 7.3 with four, 6.3 as it is).  Loads cover whole lines, eight lanes each; a
// wave passes them through LDS of its own into the matrix cores' order, where lane (q, i) holds values 8 q .. 8 q + 7 and 32 + 8 q
// .. of rank i and of row i.  (Straight from memory in that order a load's neighbouring lanes are in different lines: 4096 rows,
// K = 4096, rank 64 42 us instead of 12.)
template <typename T, int RT, int WAVES, class Row>
__device__ __forceinline__ void tile_ranks(const LoraArgs& p, RankLds<RT, WAVES>& lds, Row row, int cur, int tile0, int begin, int units) {
  constexpr int TILES = 1 + RT;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15, r8 = lane >> 3, c8 = 8 * (lane & 7);
  // two rows of each tile a lane
  const uint16_t* from[TILES][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    from[0][h] = p.x + row(r8 + 8 * h) * p.ldx + c8;
#pragma unroll
    for (int r = 0; r < RT; ++r) from[1 + r][h] = p.a + cur * p.a_stride + (int64_t)min(16 * (tile0 + r) + r8 + 8 * h, p.R - 1) * p.K + c8;
  }
  u32x4 piece[TILES][2];
  auto load = [&](int u) {
    if (u >= units) return;
    // the last unit's pieces end with K: what lies past it, or belongs to the piece before, becomes 0 in both operands
    const int k = u * kUnit + c8, at = min(k, p.K - 8) - c8, twice = k - c8 - at;
#pragma unroll
    for (int j = 0; j < TILES; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) piece[j][h] = *(const u32x4_any*)(from[j][h] + at);
    if (u * kUnit + kUnit <= p.K) return;
    u32x4 mask;
#pragma unroll
    for (int j = 0; j < 4; ++j) mask[j] = (2 * j >= twice ? 0xFFFFu : 0u) | (2 * j + 1 >= twice ? 0xFFFF0000u : 0u);
#pragma unroll
    for (int j = 0; j < TILES; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) piece[j][h] &= mask;
  };
  f32x4 acc[RT] = {};
  load(begin + wave);
  for (int u = begin + wave; u < units; u += WAVES) {
#pragma unroll
    for (int j = 0; j < TILES; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) *(u32x4*)&lds.stage[wave][16 * j + r8 + 8 * h][c8] = piece[j][h];
    load(u + WAVES);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < kUnit; k += 32) {
      const u32x4 x = *(const u32x4*)&lds.stage[wave][i][k + 8 * q];
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[r] = MfmaOp<T>::run(*(const u32x4*)&lds.stage[wave][16 * (1 + r) + i][k + 8 * q], x, acc[r]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();  // all waves are done with their stages
  // ranks 4 q .. 4 q + 3 of row i
#pragma unroll
  for (int r = 0; r < RT; ++r) lds.part[wave][r][lane] = acc[r];
  __syncthreads();
}
// f(row, rank of the block's, sum) of what lies there, a row's W ranks by W neighbouring lanes.
template <int RT, int WAVES, int W, class F>
__device__ __forceinline__ void for_ranks(const RankLds<RT, WAVES>& lds, F f) {
  for (int at = threadIdx.x; at < RT * 256; at += 64 * WAVES) {
    const int row = at / W % 16, rank = at / (16 * W) * W + at % W, j = rank & 15;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += ((const float*)&lds.part[w][rank >> 4][16 * (j >> 2) + row])[j & 3];
    f(row, rank, s);
  }
}

// A rank's parts of v, by W neighbouring lanes; rows that are not `mine` take part only.
template <typename T, int W>
__device__ __forceinline__ void put_rank(const LoraArgs& p, int64_t m, int rank, float f, float scale, bool mine) {
  const Parts h = tile_parts<T, W>(rank < p.R ? f * scale : 0.f);
  if (!mine) return;
  uint16_t* const to = p.v + m * 2 * p.ranks + 2 * (rank / W) * W + rank % W;
  to[0] = h.high, to[W] = h.low;
  if (std::is_same<T, f16>::value && rank % W == 0) p.powers[m * (p.ranks / W) + rank / W] = h.power;
}

// Few rows: a block has a group of rows and a share of K; those that share the group cut the share further, into sub-shares
// (lora_shares).  29 rows, K = 12288, rank 12: 5.2 us, latency.  What it found out about a block's group is left for the
// second launch (the same rows, N = 5001: 12.0 -> 10.5 us for both).
__device__ __forceinline__ int lora_shares(const LoraArgs& p, int parts) { return min(parts, p.shares / p.splits); }
template <typename T, int RT, int W>
__global__ void __launch_bounds__(256) lora_ranks_few_kernel(LoraArgs p) {
  __shared__ __attribute__((aligned(16))) RankLds<RT, 4> lds;
  __shared__ GroupLds groups;
  const int tile0 = blockIdx.y * RT;
  const Group g = group_of(p, groups, blockIdx.x);
  if (blockIdx.y == 0 && blockIdx.z == 0) record(g, p.records[blockIdx.x]);
  const int shares = lora_shares(p, g.parts), share = blockIdx.z * shares + g.part;
  if (g.adapter < 0 || g.part >= shares) return;
  const int units = (p.K + kUnit - 1) / kUnit, per = (units + p.splits * shares - 1) / (p.splits * shares);
  tile_ranks<T, RT, 4>(p, lds, [&](int r) { return (int64_t)__shfl(g.row, r); }, g.adapter, tile0, share * per, min((share + 1) * per, units));
  for_ranks<RT, 4, W>(lds, [&](int row, int rank, float f) {
    rank += 16 * tile0;
    const int64_t m = __shfl(g.row, row);
    if (rank < p.ranks && (g.rows >> row & 1)) p.partial[(share * p.M + m) * p.ranks + rank] = f;
  });
}

// Many rows: a block has every slots-th adapter of the tile and all of K.  Of four tiles of ranks it is bound by the lines that
// a CU's four waves load (0.7 MB of x and A for 16 rows, K = 4096) and pass through LDS, more waves made it slower (4096 rows,
// rank 64, N = 4096: 45 us, with eight 49; rank 16, 2000 rows, N = 8192 28 and 24).
constexpr int many_waves(int rt) { return rt == 4 ? 4 : 8; }
template <typename T, int RT, int W>
__global__ void __launch_bounds__(64 * many_waves(RT)) lora_ranks_kernel(LoraArgs p) {
  constexpr int WAVES = many_waves(RT);
  __shared__ __attribute__((aligned(16))) RankLds<RT, WAVES> lds;
  const int i = threadIdx.x & 15, slot = blockIdx.x / p.tiles, tile0 = blockIdx.y * RT;
  const int64_t m0 = (int64_t)(blockIdx.x % p.tiles) * 16;
  const int id = m0 + i < p.M ? lora_id(p, m0 + i) : -1;
  uint32_t left = (uint32_t)(__ballot(id >= 0) & 0xFFFF);
  for (int n = 0; left; ++n) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    const uint32_t rows = (uint32_t)(__ballot(id == cur) & 0xFFFF);
    left &= ~rows;
    if (n % p.slots != slot) continue;
    // for rows of other adapters a row that is read anyway
    tile_ranks<T, RT, WAVES>(p, lds, [&](int r) { return m0 + (rows >> r & 1 ? r : __builtin_ctz(rows)); }, cur, tile0, 0,
                             (p.K + kUnit - 1) / kUnit);
    for_ranks<RT, WAVES, W>(lds, [&](int row, int rank, float f) {
      rank += 16 * tile0;
      if (rank < p.ranks) put_rank<T, W>(p, m0 + row, rank, f, p.scales ? p.scales[cur] : 1.f, rows >> row & 1);
    });
    __syncthreads();
  }
}

// Rows of fewer than eight values, one share: a thread has a row and a rank.
template <typename T, int W, bool FINAL>
__global__ void __launch_bounds__(256) lora_ranks_short_kernel(LoraArgs p) {
  const int64_t m = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
  const int rank = blockIdx.y * W + threadIdx.x % W;
  const int id = m < p.M ? lora_id(p, m) : -1;
  float f = 0.f;
  if (id >= 0 && rank < p.R)
    for (int k = 0; k < p.K; ++k)
      f = fmaf(from_bits<T>(p.x[m * p.ldx + k]), from_bits<T>(p.a[id * p.a_stride + (int64_t)rank * p.K + k]), f);
  if constexpr (FINAL) put_rank<T, W>(p, m, rank, f, p.scales ? p.scales[max(id, 0)] : 1.f, id >= 0);
  else if (id >= 0) p.partial[m * p.ranks + rank] = f;
}

// ------------------------------------------------------------------ columns
// Columns behind p.whole, one by one, of the rows at(0), ... of `rows`, which has `count` bits; parts(row) and power(row, tile)
// give a row's v.
template <typename T, int W, class At, class Parts, class Power>
__device__ __forceinline__ void odd_columns(const LoraArgs& p, const uint16_t* b, At at, int count, uint64_t rows, bool adapter, Parts parts,
                                            Power power) {
  const int odd = p.N - p.whole;
  for (int n = threadIdx.x; n < count * odd; n += blockDim.x) {
    const int row = n / odd, col = p.whole + n - row * odd;
    if (!(rows >> row & 1)) continue;
    const int64_t m = at(row);
    float s = 0.f;
    if (adapter) {
      const uint16_t* const v = parts(row);
      for (int r0 = 0; r0 < p.R; r0 += W) {
        float c = 0.f;
#pragma unroll 4
        for (int r = r0; r < min(r0 + W, p.R); ++r) {
          const float f = from_bits<T>(b[(int64_t)col * p.R + r]);
          c = fmaf(from_bits<T>(v[r0 + r + W]), f, fmaf(from_bits<T>(v[r0 + r]), f, c));
        }
        s = fmaf(c, power(row, r0 / W), s);
      }
    }
    if (p.base) s += from_bits<T>(p.base[m * p.ldb + col]);
    p.out[m * p.ldo + col] = to_bits<T>(s);
  }
}

// A lane's eight ranks of a tile begin with this one, of either operand.
template <int W>
__device__ __forceinline__ int first_rank(int q) { return 8 * (W == 32 ? q : q & 1); }
// What the two parts of v give with eight ranks of B, on top of c.
template <typename T, int W>
__device__ __forceinline__ f32x4 both_parts(const u32x4& b, const u32x4 (&v)[W / 16], f32x4 c) {
#pragma unroll
  for (int h = 0; h < W / 16; ++h) c = MfmaOp<T>::run(b, v[h], c);
  return c;
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

// Few rows: a group by p.cols columns, B straight from memory.  A wave takes 32 columns at a time as two tiles of 16, tile c of them
// the columns 8 (i / 4) + 4 c + i % 4, so that lane (q, i) ends with the eight columns 8 q .. 8 q + 7 of row i.  RT tiles of W
// ranks at a time.  Base and B of the first columns are on their way while v is made ready: the shares of the first launch are
// added up or, OWN > 0, all OWN tiles of 16 ranks computed by the block itself, for all of its columns.  Bound by the chain of ids, A,
// sum and products: one row, K = N = 4096, rank 16 6.1 us; 64 rows of 64 adapters, N = 6144, rank 32 13 us, 28.7 MB.
constexpr int few_waves(bool own) { return own ? 8 : 4; }
template <typename T, int RT, int W, int OWN>
__global__ void __launch_bounds__(64 * few_waves(OWN > 0), OWN ? 1 : 2) lora_columns_few_kernel(LoraArgs p) {
  constexpr int SUB = W / 16, WAVES = few_waves(OWN > 0), STEP = WAVES * 32;
  __shared__ __attribute__((aligned(16))) RankLds<OWN ? OWN : 1, OWN ? WAVES : 1> own;
  extern __shared__ u32x4 dynamic_lds[];  // v: [16][ld], of each W ranks the high parts, then the low parts
  __shared__ float power[16][16];
  __shared__ GroupLds groups;
  uint16_t* const v = (uint16_t*)dynamic_lds;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15, tiles = p.ranks / W, ld = 2 * p.ranks + 8;
  const bool found = OWN == 0 && p.records;
  const Group g = found ? recorded(p.records[blockIdx.x]) : group_of(p, groups, blockIdx.x);
  if (found) record(g, groups.found);
  if (g.adapter < 0 && p.out == p.base && p.ldo == p.ldb) return;  // in place already
  const int cur = g.adapter, part = blockIdx.y * g.parts + g.part, parts = gridDim.y * g.parts;
  const int steps = (p.whole + STEP - 1) / STEP, cols = (steps + parts - 1) / parts * STEP;
  const int begin = min(part * cols, p.whole) + wave * 32, end = min((part + 1) * cols, p.whole);
  if (part * cols >= p.whole && part + 1 < parts) return;  // nothing left
  const int64_t m = g.row;
  const bool mine = g.rows >> i & 1;
  const uint16_t* const b = p.b + max(cur, 0) * p.b_stride;
  // of the last tile's eight ranks of this lane those that exist, as a mask of their bits
  const int there = p.R - (p.ranks - W) - first_rank<W>(q);
  u32x4 mask;
#pragma unroll
  for (int j = 0; j < 4; ++j) mask[j] = (2 * j < there ? 0xFFFFu : 0u) | (2 * j + 1 < there ? 0xFFFF0000u : 0u);
  u32x4 bv[2][RT], from;
  auto load_b = [&](int c0, int r0) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (r0 + r >= tiles) continue;
      const int at = W * (r0 + r) + first_rank<W>(q);
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
    const int shares = p.splits * lora_shares(p, g.parts);
    if constexpr (OWN > 0) {
      tile_ranks<T, OWN, WAVES>(p, own, [&](int r) { return (int64_t)__shfl(g.row, r); }, cur, 0, 0, (p.K + kUnit - 1) / kUnit);
      for_ranks<OWN, WAVES, W>(own, [&](int row, int rank, float f) {
        if (rank >= p.ranks) return;
        const Parts two = tile_parts<T, W>(rank < p.R ? f * scale : 0.f);
        uint16_t* const to = v + row * ld + 2 * (rank / W) * W + rank % W;
        to[0] = two.high, to[W] = two.low;
        if (rank % W == 0) power[row][rank / W] = two.power;
      });
    }
    // a wave has a row's tile, lane (q, i) the shares q, q + 4, ... of ranks i and 16 + i
    for (int j = wave; j < 16 * tiles && !OWN; j += 4) {
      const int row = j & 15, r = j >> 4;
      if (!(g.rows >> row & 1)) continue;
      const float* const at = p.partial + (int64_t)__builtin_amdgcn_readlane(g.row, row) * p.ranks + W * r + i;
      float part[SUB][4], f[SUB];
#pragma unroll
      for (int h = 0; h < SUB; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s) part[h][s] = q + 4 * s < shares ? at[(q + 4 * s) * p.M * p.ranks + 16 * h] : 0.f;
      int e = 0;
      float top = 0.f;
#pragma unroll
      for (int h = 0; h < SUB; ++h) {
        f[h] = (part[h][0] + part[h][1]) + (part[h][2] + part[h][3]);
        f[h] += __shfl_xor(f[h], 16);
        f[h] += __shfl_xor(f[h], 32);
        f[h] = W * r + 16 * h + i < p.R ? f[h] * scale : 0.f;
        top = fmaxf(top, fabsf(f[h]));
      }
      if constexpr (std::is_same<T, f16>::value) e = tile_exponent(row_max16(top));
#pragma unroll
      for (int h = 0; h < SUB; ++h) {
        const Parts two = parts_of<T>(f[h], e);
        if (q < 2) v[row * ld + 2 * W * r + W * q + 16 * h + i] = q ? two.low : two.high;
        if (lane == 0) power[row][r] = two.power;
      }
    }
    __syncthreads();
  }
  for (int c0 = begin; c0 < end; c0 += STEP) {
    f32x4 sum[2] = {};
    for (int r0 = 0; r0 < tiles && cur >= 0; r0 += RT) {
      if (r0) load_b(c0, r0);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r0 + r >= tiles) continue;
        u32x4 low[SUB];
#pragma unroll
        for (int h = 0; h < SUB; ++h) low[h] = *(const u32x4*)(v + i * ld + 2 * W * (r0 + r) + W * h + 8 * q);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (r0 + r == tiles - 1) bv[c][r] &= mask;
          if constexpr (std::is_same<T, f16>::value) {
            const f32x4 one = both_parts<T, W>(bv[c][r], low, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[c][j] = fmaf(one[j], power[i][r0 + r], sum[c][j]);
          } else {
            sum[c] = both_parts<T, W>(bv[c][r], low, sum[c]);
          }
        }
      }
    }
    const u32x4 now = from;
    if (c0 + STEP < end) {
      load_base(c0 + STEP);
      if (cur >= 0) load_b(c0 + STEP, 0);
    }
    if (mine && c0 + 8 * q < end) *(u32x4_any*)(p.out + m * p.ldo + c0 + 8 * q) = added<T>(now, sum[0], sum[1]);
  }
  if (part + 1 == parts && p.N > p.whole) {
    __syncthreads();  // groups.found
    odd_columns<T, W>(p, b, [&](int row) { return (int64_t)groups.found.row[row]; }, 16, g.rows, cur >= 0,
                      [&](int row) { return v + row * ld; }, [&](int row, int r) { return power[row][r]; });
  }
}

// Many rows: 64 by p.cols columns, 64 of them at a time: their B goes through LDS once for the four waves, which have 16 rows
// each, and the next 64 columns' is on its way meanwhile.  Tile c of the four holds the columns 16 (i / 4) + 4 c + i % 4, so
// that lane (q, i) ends with the sixteen columns 16 q .. 16 q + 15 of row i.  Neighbouring lanes swap halves of theirs, so that each
// load and store of base and out covers whole lines of 128 bytes.  Two adapters at a time, so that a tile where one request ends
// and the next begins takes no longer; the rows without an adapter go with the first two.
// Neighbouring blocks have neighbouring columns, so that (in eights) an XCD reads the same columns' B for all row tiles.
// 4096 rows, N = 24576, rank 64: 97 us, base and out at 4.1 TB/s; 82 without the products and their B.
template <typename T, int RT, int W, bool THROUGH>
__global__ void __launch_bounds__(256, 3) lora_columns_kernel(LoraArgs p) {
  constexpr int ROWS = 64, SUB = W / 16, LD = W * RT + 8, ROW = W * RT / 8, PIECES = 64 * ROW, EACH = (PIECES + 255) / 256;
  // [buffer][adapter][column][rank], the columns as the lanes take them: number 16 c + i of tile c and lane i
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][2][64][LD];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4, i = lane & 15, odd = i & 1;
  const int tiles = p.ranks / W, chunks = (tiles + RT - 1) / RT, y = blockIdx.x % p.ranges;
  const int64_t m0 = (int64_t)(blockIdx.x / p.ranges) * ROWS, mw = m0 + 16 * wave;
  const int id = m0 + lane < p.M ? lora_id(p, m0 + lane) : -2;
  const int begin = y * p.cols, end = min(begin + p.cols, p.whole);
  const bool in_place = p.out == p.base && p.ldo == p.ldb;
  uint64_t left = __ballot(id >= 0), none = __ballot(id == -1);
  for (bool more = true; more; more = left != 0) {
    // the two adapters' numbers and rows; a wave's own rows are bits 16 wave ..
    int cur[2] = {-1, -1};
    uint64_t rows[2] = {0, 0};
#pragma unroll
    for (int g = 0; g < 2; ++g)
      if (left) {
        cur[g] = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        rows[g] = __ballot(id == cur[g]);
        left &= ~rows[g];
      }
    const uint64_t written = rows[0] | rows[1] | (in_place ? 0 : none);
    const uint32_t mine[2] = {(uint32_t)(rows[0] >> 16 * wave) & 0xFFFF, (uint32_t)(rows[1] >> 16 * wave) & 0xFFFF};
    const uint32_t touched = (uint32_t)(written >> 16 * wave) & 0xFFFF;
    const bool second = mine[1] >> i & 1, neither = !((mine[0] | mine[1]) >> i & 1);
    u32x4 stage[2][EACH], bs[2], low[RT][SUB];
    float power[RT];
    auto load_b = [&](int c0, int chunk) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (cur[g] < 0) continue;
        const uint16_t* const b = p.b + cur[g] * p.b_stride;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int piece = t + 256 * e, col = piece / ROW, at = W * RT * chunk + 8 * (piece % ROW);
          if (PIECES % 256 && piece >= PIECES) continue;
          stage[g][e] = u32x4{0, 0, 0, 0};
          if (at >= p.R) continue;
          stage[g][e] = *(const u32x4_any*)(b + (int64_t)min(c0 + col, p.whole - 1) * p.R + at);
          if (at + 8 <= p.R) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            stage[g][e][j] &= (at + 2 * j < p.R ? 0xFFFFu : 0u) | (at + 2 * j + 1 < p.R ? 0xFFFF0000u : 0u);
        }
      }
    };
    // a lane's loads and stores: both rows of a pair, the even or the odd half of their sixteen columns
    auto load_base = [&](int c0) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        bs[k] = u32x4{0, 0, 0, 0};
        if (p.base && (touched >> ((i & ~1) + k) & 1) && c0 + 16 * q + 8 * odd < end)
          bs[k] = *(const u32x4_any*)(p.base + (mw + (i & ~1) + k) * p.ldb + c0 + 16 * q + 8 * odd);
      }
    };
    auto load_low = [&](int chunk) {
      const int64_t m = min(mw + i, p.M - 1);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (chunk * RT + r >= tiles) continue;
#pragma unroll
        for (int h = 0; h < SUB; ++h) low[r][h] = *(const u32x4*)(p.v + m * 2 * p.ranks + 2 * W * (chunk * RT + r) + W * h + 8 * q);
        if constexpr (std::is_same<T, f16>::value) power[r] = p.powers[m * tiles + chunk * RT + r];
      }
    };
    if (begin < end) {  // with few columns none goes by eight
      load_b(begin, 0);
      load_low(0);
      load_base(begin);
    }
    __syncthreads();  // the adapters before are done with the LDS
    int buf = 0;
    for (int c0 = begin; c0 < end; c0 += 64) {
      f32x4 sum[4] = {};
      if (cur[0] >= 0) {
        for (int chunk = 0; chunk < chunks; ++chunk, buf ^= 1) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (cur[g] < 0) continue;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
              const int piece = t + 256 * e;
              if (PIECES % 256 && piece >= PIECES) continue;
              const int col = piece / ROW;
              *(u32x4*)&lds[buf][g][16 * (col >> 2 & 3) + 4 * (col >> 4) + (col & 3)][8 * (piece % ROW)] = stage[g][e];
            }
          }
          __syncthreads();
          if (chunk + 1 < chunks) load_b(c0, chunk + 1);
          else if (c0 + 64 < end) load_b(c0 + 64, 0);
          auto multiply = [&](int g, f32x4 (&to)[4]) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              if (chunk * RT + r >= tiles) continue;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const u32x4 bv = *(const u32x4*)&lds[buf][g][16 * c + i][W * r + first_rank<W>(q)];
                if constexpr (std::is_same<T, f16>::value) {
                  const f32x4 one = both_parts<T, W>(bv, low[r], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                  for (int j = 0; j < 4; ++j) to[c][j] = fmaf(one[j], power[r], to[c][j]);
                } else {
                  to[c] = both_parts<T, W>(bv, low[r], to[c]);
                }
              }
            }
          };
          if (mine[0] && mine[1]) {  // a wave where one request ends and the next begins
            f32x4 with[4] = {sum[0], sum[1], sum[2], sum[3]};
            multiply(0, sum);
            multiply(1, with);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int j = 0; j < 4; ++j) sum[c][j] = second ? with[c][j] : sum[c][j];
          } else if (mine[0] | mine[1]) {
            multiply(mine[0] ? 0 : 1, sum);
          }
          if (chunks > 1) load_low(chunk + 1 < chunks ? chunk + 1 : 0);
        }
      }
      const u32x4 now[2] = {bs[0], bs[1]};
      if (c0 + 64 < end) load_base(c0 + 64);
      if (neither) sum[0] = sum[1] = sum[2] = sum[3] = f32x4{0.f, 0.f, 0.f, 0.f};
      const u32x4 got = from_neighbour(odd ? now[0] : now[1]);
      const u32x4 o0 = added<T>(odd ? got : now[0], sum[0], sum[1]), o1 = added<T>(odd ? now[1] : got, sum[2], sum[3]);
      const u32x4 other = from_neighbour(odd ? o0 : o1);
      const u32x4 o[2] = {odd ? other : o0, odd ? o1 : other};
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if ((touched >> ((i & ~1) + k) & 1) && c0 + 16 * q + 8 * odd < end) {
          u32x4_any* const to = (u32x4_any*)(p.out + (mw + (i & ~1) + k) * p.ldo + c0 + 16 * q + 8 * odd);
          if constexpr (THROUGH) __builtin_nontemporal_store(o[k], to);
          else *to = o[k];
        }
    }
    if (y + 1 == p.ranges) {
      auto at = [&](int row) { return m0 + row; };
      auto parts = [&](int row) { return p.v + (m0 + row) * 2 * p.ranks; };
      auto powers = [&](int row, int r) { return std::is_same<T, f16>::value ? p.powers[(m0 + row) * tiles + r] : 1.f; };
#pragma unroll
      for (int g = 0; g < 2; ++g) odd_columns<T, W>(p, p.b + max(cur[g], 0) * p.b_stride, at, 64, rows[g], true, parts, powers);
      if (!in_place) odd_columns<T, W>(p, p.b, at, 64, none, false, parts, powers);
    }
    none = 0;
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

static int64_t lora_tile(int64_t R) { return R <= 16 ? 16 : 32; }
static int64_t lora_ranks(int64_t R) { return cdiv(R, lora_tile(R)) * lora_tile(R); }

// Columns that go by eight: whole pieces of out, and B's pieces of eight ranks, of which a row's last may reach into the next
// row, end with B.
static int64_t lora_whole(int64_t N, int64_t R) {
  const int64_t past = cdiv(R, 8) * 8 - R;
  return std::max<int64_t>(0, N - cdiv(past, R)) / 8 * 8;
}

struct LoraPlan {
  bool many, own;  // own: the few rows' v by the blocks themselves
  int slots, splits, shares;
};
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t R) {
  LoraPlan l{};
  const int64_t tiles = cdiv(M, 16), units = cdiv(K, kUnit), ranks = lora_ranks(R);
  // Up to here rows may be single tokens of as many requests: 256 rows, N = 6144, rank 16, 64 adapters 17 us, by the kernels for many
  // rows 44, rank 64 26 and 82, 500 rows, N = 4096, rank 32 22 and 59.  Prompts of so many rows gain less or lose some: 256 of four
  // requests 9.7 and 11.3, rank 64 17.5 and 19.2, 500 of three, rank 32 14.1 and 12.1, 300, rank 128 31 and 19.
  l.many = M > kFewRows;
  // Of many rows a tile has one adapter or two if they are prompts, but may have 16; blocks that find none cost little but wait
  // for LDS (8192 rows of 6 requests 48 us with 4, 54 with 16).
  l.slots = (int)(l.many ? 4 : std::min<int64_t>(16, M));
  // One launch where few rows' adapters are small enough to be read by all of a row's blocks.  us with one and with two, which
  // cost the host 4 more (one row: A of 128 KB 6.3, 6.2, of 256 7.9, 6.7, of 384 11.2, 6.5; 64 rows of as many adapters: 128 KB
  // 9.9, 12.9, 256 13.5, 16.1, 512 19.8, 25.0; 128 rows: 128 KB 12.7, 16.8, 256 KB and two adapters 21.4, 18.1; 500 rows: 64 KB 21, 27).
  l.own = !l.many && ranks <= 64 && K >= 8 && ranks * K * 2 <= (M <= 32 ? 256 << 10 : M <= 64 ? 512 << 10 : 128 << 10);
  // at least four units a share, at most 16 shares
  l.splits = (int)std::max<int64_t>(1, std::min(cdiv(units, 4), std::min<int64_t>(16, 256 / (tiles * l.slots * cdiv(ranks, 64)))));
  l.shares = K < 8 ? 1 : std::min(16, l.splits * l.slots);
  return l;
}
size_t lora_workspace_bytes(int64_t M, int64_t K, int64_t R) {
  const LoraPlan l = lora_plan(M, K, R);
  const size_t values = (size_t)M * (size_t)lora_ranks(R);
  if (l.own) return 0;
  if (l.many) return values * 4 + values / (size_t)lora_tile(R) * 4;
  return (size_t)l.shares * values * 4 + (size_t)(cdiv(M, 16) * l.slots) * sizeof(GroupRecord);
}

template <typename T>
static int lora_typed(LoraArgs p, const LoraPlan& l, hipStream_t st) {
  using std::integral_constant;
  // tiles of 16 ranks a block of the first launch, of W ranks at a time in the second, and W
  auto by_rank = [&](auto f) {
    if (p.ranks == 16) f(integral_constant<int, 1>{}, integral_constant<int, 1>{}, integral_constant<int, 16>{});
    else if (p.ranks == 32) f(integral_constant<int, 2>{}, integral_constant<int, 1>{}, integral_constant<int, 32>{});
    else f(integral_constant<int, 4>{}, integral_constant<int, 2>{}, integral_constant<int, 32>{});
  };
  if (!l.own) by_rank([&](auto n, auto, auto w) {
    constexpr int N = decltype(n)::value, W = decltype(w)::value;
    if (p.K < 8) {
      const dim3 grid((unsigned)cdiv(p.M, 256 / W), (unsigned)(p.ranks / W));
      if (l.many) lora_ranks_short_kernel<T, W, true><<<grid, 256, 0, st>>>(p);
      else lora_ranks_short_kernel<T, W, false><<<grid, 256, 0, st>>>(p);
      return;
    }
    const unsigned x = (unsigned)(p.tiles * p.slots), y = (unsigned)cdiv(p.ranks, 16 * N);
    if (!l.many) lora_ranks_few_kernel<T, N, W><<<dim3(x, y, (unsigned)l.splits), 256, 0, st>>>(p);
    else if (N == 4 && p.tiles < 64) lora_ranks_kernel<T, 2, W><<<dim3(x, (unsigned)cdiv(p.ranks, 32)), 64 * many_waves(2), 0, st>>>(p);
    else lora_ranks_kernel<T, N, W><<<dim3(x, y), 64 * many_waves(N), 0, st>>>(p);
  });
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  const int64_t x = l.many ? cdiv(p.M, 64) : p.tiles * p.slots, step = l.many ? 64 : 32 * few_waves(l.own);
  const int64_t steps = std::max<int64_t>(1, cdiv(p.whole, step)), want = std::max<int64_t>(1, (l.own ? 256 : l.many || p.M <= 128 ? 2048 : 1024) / x);
  // (256 rows of four requests, rank 64: 17.3 us with 1024 blocks, 21.1 with 2048)
  p.cols = (int)(cdiv(steps, std::min(want, steps)) * step);
  // many rows: not so many columns that the last blocks' work shows (4096 rows, N = 24576: rank 16 99 us with 768 columns a
  // block, 92 with 256, rank 64 127 and, with 512, 123)
  if (l.many) p.cols = std::min(p.cols, p.ranks <= 32 ? 256 : 512);
  p.ranges = (int)std::max<int64_t>(1, cdiv(p.whole, p.cols));
  // results past the caches where they are many (and not in lines that base has brought there): N = 24576, rank 64, 4096 rows
  // 112 us, 150 through them; 8192 columns of 2000 rows gain 3 us of 24, but the next reader may want those
  const bool through = p.out != p.base && p.M * p.N >= (int64_t)32 << 20;
  by_rank([&](auto o, auto n, auto w) {
    constexpr int RT = decltype(n)::value, W = decltype(w)::value;
    const size_t lds = (size_t)16 * (2 * p.ranks + 8) * 2;
    const dim3 blocks((unsigned)(x * p.ranges));
    if (l.many && through) lora_columns_kernel<T, RT, W, true><<<blocks, 256, 0, st>>>(p);
    else if (l.many) lora_columns_kernel<T, RT, W, false><<<blocks, 256, 0, st>>>(p);
    else if (l.own) lora_columns_few_kernel<T, RT, W, decltype(o)::value><<<dim3((unsigned)x, (unsigned)p.ranges), 64 * few_waves(true), lds, st>>>(p);
    else lora_columns_few_kernel<T, RT, W, 0><<<dim3((unsigned)x, (unsigned)p.ranges), 256, lds, st>>>(p);
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
  p.tiles = (int)cdiv(c.M, 16), p.slots = l.slots, p.splits = l.splits, p.shares = l.shares;
  p.partial = (float*)c.workspace;
  if (!l.many && !l.own && c.K >= 8) p.records = (GroupRecord*)(p.partial + (size_t)l.shares * (size_t)(c.M * p.ranks));
  p.v = (uint16_t*)c.workspace, p.powers = (float*)(p.v + (size_t)c.M * 2 * p.ranks);
  return c.dtype == AWQ_DTYPE_F16 ? lora_typed<f16>(p, l, st) : lora_typed<bf16>(p, l, st);
}

}  // namespace awq_host
