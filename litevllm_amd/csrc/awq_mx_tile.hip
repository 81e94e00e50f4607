// Products of microscaled fp4 matrices, many rows: tiles of both operands in LDS (format, modes and operand
// order: awq_mx_common.h).
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"
#include "awq_mx_span.h"

namespace awq {

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"
__device__ __forceinline__ u32x4 lds_read16(uint32_t at) { return *(const __attribute__((address_space(3))) u32x4*)at; }
__device__ __forceinline__ uint32_t lds_read1(uint32_t at) { return *(const __attribute__((address_space(3))) uint8_t*)at; }
#pragma clang diagnostic pop

// LDS of a block of `rows` rows (of both operands): two stages of 256 along K, two groups of 16 scale bytes a row
// (a group serves two stages), and zeros to read as scales behind K's end.
__host__ __device__ constexpr int mx_tile_lds(int rows, int tiles16) { return rows * 2 * (128 + 16) + tiles16 * 256; }

// All but the N newest direct loads have landed and every LDS read is done, in every wave.
template <int N>
__device__ __forceinline__ void wait_loads_and_sync() {
  static_assert(N < 64, "the counter's range");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// acc[j] += b[j] . a^T for two neighbouring column tiles, as one piece of assembly: the compiler moves the builtin
// behind the reads of whole stages, runs out of registers, and copies accumulators (M = 4096, N = 24576,
// K = 4096: 404 us with it).  The wait states in front cover a copy of an operand by the VALU; the accumulators
// may be used 18 wait states after the last of these.
__device__ __forceinline__ void mfma2(f32x4& c0, f32x4& c1, const u32x4& b0, const u32x4& b1, const u32x4& a, uint32_t s0, uint32_t s1,
                                      uint32_t sa) {
  asm volatile(
      "s_nop 1\n\t"
      "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %2, %4, %0, %5, %7 op_sel_hi:[0,0,0] cbsz:4 blgp:4\n\t"
      "v_mfma_scale_f32_16x16x128_f8f6f4 %1, %3, %4, %1, %6, %7 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
      : "+v"(c0), "+v"(c1)
      : "v"(b0), "v"(b1), "v"(a), "v"(s0), "v"(s1), "v"(sa));
}

// x and y of 16 rows in 16 lanes r: afterwards lane r holds row r & 7 in x and row 8 + (r & 7) in y, both times of what was
// x where r < 8 and of what was y where not: stores of a piece of 8 rows instead of half a one of 16.
__device__ __forceinline__ void swap_rows(u32x4& x, u32x4& y, bool low) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(low ? y[d] : x[d]), 0x128 /* row_ror:8 */, 0xF, 0xF, true);
    if (low) y[d] = other;
    else x[d] = other;
  }
}

// Block: tiles of BM rows of a by BN rows of w, one after another, WM x WN waves of (BM / WM) x (BN / WN).  A stage of
// 256 along K (one line of codes a row) is loaded straight into LDS while the one before it is used, in two halves of 128; a
// wave holds the fragments of a half while it reads the next half's, so the buffer of a stage is free after its first
// half: one barrier a stage, the loads under way for a whole stage's time.  A tile's first two stages are loaded while
// the results of the tile before go out, which takes no LDS (M = 4096, N = 24576, K = 4096: 228 us with blocks of one tile
// whose results go through LDS, 221 so; K = 1024 90 and 82; 100 tokens through 64 experts 53 and 48).
//
// What bounds it (M = 4096, N = 24576, K = 4096, 221 to 235 us by card and run, 3.5 to 3.7 PFLOP/s): where it takes 221, its
// products alone take 143, its LDS reads 98, its loads 128, products and reads 168, all but the stores 204, scales that need
// not be read 212.
//
// LDS: 16-byte chunk c (block c of the stage) of a row at place c ^ (row & 7) of its 128 bytes, so that the 16
// rows of a fragment lie in different banks; the direct loads write lanes in order, so it is their sources that
// are permuted, inside the row's line.  (Loads of half a line, in stages of 128, took 139 us where these take
// 102: M = 4096, N = 24576, K = 4096, loads alone.)  The scale bytes come 16 a row, one load for two stages: a
// row's bytes start anywhere in a word (K / 32 need not be a multiple of 4), so the loads start at the word and
// the readers skip `sh` bytes, for the last ones into the next group.
// The operands enter the MFMA swapped, so that a lane holds four consecutive columns of one row of c.
//
// WK > 1 (few tiles, where the latency of a stage bounds a block): as many shares of K, each with waves and LDS of its
// own, whose sums meet at the end; such a block has one tile.
//
// K past the end: the codes are the next row's, or zeros behind the operand's last (any code is finite; what may be read:
// awq_mx_span.h), both scales are 2^-127, and the products vanish in fp32.
template <int MODE, int BM, int BN, int WM, int WN, int PER_SIMD, int WK>
__global__ void __launch_bounds__(WM * WN * WK * 64, PER_SIMD) mx_tile_kernel(MxArgs p, int row_tiles, int col_tiles) {
  constexpr int WAVES = WM * WN /* of a share of K */, TM = BM / WM / 16, TN = BN / WN / 16, ROWS = BM + BN, STAGE = ROWS * 128;
  static_assert(TN == 2 || TN == 4, "");
  extern __shared__ __align__(16) uint8_t lds[];  // codes [2][ROWS][128], scales [2][ROWS][16], zeros

  // Blocks go to the 8 XCDs in turn: each takes a run of tiles, in groups of 8 row tiles, column by column, so
  // that the tiles it runs at once share rows of a and of w in its L2.  Row tiles of a table share rows of w only where an
  // expert has several: they run one after another (64 experts, 500 tokens 65.8 us against 70.1 in groups of 8, 2048 170
  // against 176; 32 experts, H = 4096 391 and 401).
  constexpr int GROUP = MODE == kMxDense ? 8 : 1;
  if (MODE != kMxDense) row_tiles = p.tile_count[0];
  const int tiles = row_tiles * col_tiles, per = (tiles + 7) / 8;
  const int first_id = ((int)blockIdx.x & 7) * per, ids = min(per, tiles - first_id);
  int in_run = (int)blockIdx.x >> 3;
  if (in_run >= ids) return;
  constexpr int COLS = MODE == kMxGateUp ? BN / 2 : BN;

  // wave: of the WM x WN of share `part` of K
  const int tid = threadIdx.x, wave_of_all = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave_of_all / WAVES, wave = wave_of_all % WAVES;
  const int lane = tid & 63, r = lane & 15, q = lane >> 4, ptid = tid - part * (WAVES * 64);
  const int KB = p.K / 32;
  // the share's stages, as if the operands began and ended there (a share behind K's end: stages of nothing)
  const int stages = ((KB + 7) / 8 + WK - 1) / WK, s0 = part * stages, blocks = KB - 8 * s0;
  // Stages whose position is in the scalar offset: all that may have it (awq_mx_span.h) where no register is left for sums
  // (256 x 256 243 us against 245) or K is in shares (M = 57, N = 6144 11.4 and 11.7), else none, for a branch less
  // (M = 700, N = 4096 20.8 and 20.1; M = 200, N = 5001 17.2 and 16.8; 2048 tokens through 64 experts 171.5 and 170.8).
  const int whole = BM == 256 || WK > 1 ? mx_whole_stages(KB, s0, stages) : 0;
  // the wave's rows and columns in the tile
  const int m0 = (wave / WN) * TM * 16, c0 = BM + (wave % WN) * TN * 16;

  // this wave's loads of a stage: LOADS of 8 rows, the first A_LOADS of them a's; of a group of scales: those
  // of 64 rows, in SLOADS loads (the last one not of every wave)
  constexpr int LOADS = ROWS / (8 * WAVES), A_LOADS = BM / (8 * WAVES), SLOADS = (ROWS + 64 * WAVES - 1) / (64 * WAVES);
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && BM % 64 == 0 && BN % 64 == 0, "whole loads");
  // of the tile at hand: its rows, its first column (of c, or of the gate half), what its loads read
  MxRows t;
  int n0;
  u32x4 ars, wrs, asrs, wsrs;
  uint32_t src[LOADS], ssrc[SLOADS], sh_a, sh_b;
  constexpr int PLACES = MODE == kMxDown ? 2 * TM : 1;
  int place[PLACES] = {};  // kMxDown: rows of y of this lane's stores
  auto set_tile = [&](int id) {
    const int group = id / (GROUP * col_tiles), in_group = id - group * GROUP * col_tiles;
    const int group_rows = min(GROUP, row_tiles - GROUP * group);
    t = mx_rows<MODE, BM>(p, GROUP * group + in_group % group_rows);
    n0 = in_group / group_rows * COLS;
    const int64_t a_base = MODE == kMxGateUp ? 0 : t.first, w_base = (int64_t)t.expert * p.wrows + n0;
    const int last = p.N - 1 - n0;
    // row i of a stage (a's rows, then w's: a wave's gate columns and then their up columns) behind the operand's base
    auto row_of = [&](int i) -> uint32_t {
      if (i < BM) return (uint32_t)(mx_a_row<MODE>(p, t, i) - a_base);
      return mx_w_row(MODE == kMxGateUp, i - BM, last, p.N);
    };
    // what the tile's loads may read: gathered rows are all of a's; scales begin with the word that holds the first one
    const uint32_t a_rows = MODE == kMxGateUp ? (uint32_t)p.a_rows : (uint32_t)t.rows, w_rows = mx_w_rows(MODE == kMxGateUp, BN, last, p.N);
    const uint64_t as = (uint64_t)(uintptr_t)p.as + (uint64_t)(a_base * p.as_ld), ws = (uint64_t)(uintptr_t)p.ws + (uint64_t)(w_base * KB);
    const uint32_t a_in = (uint32_t)as & 3u, w_in = (uint32_t)ws & 3u;
    auto rsrc = [](uint64_t base, uint32_t bytes) { return u32x4{(uint32_t)base, (uint32_t)(base >> 32) & 0xFFFFu, bytes, 0x00020000u}; };
    ars = rsrc((uint64_t)(uintptr_t)p.a + (uint64_t)(a_base * KB * 16), mx_code_bytes(a_rows, KB));
    wrs = rsrc((uint64_t)(uintptr_t)p.w + (uint64_t)(w_base * KB * 16), mx_code_bytes(w_rows, KB));
    asrs = rsrc(as - a_in, mx_scale_bytes(a_rows, p.as_ld, KB, a_in));
    wsrs = rsrc(ws - w_in, mx_scale_bytes(w_rows, KB, KB, w_in));
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = (u * WAVES + wave) * 8 + (lane >> 3);
      src[u] = mx_code_offset(row_of(i), KB, lane);
    }
#pragma unroll
    for (int u = 0; u < SLOADS; ++u) {
      const int i = min((u * WAVES + wave) * 64 + lane, ROWS - 1);
      ssrc[u] = mx_scale_offset(row_of(i), i < BM ? p.as_ld : KB, i < BM ? a_in : w_in);
    }
    // the rows of a fragment's next 16 are a multiple of 16 bytes on, and those of a gathered operand whole words: a
    // lane's scale bytes start alike in all its row tiles
    sh_a = ((MODE == kMxGateUp ? 0u : (uint32_t)r * (uint32_t)p.as_ld) + a_in & 3u) + (uint32_t)q;
    sh_b = (row_of(c0 + r) * (uint32_t)KB + w_in & 3u) + (uint32_t)q;
    if constexpr (MODE == kMxDown) {
#pragma unroll
      for (int k = 0; k < PLACES; ++k) place[k] = p.order[t.first + min(m0 + 8 * k + (r & 7), t.rows - 1)];
    }
  };
  constexpr uint32_t SHARE_LDS = mx_tile_lds(ROWS, TM > TN ? TM : TN);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + part * SHARE_LDS;
  constexpr uint32_t SCALES = 2 * STAGE, ZEROS = SCALES + 2 * ROWS * 16;
  // loads `from` .. `to` - 1 of stage s's LOADS
  auto load_codes = [&](int s, int from, int to) {
    auto all = [&](uint32_t voff, uint32_t soff) {
#pragma unroll
      for (int u = from; u < to && u < LOADS; ++u)
        lds_dma16<true>(u < A_LOADS ? ars : wrs, lds0 + (uint32_t)((s & 1) * STAGE + (u * WAVES + wave) * 1024), src[u] + voff, soff);
    };
    if (s < whole) all(0u, mx_code_position(s0 + s));
    else all(mx_code_position(s0 + s), 0u);
  };
  auto load_scales = [&](int g) {
#pragma unroll
    for (int u = 0; u < SLOADS; ++u) {
      const int at = u * WAVES + wave;
      if (ROWS % (64 * WAVES) != 0 && at * 64 >= ROWS) continue;
      lds_dma16<true>(at * 64 < BM ? asrs : wsrs, lds0 + SCALES + (uint32_t)((g & 1) * ROWS * 16 + at * 1024), ssrc[u] + mx_scale_position(s0, g), 0u);
    }
  };

  f32x4 acc[TM][TN];
  // where this lane reads its fragments (16 rows on: 2048 bytes) and their scales (256 bytes)
  uint32_t rd_a[2], rd_b[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t chunk = (uint32_t)((4 * h + q) ^ (r & 7)) * 16u;
    rd_a[h] = lds0 + (uint32_t)(m0 + r) * 128u + chunk;
    rd_b[h] = lds0 + (uint32_t)(c0 + r) * 128u + chunk;
  }
  // address of the scale of block q of half h of stage s
  auto scale_at = [&](int s, int h, uint32_t row, uint32_t sh) -> uint32_t {
    const uint32_t at = sh + (uint32_t)(8 * (s & 1) + 4 * h);  // byte in the group of 16
    const uint32_t group = (uint32_t)(s >> 1) + (at >> 4);
    uint32_t place = lds0 + SCALES + (group & 1) * (ROWS * 16) + row * 16u + (at & 15u);
    asm("" : "+v"(place));  // a select, no branch around it
    return 8 * s + 4 * h + q < blocks ? place : lds0 + ZEROS;
  };
  // the fragments of a half: a's row tile i, and all of w's, with their scales
  u32x4 a[TM];
  uint32_t sa[TM];
  struct Cols {
    u32x4 b[TN];
    uint32_t s[TN];
  };
  auto read_a = [&](int s, int h, uint32_t scales, int i) {
    a[i] = lds_read16(rd_a[h] + (uint32_t)(s & 1) * STAGE + i * 2048);
    sa[i] = lds_read1(scales + i * 256);
  };
  auto read_cols = [&](int s, int h, Cols& c) {
    const uint32_t at = scale_at(s, h, (uint32_t)(c0 + r), sh_b);
#pragma unroll
    for (int j = 0; j < TN; ++j) c.b[j] = lds_read16(rd_b[h] + (uint32_t)(s & 1) * STAGE + j * 2048);
#pragma unroll
    for (int j = 0; j < TN; ++j) c.s[j] = lds_read1(at + j * 256);
  };
  Cols first, second;
  auto products = [&](int i, const Cols& now) {
#pragma unroll
    for (int j = 0; j < TN; j += 2) mfma2(acc[i][j], acc[i][j + 1], now.b[j], now.b[j + 1], a[i], now.s[j], now.s[j + 1], sa[i]);
  };
  // a's fragments have one place: each is read again, for the next half, as soon as its products are under way

  // the loads of a tile's first two stages
  auto load_first = [&]() {
    load_scales(0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= stages) break;
      if (s & 1) load_scales(1);  // before the codes of the first stage that reads from it
      load_codes(s, 0, LOADS);
    }
  };
  // the results of a tile go out behind the next one's first loads, in at least STORES stores where this wave's part of
  // the tile is full (`stored`): its waits leave them under way, too
  constexpr int STORES = MODE == kMxDense ? TM * TN / 2 : (MODE == kMxDown ? TM * TN : 2 * TM);
  bool stored = false;
  // stage s + 1 is there, stage s has been read
  auto next_stage = [&](int s) {
    if (s == 0 && stored) wait_loads_and_sync<STORES>();
    else wait_loads_and_sync<0>();
  };

  for (int i = ptid; i < (TM > TN ? TM : TN) * 64; i += WAVES * 64) ((uint32_t*)(lds + part * SHARE_LDS + ZEROS))[i] = 0u;
  set_tile(first_id + in_run);
  load_first();
  for (;;) {
    // the sums begin with the bias
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      f32x4 from = {0.f, 0.f, 0.f, 0.f};
      if constexpr (MODE == kMxDense) {
        const int n = n0 + c0 - BM + 16 * j + 4 * q;
        if (p.bias && part == 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) from[e] = n + e < p.N ? load_bias(p.bias, p.bias_dtype, n + e) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = from;
    }
    if (stages < 2) wait_loads_and_sync<0>();
    else if (stored) wait_loads_and_sync<LOADS + STORES>();
    else wait_loads_and_sync<LOADS>();
    {
      const uint32_t at = scale_at(0, 0, (uint32_t)(m0 + r), sh_a);
      read_cols(0, 0, first);
#pragma unroll
      for (int i = 0; i < TM; ++i) read_a(0, 0, at, i);
    }
    // a wave whose rows all lie behind the tile's last only loads (an expert's last tile is half empty on average)
    const bool idle = MODE != kMxDense && m0 >= t.rows;
    for (int s = 0; idle && s < stages; ++s) {
      next_stage(s);
      if (s + 2 < stages) {
        if (s & 1) load_scales((s + 3) >> 1);
        load_codes(s + 2, 0, LOADS);
      }
    }
    for (int s = 0; !idle && s < stages; ++s) {
      {
        const uint32_t at = scale_at(s, 1, (uint32_t)(m0 + r), sh_a);
        read_cols(s, 1, second);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          products(i, first);
          read_a(s, 1, at, i);
        }
      }
      // The second half's reads are of the next stage, so they begin behind the barrier, which comes after its first
      // products: by then the reads that it waits for have come back.  The loads of stage s + 2 go out between the
      // products.  (After the last stage the fragments are of nothing, and nobody uses them.)
      constexpr int SHARE = (LOADS + TM - 1) / TM;
      const uint32_t at = scale_at(s + 1, 0, (uint32_t)(m0 + r), sh_a);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        products(i, second);
        if (i == 0) {
          next_stage(s);
          read_cols(s + 1, 0, first);
          if ((s & 1) && s + 2 < stages) load_scales((s + 3) >> 1);
        }
        read_a(s + 1, 0, at, i);
        if (s + 2 < stages) load_codes(s + 2, i * SHARE, (i + 1) * SHARE);
      }
    }
    // no use of an accumulator before the last product is through
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[i][j]));

    if constexpr (WK > 1) {
      // the shares' sums meet in LDS, in order: [share - 1][accumulator][thread]
      static_assert(MODE == kMxDense, "");
      constexpr int N4 = TM * TN, THREADS = WAVES * 64;
      static_assert((WK - 1) * N4 * THREADS * 16 <= WK * SHARE_LDS, "the shares' sums");
      f32x4* sums = (f32x4*)lds;
      __syncthreads();
      if (part > 0) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) sums[((part - 1) * N4 + i * TN + j) * THREADS + ptid] = acc[i][j];
      }
      __syncthreads();
      if (part > 0) return;
#pragma unroll
      for (int k = 0; k < WK - 1; ++k)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] += sums[(k * N4 + i * TN + j) * THREADS + ptid];
    }

    // what the results need of this tile; all waves are past the last stage's barrier, so the LDS is free for the next
    const MxRows done = t;
    const int nw = n0 + (MODE == kMxGateUp ? (c0 - BM) / 2 : c0 - BM), rows = t.rows - m0;  // the wave's first column, its rows
    int put[PLACES];
#pragma unroll
    for (int k = 0; k < PLACES; ++k) put[k] = place[k];
    in_run += (int)gridDim.x >> 3;
    const bool more = WK == 1 && in_run < ids;
    if (more) {
      set_tile(first_id + in_run);
      load_first();
    }

    // lane: row m0 + 16 i + r, columns 16 j + 4 q .. + 3
    int er = r;
    asm volatile("" : "+v"(er));  // addresses are formed here, not kept in registers (or behind them) over the loop
    const bool low = er < 8;
    const int r8 = er & 7;
    if constexpr (MODE == kMxGateUp) {
      // tiles 0, 1: 32 gate columns, 2, 3: their up columns, a block of h
      static_assert(TN == 4, "");
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = 16 * i + er;
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[4 * d + e] = mx_gated(acc[i][d][e], acc[i][d + 2][e], p.act);
            top = max(top, mx_abs_bits(v[4 * d + e]));
          }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const uint32_t byte = mx_scale_byte(top);
        const uint32_t codes = byte == 255u ? 0u : mx_codes8(v, mx_scale_value(byte));
        if (m < rows && nw < p.N) {
          const int64_t at = done.first + m0 + m;
          uint8_t* o = p.h + at * (p.N / 2) + nw / 2 + 2 * q;
          *(uint16_t*)o = (uint16_t)codes;
          *(uint16_t*)(o + 8) = (uint16_t)(codes >> 16);
          if (q == 0) p.hs[at * (p.N / 32) + nw / 32] = (uint8_t)byte;
        }
      }
      stored = rows >= TM * 16 && nw < p.N;
    } else if constexpr (MODE == kMxDown) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
          u32x4 v[2] = {__builtin_bit_cast(u32x4, acc[i][j]), __builtin_bit_cast(u32x4, acc[i][j + 1])};
          swap_rows(v[0], v[1], low);
          const int n = nw + 16 * (low ? j : j + 1) + 4 * q;
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (16 * i + 8 * k + r8 < rows && n < p.N) *(u32x4*)(p.y + (int64_t)put[2 * i + k] * p.N + n) = v[k];
        }
      stored = rows >= TM * 16 && nw + TN * 16 <= p.N;
    } else {
      uint16_t* out = p.c + (int64_t)(done.first + m0) * p.ldc;
      auto pack = [&](int i, int j) {
        const f32x4& v = acc[i][j];
        return p.out_bf16 ? u32x2{pack2<bf16>(v[0], v[1]), pack2<bf16>(v[2], v[3])} : u32x2{pack2<f16>(v[0], v[1]), pack2<f16>(v[2], v[3])};
      };
      const int n = nw + 16 * (q & 1) + 8 * (q >> 1) + (TN == 2 || low ? 0 : 32), m = TN == 4 ? r8 : er;
      uint16_t* at = out + (int64_t)m * p.ldc + n;
      const int64_t step = (TN == 4 ? 8 : 16) * p.ldc;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        // lanes q and q ^ 1 put their halves of two column tiles together: columns 16 (q & 1) + 8 (q >> 1) .. + 7 of the two
        u32x4 v[TN / 2];
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
          const u32x2 x = pack(i, j), y = pack(i, j + 1);
          const auto w0 = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false), w1 = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
          v[j / 2] = u32x4{w0[0], w1[0], w0[1], w1[1]};
        }
        if constexpr (TN == 4) swap_rows(v[0], v[1], low);
#pragma unroll
        for (int k = 0; k < TN / 2; ++k, at += step) {
          if (m + 16 * i + 8 * k >= rows) continue;
          if (n + 8 <= p.N) {
            __builtin_memcpy(at, &v[k], 16);  // rows begin anywhere
          } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
              if (n + e < p.N) at[e] = (uint16_t)(v[k][e >> 1] >> (16 * (e & 1)));
          }
        }
      }
      stored = rows >= TM * 16 && nw + TN * 16 <= p.N;
    }
    if (!more) return;
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

template <int MODE, int BM, int BN, int WM, int WN, int PER_SIMD, int WK = 1>
static int launch_tile(const MxArgs& p, int64_t row_tiles, hipStream_t st) {
  constexpr int COLS = MODE == kMxGateUp ? BN / 2 : BN;
  const int64_t col_tiles = cdiv(p.N, COLS);
  if (row_tiles * col_tiles > 0x7FFFFFFLL) return AWQ_ERR_UNSUPPORTED;
  constexpr int lds = WK * mx_tile_lds(BM + BN, BM / WM > BN / WN ? BM / WM / 16 : BN / WN / 16);
  auto kernel = mx_tile_kernel<MODE, BM, BN, WM, WN, PER_SIMD, WK>;
  if (lds > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    (void)hipGetLastError();
    return AWQ_ERR_LAUNCH;
  }
  // As many blocks as run at once, each with several tiles (a tile each: 500 tokens through 64 experts 66.7 us against 63.2,
  // 100 49.4 and 47.1, 2048 170.5 and 169.5; 4096 through 32, H = 4096 391 and 397).
  constexpr int64_t AT_ONCE = WK > 1 ? 0x7FFFFFFF : 256 * (4 * PER_SIMD / (WM * WN));
  kernel<<<dim3((unsigned)std::min(cdiv(row_tiles * col_tiles, 8) * 8, AT_ONCE)), dim3(WM * WN * WK * 64), lds, st>>>(p, (int)row_tiles, (int)col_tiles);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

// Tiles of 256 x 256 run in rounds of one a CU, those of 128 x 128 two a CU; K = 4096, us with one and the other:
// M = 2048, N = 24576 112, 148; M = 3000, N = 5000 39, 48; M = 2048, N = 6144 36.5, 37.7; M = 1000, N = 24576 72, 77;
// M = 700, N = 24576 68, 59; M = 2048, N = 4096 36, 27: about 38 a round against 26 for 512 tiles.  Fewer than 160 of these:
// tiles of 64 x 64 (M = 500, N = 4096 12.2 against 14.2; 640 16.1 and 14.4; 1000 19.3 and 16.9).  Up to a tile per CU of
// these K goes in shares: two from 4 stages on, four from 24 on (M = 64, N = 4096, us with 1, 2, 4: K = 512 4.0, 4.1, 5.5;
// K = 1024 4.7, 4.5, 5.6; K = 4096 9.0, 7.3, 7.7; K = 6144 11.9, 9.1, 9.1; K = 12288 20.9, 15.2, 14.8); up to two a CU two
// from 20 on (M = 300: K = 2048 7.6, 7.7, K = 4128 12.1, 12.6, K = 8192 18.0, 16.7).
int launch_mx_tile_gemm(const MxArgs& p, hipStream_t st) {
  const int64_t big = cdiv(p.M, 256) * cdiv(p.N, 256), mid = cdiv(p.M, 128) * cdiv(p.N, 128);
  if (512 * 38 * cdiv(big, 256) <= 26 * std::max<int64_t>(512, mid)) return launch_tile<kMxDense, 256, 256, 2, 4, 2>(p, cdiv(p.M, 256), st);
  if (mid >= 160) return launch_tile<kMxDense, 128, 128, 2, 4, 4>(p, cdiv(p.M, 128), st);
  const int64_t rows = cdiv(p.M, 64), tiles = rows * cdiv(p.N, 64), stages = cdiv(p.K, 256);
  if (tiles <= 256 && stages >= 24) return launch_tile<kMxDense, 64, 64, 2, 2, 4, 4>(p, rows, st);
  if (tiles <= 256 ? stages >= 4 : tiles <= 512 && stages >= 20) return launch_tile<kMxDense, 64, 64, 2, 2, 4, 2>(p, rows, st);
  return launch_tile<kMxDense, 64, 64, 2, 2, 4>(p, rows, st);
}

// Waves of 16 or 32 rows x 64 columns (64 x 128 tiles, us with them and with 4 waves: 20 tokens through 64 experts 43.5, 44.9;
// 64 46.4, 47.5; 200 51.6, 51.3), but for down's 128 x 128 64 x 64, fewer LDS reads a product: 2048 tokens 170.5 against
// 172.5, with gate_up's so, too, 170.8, 1024 118.7 against 113.3.
int launch_mx_tile_grouped(const MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st) {
  if (rows == 128)
    return gate_up ? launch_tile<kMxGateUp, 128, 128, 4, 2, 4>(p, row_tiles, st) : launch_tile<kMxDown, 128, 128, 2, 2, 2>(p, row_tiles, st);
  return gate_up ? launch_tile<kMxGateUp, 64, 128, 4, 2, 4>(p, row_tiles, st) : launch_tile<kMxDown, 64, 128, 4, 2, 4>(p, row_tiles, st);
}

}  // namespace awq_host
