// Products of microscaled fp4 matrices, many rows: tiles of both operands in LDS (format, modes and operand
// order: awq_mx_common.h).
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"
__device__ __forceinline__ u32x4 lds_read16(uint32_t at) { return *(const __attribute__((address_space(3))) u32x4*)at; }
__device__ __forceinline__ uint32_t lds_read1(uint32_t at) { return *(const __attribute__((address_space(3))) uint8_t*)at; }
#pragma clang diagnostic pop

// LDS of a block of `rows` rows (of both operands): NBUF stages of 256 along K, NBUF groups of 16 scale bytes a row
// (a group serves two stages; NBUF / 2 + 1 of them live), and zeros to read as scales behind K's end.
__host__ __device__ constexpr int mx_tile_lds(int rows, int nbuf, int tiles16) { return rows * nbuf * (128 + 16) + tiles16 * 256; }

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

// Block: BM rows of a by BN rows of w, WM x WN waves of (BM / WM) x (BN / WN).  A stage of 256 along K (one line
// of codes a row) is loaded straight into LDS while the NBUF - 1 before it are used, in two halves of 128; a wave holds
// the fragments of a half while it reads the next half's, so the buffer of a stage is free after its first
// half: one barrier a stage, the loads under way for a whole stage's time.
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
// own, whose sums meet at the end (M = 64, K = N = 4096 9.8 us with one).
//
// K past the end: the codes are whatever follows (any code is finite, and the loads stop at the operand's end),
// both scales are 2^-127, and the products vanish in fp32.
template <int MODE, int BM, int BN, int WM, int WN, int PER_SIMD, int NBUF, int WK>
__global__ void __launch_bounds__(WM * WN * WK * 64, PER_SIMD) mx_tile_kernel(MxArgs p, int row_tiles, int col_tiles) {
  constexpr int WAVES = WM * WN /* of a share of K */, TM = BM / WM / 16, TN = BN / WN / 16, ROWS = BM + BN, STAGE = ROWS * 128;
  static_assert(TN % 2 == 0, "");
  extern __shared__ __align__(16) uint8_t lds[];  // codes [NBUF][ROWS][128], scales [NBUF][ROWS][16], zeros

  // blocks go to the 8 XCDs in turn: each takes a run of tiles, in groups of 8 row tiles, column by column, so
  // that the tiles it runs at once share rows of a and of w in its L2
  if (MODE != kMxDense) row_tiles = p.tile_count[0];
  const int tiles = row_tiles * col_tiles, per = (tiles + 7) / 8;
  const int id = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (((int)blockIdx.x >> 3) >= per || id >= tiles) return;
  const int group = id / (8 * col_tiles), in_group = id - group * 8 * col_tiles;
  const int group_rows = min(8, row_tiles - 8 * group);
  const int tm = 8 * group + in_group % group_rows, tn = in_group / group_rows;
  const MxRows t = mx_rows<MODE, BM>(p, tm);
  constexpr int COLS = MODE == kMxGateUp ? BN / 2 : BN;
  const int n0 = tn * COLS;

  // wave: of the WM x WN of share `part` of K
  const int tid = threadIdx.x, wave_of_all = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave_of_all / WAVES, wave = wave_of_all % WAVES;
  const int lane = tid & 63, r = lane & 15, q = lane >> 4, ptid = tid - part * (WAVES * 64);
  const int KB = p.K / 32;
  // the share's stages, as if the operands began and ended there (a share behind K's end: stages of nothing)
  const int stages = ((KB + 7) / 8 + WK - 1) / WK, s0 = part * stages, blocks = KB - 8 * s0;
  const int64_t a_base = MODE == kMxGateUp ? 0 : t.first, w_base = (int64_t)t.expert * p.wrows + n0;
  const int last = p.N - 1 - n0;
  // Row i of a stage (a's rows, then w's) behind the operand's base, and the offsets of its codes (in 16 bytes) and
  // of its scales (32 bits hold them: checked on the host)
  auto row_of = [&](int i) -> uint32_t {
    if (i < BM) return (uint32_t)(mx_a_row<MODE>(p, t, i) - a_base);
    const int j = i - BM;
    if constexpr (MODE == kMxGateUp) return (uint32_t)(min(j < COLS ? j : j - COLS, last) + (j < COLS ? 0 : p.N));
    else return (uint32_t)min(j, last);
  };
  auto code_offset = [&](int i) -> uint32_t { return row_of(i) * (uint32_t)KB; };
  auto scale_offset = [&](int i) -> uint32_t { return row_of(i) * (uint32_t)(i < BM ? p.as_ld : KB); };
  auto rsrc = [&](const uint8_t* base, int64_t bytes) {
    const uint64_t u = (uint64_t)(uintptr_t)base;
    return u32x4{(uint32_t)u, (uint32_t)(u >> 32) & 0xFFFFu, bytes < 0xFFFFFFF0LL ? (uint32_t)bytes : 0xFFFFFFF0u, 0x00020000u};
  };
  const int64_t a_rows = p.a_rows - a_base, w_blocks = (p.wrows - n0) * KB;
  const u32x4 ars = rsrc(p.a + a_base * KB * 16, a_rows * KB * 16), wrs = rsrc(p.w + w_base * KB * 16, w_blocks * 16);
  // scales from the word that holds the operand's first one, to the end of the word of its last
  const uint8_t *as = p.as + a_base * p.as_ld, *ws = p.ws + w_base * KB;
  const uint32_t a_in = (uint32_t)(uintptr_t)as & 3u, w_in = (uint32_t)(uintptr_t)ws & 3u;
  const u32x4 asrs = rsrc(as - a_in, ((a_rows - 1) * p.as_ld + KB + a_in + 3) & ~(int64_t)3), wsrs = rsrc(ws - w_in, (w_blocks + w_in + 3) & ~(int64_t)3);

  // this wave's loads of a stage: LOADS of 8 rows, the first A_LOADS of them a's; of a group of scales: those
  // of 64 rows, in SLOADS loads (the last one not of every wave)
  constexpr int LOADS = ROWS / (8 * WAVES), A_LOADS = BM / (8 * WAVES), SLOADS = (ROWS + 64 * WAVES - 1) / (64 * WAVES);
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && BM % 64 == 0 && BN % 64 == 0, "whole loads");
  uint32_t src[LOADS], ssrc[SLOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u)
    src[u] = (code_offset((u * WAVES + wave) * 8 + (lane >> 3)) + (uint32_t)((lane & 7) ^ (lane >> 3))) * 16u;
#pragma unroll
  for (int u = 0; u < SLOADS; ++u) {
    const int i = min((u * WAVES + wave) * 64 + lane, ROWS - 1);
    ssrc[u] = (scale_offset(i) + (i < BM ? a_in : w_in)) & ~3u;
  }
  constexpr uint32_t SHARE_LDS = mx_tile_lds(ROWS, NBUF, TM > TN ? TM : TN);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + part * SHARE_LDS;
  constexpr uint32_t SCALES = NBUF * STAGE, ZEROS = SCALES + NBUF * ROWS * 16;
  auto load_code = [&](int s, int u) {
    lds_dma16(u < A_LOADS ? ars : wrs, lds0 + (uint32_t)((s & (NBUF - 1)) * STAGE + (u * WAVES + wave) * 1024), src[u], (uint32_t)(s0 + s) * 128u);
  };
  auto load_scales = [&](int g) {
#pragma unroll
    for (int u = 0; u < SLOADS; ++u) {
      const int at = u * WAVES + wave;
      if (ROWS % (64 * WAVES) != 0 && at * 64 >= ROWS) continue;
      lds_dma16(at * 64 < BM ? asrs : wsrs, lds0 + SCALES + (uint32_t)((g & (NBUF - 1)) * ROWS * 16 + at * 1024), ssrc[u], (uint32_t)(s0 * 8 + g * 16));
    }
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // where this lane reads its fragments (16 rows on: 2048 bytes) and their scales (256 bytes)
  const int m0 = (wave / WN) * TM * 16, c0 = BM + (wave % WN) * TN * 16;
  uint32_t rd_a[2], rd_b[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t chunk = (uint32_t)((4 * h + q) ^ (r & 7)) * 16u;
    rd_a[h] = lds0 + (uint32_t)(m0 + r) * 128u + chunk;
    rd_b[h] = lds0 + (uint32_t)(c0 + r) * 128u + chunk;
  }
  // the rows of a fragment's next 16 are a multiple of 16 bytes on, and those of a gathered operand whole words: a
  // lane's scale bytes start alike in all its row tiles
  const uint32_t sh_a = ((MODE == kMxGateUp ? 0u : (uint32_t)r * (uint32_t)p.as_ld) + a_in & 3u) + (uint32_t)q;
  const uint32_t sh_b = (scale_offset(c0 + r) + w_in & 3u) + (uint32_t)q;
  // address of the scale of block q of half h of stage s
  auto scale_at = [&](int s, int h, uint32_t row, uint32_t sh) -> uint32_t {
    const uint32_t at = sh + (uint32_t)(8 * (s & 1) + 4 * h);  // byte in the group of 16
    const uint32_t group = (uint32_t)(s >> 1) + (at >> 4);
    uint32_t place = lds0 + SCALES + (group & (NBUF - 1)) * (ROWS * 16) + row * 16u + (at & 15u);
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
    a[i] = lds_read16(rd_a[h] + (uint32_t)(s & (NBUF - 1)) * STAGE + i * 2048);
    sa[i] = lds_read1(scales + i * 256);
  };
  auto read_cols = [&](int s, int h, Cols& c) {
    const uint32_t at = scale_at(s, h, (uint32_t)(c0 + r), sh_b);
#pragma unroll
    for (int j = 0; j < TN; ++j) c.b[j] = lds_read16(rd_b[h] + (uint32_t)(s & (NBUF - 1)) * STAGE + j * 2048);
#pragma unroll
    for (int j = 0; j < TN; ++j) c.s[j] = lds_read1(at + j * 256);
  };
  Cols first, second;
  auto products = [&](int i, const Cols& now) {
#pragma unroll
    for (int j = 0; j < TN; j += 2) mfma2(acc[i][j], acc[i][j + 1], now.b[j], now.b[j + 1], a[i], now.s[j], now.s[j + 1], sa[i]);
  };
  // a's fragments have one place: each is read again, for the next half, as soon as its products are under way

  load_scales(0);
#pragma unroll
  for (int s = 0; s < NBUF; ++s) {
    if (s >= stages) break;
    if (s & 1) load_scales((s + 1) >> 1);  // before the codes of the first stage that reads from it
#pragma unroll
    for (int u = 0; u < LOADS; ++u) load_code(s, u);
  }
  for (int i = ptid; i < (TM > TN ? TM : TN) * 64; i += WAVES * 64) ((uint32_t*)(lds + part * SHARE_LDS + ZEROS))[i] = 0u;
  if (stages >= NBUF) wait_loads_and_sync<(NBUF - 1) * LOADS>();
  else wait_loads_and_sync<0>();
  {
    const uint32_t at = scale_at(0, 0, (uint32_t)(m0 + r), sh_a);
    read_cols(0, 0, first);
#pragma unroll
    for (int i = 0; i < TM; ++i) read_a(0, 0, at, i);
  }
  // a wave whose rows all lie behind the tile's last only loads (an expert's last tile is half empty on average)
  const bool idle = MODE != kMxDense && m0 >= t.rows;
  for (int s = 0; idle && s < stages; ++s) {
    if (s + NBUF - 1 < stages) wait_loads_and_sync<(NBUF - 2) * LOADS>();
    else wait_loads_and_sync<0>();
    if (s + NBUF < stages) {
      if (s & 1) load_scales((s + NBUF + 1) >> 1);
#pragma unroll
      for (int u = 0; u < LOADS; ++u) load_code(s + NBUF, u);
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
    // products: by then the reads that it waits for have come back.  The loads of stage s + NBUF go out between the
    // products.  (After the last stage the fragments are of nothing, and nobody uses them.)
    constexpr int SHARE = (LOADS + TM - 1) / TM;
    const uint32_t at = scale_at(s + 1, 0, (uint32_t)(m0 + r), sh_a);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      products(i, second);
      if (i == 0) {
        // stage s + 1 is there, stage s has been read
        if (s + NBUF - 1 < stages) wait_loads_and_sync<(NBUF - 2) * LOADS>();
        else wait_loads_and_sync<0>();
        read_cols(s + 1, 0, first);
        if ((s & 1) && s + NBUF < stages) load_scales((s + NBUF + 1) >> 1);
      }
      read_a(s + 1, 0, at, i);
      if (s + NBUF < stages) {
#pragma unroll
        for (int u = i * SHARE; u < (i + 1) * SHARE && u < LOADS; ++u) load_code(s + NBUF, u);
      }
    }
  }
  // no use of an accumulator before the last product is through
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[i][j]));
  __syncthreads();

  if constexpr (WK > 1) {
    // the shares' sums meet in LDS, in order: [share - 1][accumulator][thread]
    constexpr int N4 = TM * TN, THREADS = WAVES * 64;
    static_assert((WK - 1) * N4 * THREADS * 16 <= WK * SHARE_LDS, "the shares' sums");
    f32x4* sums = (f32x4*)lds;
    if (part > 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) sums[((part - 1) * N4 + i * TN + j) * THREADS + ptid] = acc[i][j];
    }
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int k = 0; k < WK - 1; ++k)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] += sums[(k * N4 + i * TN + j) * THREADS + ptid];
    }
    __syncthreads();
    if (part > 0) return;  // no barrier follows but the gated one, which has no shares
    static_assert(MODE != kMxGateUp, "");
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
              v[4 * d + e] = mx_gated(acc[i][j + d][e], u[e], p.act);
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
    // through LDS, as below, in fp32
    constexpr int LD = TN * 64 + 16, LANES = TN * 4;  // bytes of a row; lanes of 16 bytes to it
    static_assert(WAVES * TM * 16 * LD <= mx_tile_lds(ROWS, NBUF, TM > TN ? TM : TN), "the output tile");
    uint8_t* mine = lds + wave * (TM * 16 * LD);
    const int nw = n0 + c0 - BM, n = nw + lane % LANES * 4;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) *(f32x4*)(mine + (16 * i + r) * LD + 64 * j + 16 * q) = acc[i][j];
    const int rows = min(TM * 16, t.rows - m0);
    if (n < p.N)
      for (int m = lane / LANES; m < rows; m += 64 / LANES)
        *(f32x4*)(p.y + (int64_t)p.order[t.first + m0 + m] * p.N + n) = *(const f32x4*)(mine + m * LD + lane % LANES * 16);
  } else {
    // through LDS, a region of each wave's own: rows of whole lines instead of 8 bytes in 16 rows at a time
    // (M = 4096, N = 24576: 140 us of 412 before)
    constexpr int LD = TN * 32 + 16;  // bytes of a row, and 16 so that the rows of a store lie in different banks
    static_assert(WAVES * TM * 16 * LD <= mx_tile_lds(ROWS, NBUF, TM > TN ? TM : TN), "the output tile");
    uint8_t* mine = lds + wave * (TM * 16 * LD);
    const int nw = n0 + c0 - BM;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = nw + 16 * j + 4 * q + e;
        bias[e] = n < p.N ? load_bias(p.bias, p.bias_dtype, n) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const f32x4 v = {acc[i][j][0] + bias[0], acc[i][j][1] + bias[1], acc[i][j][2] + bias[2], acc[i][j][3] + bias[3]};
        *(u32x2*)(mine + (16 * i + r) * LD + 32 * j + 8 * q) =
            p.out_bf16 ? u32x2{pack2<bf16>(v[0], v[1]), pack2<bf16>(v[2], v[3])} : u32x2{pack2<f16>(v[0], v[1]), pack2<f16>(v[2], v[3])};
      }
    }
    const int rows = min(TM * 16, t.rows - m0);
    uint16_t* out = p.c + (int64_t)(t.first + m0) * p.ldc + nw;
    if ((p.ldc & 7) == 0 && ((uintptr_t)p.c & 15) == 0 && nw + TN * 16 <= p.N) {
      constexpr int LANES = TN * 2;  // of 16 bytes, to a row
      for (int m = lane / LANES; m < rows; m += 64 / LANES)
        *(u32x4*)(out + (int64_t)m * p.ldc + lane % LANES * 8) = *(const u32x4*)(mine + m * LD + lane % LANES * 16);
    } else {
      constexpr int LANES = TN * 16 < 64 ? TN * 16 : 64;
      for (int m = lane / LANES; m < rows; m += 64 / LANES)
        for (int n = lane % LANES; n < TN * 16 && nw + n < p.N; n += LANES) out[(int64_t)m * p.ldc + n] = *(const uint16_t*)(mine + m * LD + 2 * n);
    }
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

template <int MODE, int BM, int BN, int WM, int WN, int PER_SIMD, int NBUF, int WK = 1>
static int launch_tile(const MxArgs& p, int64_t row_tiles, hipStream_t st) {
  constexpr int COLS = MODE == kMxGateUp ? BN / 2 : BN;
  const int64_t col_tiles = cdiv(p.N, COLS);
  if (row_tiles * col_tiles > 0x7FFFFFFLL) return AWQ_ERR_UNSUPPORTED;
  constexpr int lds = WK * mx_tile_lds(BM + BN, NBUF, BM / WM > BN / WN ? BM / WM / 16 : BN / WN / 16);
  static_assert(MODE != kMxGateUp || BM * (BN / 2 + 4) * 4 <= lds, "the up half");
  auto kernel = mx_tile_kernel<MODE, BM, BN, WM, WN, PER_SIMD, NBUF, WK>;
  if (lds > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    (void)hipGetLastError();
    return AWQ_ERR_LAUNCH;
  }
  kernel<<<dim3((unsigned)(cdiv(row_tiles * col_tiles, 8) * 8)), dim3(WM * WN * WK * 64), lds, st>>>(p, (int)row_tiles, (int)col_tiles);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

// Tiles of 256 x 256 run in rounds of one a CU, those of 128 x 128 two a CU, whose rounds run into each other: K = 4096, us
// with one and the other: M = 2048, N = 24576 121, 146; M = 3000, N = 5000 44, 54; M = 2048, N = 6144 41, 43; M = 1000,
// N = 24576 77, 78; M = 700, N = 4096 31, 17: about 38 a round against 26 for 512 tiles.  Fewer than 192 of them: tiles
// of 64 x 64 (M = 512, N = 4096 13 against 15; M = 1024 22 against 19).  Up to a tile per CU of these
// K goes in shares: two from 8 stages on, four from 24 on (M = 64, N = 4096, us with 1, 2, 4: K = 1024 5.1, 5.2, 6.1;
// K = 4096 9.4, 8.2, 8.6; K = 12288 22.7, 18.2, 15.6; with 316 tiles, M = 200, N = 5001, K = 4128 14.2, 15.3, 22.2).
int launch_mx_tile_gemm(const MxArgs& p, hipStream_t st) {
  const int64_t big = cdiv(p.M, 256) * cdiv(p.N, 256), mid = cdiv(p.M, 128) * cdiv(p.N, 128);
  if (512 * 38 * cdiv(big, 256) <= 26 * std::max<int64_t>(512, mid)) return launch_tile<kMxDense, 256, 256, 2, 4, 2, 2>(p, cdiv(p.M, 256), st);
  if (mid >= 192) return launch_tile<kMxDense, 128, 128, 2, 4, 4, 2>(p, cdiv(p.M, 128), st);
  const int64_t rows = cdiv(p.M, 64), tiles = rows * cdiv(p.N, 64), stages = cdiv(p.K, 256);
  if (tiles <= 256 && stages >= 24) return launch_tile<kMxDense, 64, 64, 2, 2, 4, 2, 4>(p, rows, st);
  if (tiles <= 256 && stages >= 8) return launch_tile<kMxDense, 64, 64, 2, 2, 4, 2, 2>(p, rows, st);
  return launch_tile<kMxDense, 64, 64, 2, 2, 4, 2>(p, rows, st);
}

int launch_mx_tile_grouped(const MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st) {
  if (rows == 128)
    return gate_up ? launch_tile<kMxGateUp, 128, 128, 2, 4, 4, 2>(p, row_tiles, st) : launch_tile<kMxDown, 128, 128, 2, 4, 4, 2>(p, row_tiles, st);
  return gate_up ? launch_tile<kMxGateUp, 64, 128, 2, 2, 2, 2>(p, row_tiles, st) : launch_tile<kMxDown, 64, 128, 2, 2, 2, 2>(p, row_tiles, st);
}

}  // namespace awq_host
