// Walks every direct load of the MXFP4 tile kernel's blocks on the host, with the kernel's own address arithmetic
// (csrc/awq_mx_span.h), and checks that a load touches nothing outside its operand and finds what it is for.
// Scales are loaded by words: the words of the operand's first and last byte count as its own.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "awq_mx_span.h"

namespace {
using namespace awq;

// words of a descriptor: where an operand begins, and its bytes
struct Rsrc {
  uint64_t base;
  uint32_t bytes;
};
struct Operand {
  uint64_t lo, hi;
};
enum Mode { kDense, kGateUp, kDown };
struct Case {
  Mode mode;
  int BM, BN, WK, KB, rows, a_rows, N, n0;  // rows: of the tile; a_rows: of a, where they are gathered
  uint32_t in;                              // the scales' first byte in its word
  bool scalar;                              // whether whole stages have their position in the scalar offset
};
long walked = 0;

void fail(const Case& c, const char* what, int part, int stage, int row) {
  std::printf("%s: mode %d tile %dx%d shares %d KB %d rows %d a_rows %d N %d n0 %d in %u: share %d, stage or group %d, row %d\n", what, c.mode,
              c.BM, c.BN, c.WK, c.KB, c.rows, c.a_rows, c.N, c.n0, c.in, part, stage, row);
  std::exit(1);
}
// A 16-byte load: every dword that the range check lets through is the operand's, whether or not the check counts the SGPR
// offset (leaving it out lets more through).
void touch(const Case& c, const Rsrc& rs, uint32_t voff, uint32_t soff, const Operand& o, int part, int stage, int row) {
  for (uint32_t d = 0; d < 16; d += 4) {
    if ((uint64_t)voff + d + 4 > rs.bytes) continue;
    const uint64_t at = rs.base + voff + soff + d;
    if (at < (o.lo & ~(uint64_t)3) || at + 4 > ((o.hi + 3) & ~(uint64_t)3)) fail(c, "outside the operand", part, stage, row);
  }
  ++walked;
}

void walk(const Case& c) {
  const bool gate_up = c.mode == kGateUp;
  const int KB = c.KB, ROWS = c.BM + c.BN, last = c.N - 1 - c.n0;
  const uint32_t a_ld = gate_up ? (uint32_t)(KB + 3) / 4 * 4 : (uint32_t)KB;
  const uint32_t a_rows = (uint32_t)(gate_up ? c.a_rows : c.rows), w_rows = mx_w_rows(gate_up, c.BN, last, c.N);
  const uint32_t w_left = (uint32_t)((gate_up ? 2 : 1) * c.N - c.n0);  // of the expert, from n0 on
  const uint64_t a0 = 0x3FFFFFFF0ull, w0 = 0x4FFFFFFE0ull, as0 = 0x1FFFFFFFCull + (gate_up ? 0 : c.in), ws0 = 0x2FFFFFFF8ull + c.in;
  const Operand oa{a0, a0 + (uint64_t)a_rows * KB * 16}, ow{w0, w0 + (uint64_t)w_left * KB * 16};
  const Operand osa{as0, as0 + (uint64_t)(a_rows - 1) * a_ld + KB}, osw{ws0, ws0 + (uint64_t)w_left * KB};
  const int stages = ((KB + 7) / 8 + c.WK - 1) / c.WK;
  auto row_of = [&](int i) -> uint32_t {
    if (i >= c.BM) return mx_w_row(gate_up, i - c.BM, last, c.N);
    const int r = i < c.rows ? i : c.rows - 1;
    return (uint32_t)(gate_up ? (c.a_rows - 1 - r * 7 % c.a_rows) : r);
  };
  for (int part = 0; part < c.WK; ++part) {
    const int s0 = part * stages;
    const uint32_t a_in = (uint32_t)as0 & 3u, w_in = (uint32_t)ws0 & 3u;
    const int whole = c.scalar ? mx_whole_stages(KB, s0, stages) : 0;
    const Rsrc ars{a0, mx_code_bytes(a_rows, KB)}, wrs{w0, mx_code_bytes(w_rows, KB)};
    const Rsrc asrs{as0 - a_in, mx_scale_bytes(a_rows, a_ld, KB, a_in)}, wsrs{ws0 - w_in, mx_scale_bytes(w_rows, KB, KB, w_in)};
    auto codes = [&](int s) {
      for (int i = 0; i < ROWS; ++i)
        for (int l = 8 * (i & 7); l < 8 * (i & 7) + 8; ++l) {
          const bool a = i < c.BM;
          const Rsrc& rs = a ? ars : wrs;
          const uint32_t row = row_of(i), src = mx_code_offset(row, KB, l), position = mx_code_position(s0 + s);
          const uint32_t voff = s < whole ? src : src + position, soff = s < whole ? position : 0u;
          touch(c, rs, voff, soff, a ? oa : ow, part, s, i);
          const int block = 8 * (s0 + s) + ((l & 7) ^ (l >> 3));
          if (block < KB && ((uint64_t)voff + soff + 16 > rs.bytes || rs.base + voff + soff != (a ? a0 : w0) + ((uint64_t)row * KB + block) * 16))
            fail(c, "not its codes", part, s, i);
        }
    };
    auto scales = [&](int g) {
      for (int i = 0; i < ROWS; ++i) {
        const bool a = i < c.BM;
        const Rsrc& rs = a ? asrs : wsrs;
        const uint32_t row = row_of(i), off = mx_scale_offset(row, a ? a_ld : KB, a ? a_in : w_in) + mx_scale_position(s0, g);
        touch(c, rs, off, 0, a ? osa : osw, part, g, i);
        // the row's bytes of this share that lie in the group
        const uint64_t mine = (a ? as0 + (uint64_t)row * a_ld : ws0 + (uint64_t)row * KB) + 8 * s0, from = rs.base + off;
        for (uint64_t b = mine; b < mine + 8 * stages && b < mine + (uint64_t)(KB - 8 * s0 > 0 ? KB - 8 * s0 : 0); ++b) {
          if (b < from || b >= from + 16) continue;
          if ((uint64_t)off + ((b - from) & ~(uint64_t)3) + 4 > rs.bytes) fail(c, "not its scales", part, g, i);
        }
        if (from != (mine & ~(uint64_t)3) + 16 * (uint64_t)g) fail(c, "not its group", part, g, i);
      }
    };
    // as the kernel issues them
    scales(0);
    for (int s = 0; s < 2 && s < stages; ++s) {
      if (s & 1) scales(1);
      codes(s);
    }
    for (int s = 0; s + 2 < stages; ++s) {
      if (s & 1) scales((s + 3) >> 1);
      codes(s + 2);
    }
  }
}
}  // namespace

int main() {
  const int tiles[][4] = {{kDense, 256, 256, 1}, {kDense, 128, 128, 1}, {kDense, 64, 64, 1}, {kDense, 64, 64, 2}, {kDense, 64, 64, 4},
                          {kGateUp, 64, 128, 1}, {kGateUp, 128, 128, 1}, {kDown, 64, 128, 1}, {kDown, 128, 128, 1}};
  for (const auto& t : tiles)
    for (int KB : {1, 3, 7, 8, 9, 16, 31, 129})
      for (int rows : {1, 6, t[1] - 1, t[1]})
        for (int N : {1, 32, 64, 200, 1000}) {
          if (t[0] == kGateUp && N % 32) continue;
          const int cols = t[0] == kGateUp ? t[2] / 2 : t[2], n0 = (N - 1) / cols * cols;  // the last column tile, and the first
          for (int first : {0, n0})
            for (uint32_t in = 0; in < 4; ++in)
              for (bool scalar : {false, true}) walk({(Mode)t[0], t[1], t[2], t[3], KB, rows, rows < 9 ? 1 : 90, N, first, in, scalar});
        }
  std::printf("%ld loads\n", walked);
  return 0;
}
