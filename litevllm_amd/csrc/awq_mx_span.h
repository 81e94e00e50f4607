// What the direct loads of the microscaled tile kernel read (awq_mx_tile.hip): plain C++, so that a host program can walk
// every address (tests/mx_span_walk.cpp).
//
// The range check covers the VGPR offset, per dword of a load; whether the SGPR offset counts is documented as no, and
// measured as yes on gfx950.  So a stage's position along K may be in the SGPR offset only where all of the stage lies inside
// K, and no load of it leaves its row; the stages that pass K's end have it in the VGPR offset, and so have all scales, and
// the check ends them with the operand.
#pragma once

#include <cstdint>

namespace awq {

// Of the `stages` stages of 8 blocks from block 8 s0 on, those that lie inside K.
constexpr int mx_whole_stages(int KB, int s0, int stages) {
  const int whole = KB / 8 - s0;
  return whole < 0 ? 0 : (whole < stages ? whole : stages);
}
constexpr uint32_t mx_code_position(int s) { return (uint32_t)s * 128u; }
constexpr uint32_t mx_scale_position(int s0, int group) { return (uint32_t)(s0 * 8 + group * 16); }

// Rows of w of a tile from its first on: the last one read, and how many that spans.  gate_up: row j of the tile's BN is a
// gate column's (the first 32 of 64) or its up column's, N rows on.
constexpr uint32_t mx_w_row(bool gate_up, int j, int last, int N) {
  if (!gate_up) return (uint32_t)(j < last ? j : last);
  const int c = j / 64 * 32 + j % 32;
  return (uint32_t)((c < last ? c : last) + (j % 64 < 32 ? 0 : N));
}
constexpr uint32_t mx_w_rows(bool gate_up, int BN, int last, int N) { return mx_w_row(gate_up, BN - 1, last, N) + 1u; }

// Codes: KB blocks of 16 bytes a row.  Lane l of a wave's load of eight rows reads chunk (l & 7) ^ (l >> 3) of a line.
// 32 bits hold them, and the positions behind K's end with them: checked on the host.
constexpr uint32_t mx_code_bytes(uint32_t rows, uint32_t KB) { return rows * KB * 16u; }
constexpr uint32_t mx_code_offset(uint32_t row, uint32_t KB, int lane) {
  return (row * KB + (uint32_t)((lane & 7) ^ (lane >> 3))) * 16u;
}

// Scales: KB bytes a row, `ld` from row to row, the first `in` bytes behind a word's start; loads start at words and end
// with the word of the last byte.
constexpr uint32_t mx_scale_bytes(uint32_t rows, uint32_t ld, uint32_t KB, uint32_t in) {
  return ((rows - 1u) * ld + KB + in + 3u) & ~3u;
}
constexpr uint32_t mx_scale_offset(uint32_t row, uint32_t ld, uint32_t in) { return (row * ld + in) & ~3u; }

}  // namespace awq
