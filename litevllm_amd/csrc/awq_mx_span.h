// What the direct loads of the microscaled tile kernel read (awq_mx_tile.hip): plain C++, so that a host program can walk
// every address (tests/mx_span_walk.cpp).
//
// A load's position along K is part of its descriptor's base, and what is left of the operand behind it is the
// descriptor's size: the range check, per dword of a load, then ends every load at the operand's end, whether or not it
// counts the SGPR offset (gfx950 does; it is documented as left out).
#pragma once

#include <cstdint>

namespace awq {

// Words 0 .. 2 of a buffer descriptor: 48 bits of address, and the bytes behind it that may be read.
template <typename Rsrc>
constexpr void mx_span_set(Rsrc& rs, uint64_t base, uint32_t bytes) {
  rs[0] = (uint32_t)base;
  rs[1] = (uint32_t)(base >> 32) & 0xFFFFu;
  rs[2] = bytes;
}
#ifdef __HIPCC__
#define AWQ_SPAN_FN __host__ __device__ __forceinline__
#else
#define AWQ_SPAN_FN inline
#endif
template <typename Rsrc>
AWQ_SPAN_FN void mx_span_advance(Rsrc& rs, uint32_t by) {
  const uint32_t lo = rs[0] + by;
  rs[1] += lo < by ? 1u : 0u;
  rs[0] = lo;
  uint32_t left = rs[2] > by ? rs[2] : by;
#ifdef __HIP_DEVICE_COMPILE__
  asm("" : "+s"(left));  // a maximum and a difference in scalar registers, no saturating subtraction, which only vectors have
#endif
  rs[2] = left - by;
}

// Rows of w of a tile from its first on: the last one read, and how many that spans.  gate_up: row j of the tile's BN is a
// gate column's (the first 32 of 64) or its up column's, N rows on.
constexpr uint32_t mx_w_row(bool gate_up, int j, int last, int N) {
  if (!gate_up) return (uint32_t)(j < last ? j : last);
  const int c = j / 64 * 32 + j % 32;
  return (uint32_t)((c < last ? c : last) + (j % 64 < 32 ? 0 : N));
}
constexpr uint32_t mx_w_rows(bool gate_up, int BN, int last, int N) { return mx_w_row(gate_up, BN - 1, last, N) + 1u; }

// Codes: KB blocks of 16 bytes a row.  Lane l of a wave's load of eight rows reads chunk (l & 7) ^ (l >> 3) of a line.
// 32 bits hold them: checked on the host.
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
