// sx_kv8_units.h -- which 16-token block of which sequence a CTA of the paged 8-bit append takes.
// Integers only and no CUDA, so the same code runs under a host compiler (tests/test_kv8_units_cpu.py).
//
// Sequence b has rows [row_start[b], row_start[b + 1]), the last tokens of its kv_len[b].  Unit u of a
// call is a block that holds new tokens: those of sequence b are kv8_unit_base(b) + 0, 1, ..., one per
// block, and u belongs to the last sequence whose base is at most u.  n rows touch at most n / 16 + 2
// blocks, so while row_start rises the bases of two sequences are never closer than the blocks of the
// first, and kv8_unit_count units hold them all: the grid follows from the row and sequence counts alone.
// Units between a sequence's last block and the next base, and those below the first base (rows before
// row_start[0] belong to nobody), are empty.  Where row_start falls a unit may be given to the wrong
// sequence, or lie below the base of the one it is given to; it is then one of that sequence's own
// blocks, or empty.
#pragma once

#include <stdint.h>

#ifndef SX_HD
#define SX_HD inline
#endif

namespace sx {

constexpr int kKv8Block = 16;  // tokens per record

// Rows of a sequence: [r0, r0 + n), its length with them.
struct Kv8Rows {
  uint32_t r0, n, len;
};

// False when the rows or the length do not fit (include/sx.h: the sequence is skipped).
SX_HD bool kv8_rows_fit(uint32_t r0, uint32_t r1, uint32_t len, uint32_t tokens, uint32_t max_len, Kv8Rows *r) {
  r->r0 = r0;
  r->n = r1 - r0;
  r->len = len;
  return r0 <= r1 && r1 <= tokens && r->n <= len && len <= max_len;
}

SX_HD uint32_t kv8_unit_base(uint32_t row_start, uint32_t b) { return row_start / kKv8Block + 2 * b; }
SX_HD uint32_t kv8_unit_count(uint32_t tokens, uint32_t seqs) { return tokens / kKv8Block + 2 * seqs; }

// One 16-token block of one sequence.
struct Kv8Unit {
  uint32_t block;         // of the sequence
  uint32_t row0, cnt, t0; // its new rows, how many, the first one's place in the block
};

// Block `rel` of those that rows of r touch; false when there is none, as for a rel below 0 (2^31 and on).
SX_HD bool kv8_unit(const Kv8Rows &r, uint32_t rel, Kv8Unit *u) {
  const uint32_t pos0 = r.len - r.n;  // position of the first new row
  const uint32_t first = pos0 / kKv8Block;
  if (r.n == 0 || rel > (r.len - 1) / kKv8Block - first) return false;
  u->block = first + rel;
  const uint32_t at = u->block * kKv8Block;
  const uint32_t lo = pos0 > at ? pos0 : at, hi = r.len - at > (uint32_t)kKv8Block ? at + kKv8Block : r.len;
  u->row0 = r.r0 + (lo - pos0);
  u->cnt = hi - lo;
  u->t0 = lo - at;
  return true;
}

}  // namespace sx
