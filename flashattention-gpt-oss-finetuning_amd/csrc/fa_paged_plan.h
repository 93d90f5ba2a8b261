// fa_paged_plan.h - index arithmetic of the paged key-value cache's kernels: which keys the query of a sequence
// sees, how the work is cut into pieces and which page a key lies on.
//
// Shared by the kernels (device) and the host: fa_paged.cpp sizes the workspace with it, and
// tests/paged_plan_check.cpp compiles it with g++ (FA_HOST_ONLY) to check that every visible key belongs to exactly
// one piece and that no two pieces share a slot of the workspace.
#pragma once

#include <stdint.h>

#include "fa_plan.h"

namespace fa {

// Keys of a unit, the grain of a sequence's pieces: a tile of 32 keys for each of a workgroup's 4 waves.
constexpr int kPagedUnit = 128;
// Tokens of one sequence are fewer than this, so that positions and unit counts stay far from the ends of int32.
constexpr int64_t kPagedMaxTokens = int64_t(1) << 30;

// n / d for n < 2^31 as a product: with 2^(s-1) < d <= 2^s and mul = floor(2^(31+s) / d) + 1, mul d exceeds 2^(31+s) by
// at most d <= 2^s, so (n mul) / 2^(31+s) exceeds n / d by less than 1 / d.
struct PageDiv {
  uint32_t mul, shift;
};
inline PageDiv page_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return PageDiv{uint32_t((uint64_t(1) << (31 + s)) / d + 1), 31 + s};
}
FA_HD int page_of(PageDiv d, int n) { return int((uint64_t(uint32_t(n)) * d.mul) >> d.shift); }

// The keys that the query of a sequence of n tokens (its last one) sees: key k < n with n - 1 - k < W or k < S.  They
// are counted through: the v-th of them is key v for v < first, else v + gap.
struct Visible {
  int first, gap, count;
};
FA_HD Visible visible(int n, int W, int S) {
  const int lo = imax(0, n - W);
  Visible r;
  r.first = imin(S, lo);
  r.gap = lo - r.first;
  r.count = n - r.gap;
  return r;
}
FA_HD int visible_key(const Visible& r, int v) { return v < r.first ? v : v + r.gap; }

// Units of a sequence; one for a sequence without keys, whose outputs are written all the same.
FA_HD int paged_units(int count) { return imax(1, (count + kPagedUnit - 1) / kPagedUnit); }

// Split calls: the units of all sequences, one sequence after the other, are dealt out to `parts` workgroups in runs of
// `per` units.  A run holds pieces of its first and its last sequence at most that are not the whole sequence, so a
// workgroup needs two slots for partial results: slot 0 for the sequence in which its run begins, slot 1 for one
// that begins inside it.
FA_HD int units_per_part(int total, int parts, int least) { return imax(least, (total + parts - 1) / parts); }
FA_HD int part_slot(int part, int per, int seq_start) { return 2 * part + (seq_start > part * per ? 1 : 0); }

}  // namespace fa
