// paged_few_check.cpp - host check of split calls that use only the first `few` of the parts that their workspace has room
// for (csrc/fa_paged_plan.h compiled with g++, as tests/paged_plan_check.cpp).
//
// Walks the runs of paged_attn_kernel and the join of paged_finish_kernel (fa_paged_attn.hip) for grids of `parts` workgroups a
// stream whose runs are sized for `parts` or, where the call has at most many_units units, for `few`; slots lie 2 `parts`
// apart from stream to stream either way.  Checks that every unit belongs to one workgroup, that the pieces of all streams have
// slots of their own inside the workspace, and that the join reads exactly those.
// Prints "OK <cases>" or the first failing case; exit status 0 on success.
#define FA_HOST_ONLY 1
#include <cstdio>
#include <map>
#include <utility>
#include <vector>

#include "../flashattention-gpt-oss-finetuning_amd/csrc/fa_paged_plan.h"

using namespace fa;

static int fails(const char* what, int a, int b, int c, int d) {
  std::printf("FAIL %s %d %d %d %d\n", what, a, b, c, d);
  return 1;
}

static int check(const std::vector<int>& counts, int streams, int parts, int few, int many_units, int least) {
  const int B = int(counts.size());
  std::vector<int> start(B + 1, 0);
  for (int b = 0; b < B; ++b) start[b + 1] = start[b] + paged_units(counts[b]);
  const int total = start[B], used = total > many_units ? parts : few, per = units_per_part(total, used, least);
  std::map<int, std::pair<int, int>> slots;  // slot -> (sequence, part)
  for (int wg = 0; wg < streams * parts; ++wg) {
    const int stream = wg / parts, part = wg % parts;
    if (int64_t(part) * per >= total) continue;
    if (part >= used) return fails("a part that is not used has units", part, used, total, per);
    int b = 0, u = part * per;
    const int end = imin(total, u + per);
    while (start[b + 1] <= u) ++b;
    for (; u < end; ++b) {
      if (b >= B) return fails("run past the batch", part, u, end, per);
      const int stop = imin(end, start[b + 1]);
      if (u != start[b] || stop != start[b + 1]) {
        const int slot = 2 * parts * stream + part_slot(part, per, start[b]);
        if (slot < 0 || slot >= 2 * parts * streams || slots.count(slot)) return fails("slot", slot, part, b, per);
        slots[slot] = {b, part};
      }
      u = stop;
    }
  }
  size_t joined = 0;
  for (int stream = 0; stream < streams; ++stream)
    for (int b = 0; b < B; ++b) {
      const int first = imin(imax(start[b] / per, 0), parts - 1), last = imin((start[b + 1] - 1) / per, parts - 1);
      for (int p = first; first < last && p <= last; ++p, ++joined) {
        const auto s = slots.find(2 * parts * stream + part_slot(p, per, start[b]));
        if (s == slots.end() || s->second != std::make_pair(b, p)) return fails("join", b, p, first, last);
      }
    }
  return joined == slots.size() ? 0 : fails("slots not joined", int(joined), int(slots.size()), parts, few);
}

int main() {
  long cases = 0;
  unsigned seed = 7;
  auto rnd = [&](int n) { return int((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
  for (int i = 0; i < 20000; ++i) {
    std::vector<int> counts(1 + rnd(i % 3 ? 6 : 100));
    for (int& c : counts) c = rnd(4) ? rnd(1 << rnd(14)) : rnd(3) * kPagedUnit;
    int units = 0;
    for (int c : counts) units += paged_units(c);
    const int few = 8 * (1 + rnd(i % 2 ? 2 : 16)), border = units - 2 + rnd(4);
    if (check(counts, 1 + rnd(3), 2 * few, few, i % 4 ? border : rnd(1000), 1)) return 1;
    ++cases;
  }
  std::printf("OK %ld\n", cases);
  return 0;
}
