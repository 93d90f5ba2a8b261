// paged_plan_check.cpp - host check of the paged cache's index arithmetic (csrc/fa_paged_plan.h compiled with g++).
//
// Walks the loops of paged_attn_kernel and paged_join_kernel (fa_paged_attn.hip) over many batches and checks that
//   * visible_key counts through exactly the keys that the mask allows, in ascending order,
//   * every unit of every sequence belongs to exactly one workgroup's run, and runs stay inside the batch,
//   * the pieces that are no whole sequence have slots of their own, inside the workspace, and the join looks for
//     exactly those,
//   * page_of(n) = n / page_size.
// Prints "OK <cases>" or the first failing case; exit status 0 on success.
#define FA_HOST_ONLY 1
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>

#include "../flashattention-gpt-oss-finetuning_amd/csrc/fa_paged_plan.h"

using namespace fa;

static int fails(const char* what, int a, int b, int c, int d) {
  std::printf("FAIL %s %d %d %d %d\n", what, a, b, c, d);
  return 1;
}

static int check_visible(int n, int W, int S) {
  const Visible r = visible(n, W, S);
  int v = 0;
  for (int k = 0; k < n; ++k)
    if (n - 1 - k < W || k < S) {
      if (v >= r.count || visible_key(r, v) != k) return fails("visible", n, W, S, k);
      ++v;
    }
  return v == r.count ? 0 : fails("count", n, W, S, v);
}

static int check_split(const std::vector<int>& counts, int parts, int least) {
  const int B = int(counts.size());
  std::vector<int> start(B + 1, 0);
  for (int b = 0; b < B; ++b) start[b + 1] = start[b] + paged_units(counts[b]);
  const int total = start[B], per = units_per_part(total, parts, least);
  std::vector<std::vector<int>> seen(B);
  for (int b = 0; b < B; ++b) seen[b].assign(paged_units(counts[b]), 0);
  std::map<int, std::pair<int, int>> slots;  // slot -> (sequence, part)
  for (int part = 0; part < parts; ++part) {
    if (int64_t(part) * per >= total) continue;
    int u = part * per;
    const int end = imin(total, u + per);
    int b = 0;
    while (!(start[b + 1] > u)) ++b;  // find_unit: the first sequence whose units reach past u
    while (u < end) {
      if (b >= B) return fails("run past the batch", part, u, end, per);
      const int stop = imin(end, start[b + 1]);
      const bool whole = u == start[b] && stop == start[b + 1];
      for (int x = u; x < stop; ++x) ++seen[b][x - start[b]];
      if (!whole) {
        const int slot = part_slot(part, per, start[b]);
        if (slot < 0 || slot >= 2 * parts || slots.count(slot)) return fails("slot", slot, part, b, per);
        slots[slot] = {b, part};
      }
      u = stop;
      ++b;
    }
  }
  std::set<int> joined;
  for (int b = 0; b < B; ++b) {
    for (int x : seen[b])
      if (x != 1) return fails("unit", b, x, parts, per);
    const int first = start[b] / per, last = (start[b + 1] - 1) / per;
    if (first == last) continue;
    for (int p = first; p <= last; ++p) {
      const int slot = part_slot(p, per, start[b]);
      if (!slots.count(slot) || slots[slot] != std::make_pair(b, p) || !joined.insert(slot).second) return fails("join", b, p, slot, per);
    }
  }
  return joined.size() == slots.size() ? 0 : fails("slots not joined", int(joined.size()), int(slots.size()), parts, per);
}

int main() {
  long cases = 0;
  for (int n = 0; n <= 40; ++n)
    for (int W = 0; W <= 42; ++W)
      for (int S = W ? 0 : 1; S <= 42; S += 1 + S / 4) {
        if (check_visible(n, W, S)) return 1;
        ++cases;
      }
  unsigned seed = 1;
  auto rnd = [&](int n) { return int((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
  for (int i = 0; i < 20000; ++i) {
    std::vector<int> counts(1 + rnd(i % 3 ? 6 : 150));
    for (int& c : counts) c = rnd(4) ? rnd(1 << rnd(14)) : rnd(3) * kPagedUnit;
    if (check_split(counts, 1 + rnd(i % 2 ? 9 : 130), 1 + rnd(4))) return 1;
    ++cases;
  }
  for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 16u, 24u, 33u, 64u, 100u, 255u, 256u, 257u, 4096u, 65535u, 1000003u, (1u << 30) - 1}) {
    const PageDiv m = page_div(d);
    auto bad = [&](uint32_t n) { return n < (1u << 31) && uint32_t(page_of(m, int(n))) != n / d; };
    for (int i = 0; i < 20000; ++i) {
      const uint32_t n = uint32_t(rnd(1 << 16)) << 15 | uint32_t(rnd(1 << 15)), near = n / d * d;
      if (bad(n) || bad(near) || (near && bad(near - 1)) || bad(uint32_t(i)) || bad((1u << 31) - 1 - uint32_t(i))) return fails("page_of", int(d), int(n), 0, 0);
    }
    ++cases;
  }
  std::printf("OK %ld\n", cases);
  return 0;
}
