// Host-side check of rd::counted_rows() (gpu_ragged_dot_amd/csrc/rd_int4_rows.h), by which the kernels of the product on 4-bit weights sum
// up group sizes, 64 to a wave: over sizes of every kind - negative, zero, ordinary, at and beyond m, the largest 32-bit number -
// and for m up to the largest that a call takes,
//   - no sum on the way leaves 32 bits;
//   - every group's rows are those of 64-bit arithmetic: behind the groups before it, cut off at m.
// Built without GPU code by the library's Makefile; run by tests/test_int4_group_scan.py.
#include <limits.h>
#include <stdio.h>
#include <random>
#include <vector>
#include "rd_int4_rows.h"

static long long g_checked = 0;

static bool check(const std::vector<int>& sizes, int m) {
  long long exact = 0;  // rows before a group, not cut off
  int before = 0;       // as scan_groups() carries it from one 64 groups to the next
  for (size_t base = 0; base < sizes.size(); base += 64) {
    long long sum = 0;
    int first = before;
    for (int lane = 0; lane < 64; ++lane) {
      const int size = base + lane < sizes.size() ? sizes[base + lane] : 0;
      sum += rd::counted_rows(size, before, m);
      if (sum < 0 || before + sum > INT_MAX) {
        fprintf(stderr, "m=%d group %zu: a sum of %lld\n", m, base + lane, before + sum);
        return false;
      }
      const int end = rd::imin(before + (int)sum, m);
      const long long want_first = exact < m ? exact : m;
      exact += size > 0 ? size : 0;
      const long long want_end = exact < m ? exact : m;
      if (first != want_first || end != want_end) {
        fprintf(stderr, "m=%d group %zu: rows [%d, %d), not [%lld, %lld)\n", m, base + lane, first, end, want_first, want_end);
        return false;
      }
      first = end;
      ++g_checked;
    }
    before = first;
  }
  return true;
}

int main() {
  std::mt19937 rng(1);
  for (int m : {0, 1, 63, 1000, 33038209, 33038210, rd::kInt4MaxRows}) {
    for (int g : {1, 63, 64, 65, 128, 129, 192, 193, 600})
      for (int size : {INT_MIN, -1, 0, 1, m / 64, m / 2, m, m + 1, INT_MAX})
        if (!check(std::vector<int>(g, size), m)) return 1;
    for (int n = 0; n < 2000; ++n) {
      std::vector<int> sizes(1 + rng() % 400);
      for (int& s : sizes) {
        const unsigned kind = rng() % 8;
        s = kind < 4 ? (int)(rng() % (m / (int)sizes.size() + 2)) : kind == 4 ? 0 : kind == 5 ? -(int)(rng() % 1000) : kind == 6 ? (int)(rng() >> 1) : m;
      }
      if (!check(sizes, m)) return 1;
    }
  }
  printf("group_scan ok %lld\n", g_checked);
  return 0;
}
