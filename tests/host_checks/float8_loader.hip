// Host-side check of F8Loader (gpu_ragged_dot_amd/csrc/rd_float8_tile.h), which moves the slabs of float8 codes to LDS: for every tile
// shape of the product, over live rows and columns, pitches and blocks,
//   - every load of every slab that is not masked lies inside the tile's window, and inside the operand;
//   - a slab's cells in LDS are each written once, with the codes that the fragment readers look for there;
//   - masked loads are beyond every window.
// Built without GPU code by the library's Makefile; run by tests/test_float8_host.py.
#include <stdio.h>
#include <vector>
#include "rd_float8_tile.h"

static long long g_checked = 0;

template <int T, int NW, bool KMAJOR>
static bool check(int lim, int ld, int blocks) {
  typedef rd::F8Loader<T, NW, KMAJOR> L;
  const long long rows = KMAJOR ? lim : 128ll * blocks;  // of the operand behind the tile's first code
  const long long bytes = (rows - 1) * ld + (KMAJOR ? 128ll * blocks : lim);
  std::vector<int> written(T * 128 / 16);
  for (int at = 0; at < blocks; ++at) {
    std::fill(written.begin(), written.end(), 0);
    for (int wave = 0; wave < NW; ++wave)
      for (int lane = 0; lane < 64; ++lane) {
        L l;
        l.init(nullptr, ld, lim, blocks, wave, lane);
        if (l.records != bytes || (long long)at * l.step > 0x7fffffff) { fprintf(stderr, "window %d, not %lld\n", l.records, bytes); return false; }
        for (int j = 0; j < L::PER; ++j) {
          const int cell = (wave + NW * j) * 64 + lane;  // 16 bytes of LDS
          const int r = cell / L::CPR, c = (cell % L::CPR) ^ L::swizzle(r);
          ++written[cell];
          const bool live = KMAJOR ? r < lim : c * 16 < lim;
          if (live != (l.voff[j] != rd::kOobOffset)) { fprintf(stderr, "T %d row %d chunk %d: masked %d\n", T, r, c, !live); return false; }
          if (!live) {
            if ((unsigned)l.voff[j] < (unsigned)l.records) { fprintf(stderr, "a masked load inside the window\n"); return false; }
            continue;
          }
          const long long from = l.voff[j] + (long long)at * l.step;
          const long long want = KMAJOR ? (long long)r * ld + 128ll * at + 16 * c : (128ll * at + r) * ld + 16 * c;
          if (from != want || from < 0 || from + 16 > bytes) { fprintf(stderr, "T %d NW %d kmajor %d row %d chunk %d: %lld, not %lld of %lld\n", T, NW, KMAJOR, r, c, from, want, bytes); return false; }
          ++g_checked;
        }
      }
    for (int w : written)
      if (w != 1) { fprintf(stderr, "T %d NW %d kmajor %d: a cell written %d times\n", T, NW, KMAJOR, w); return false; }
  }
  return true;
}

template <int T, int NW>
static bool check_all() {
  for (int blocks : {1, 2, 3, 33, 112})
    for (int more : {0, 1, 7}) {
      for (int lim : {1, 15, 16, T / 2, T / 2 + 1, T - 1, T})
        if (!check<T, NW, true>(lim, 128 * (blocks + more), blocks)) return false;
      if constexpr (T >= 64)
        for (int lim : {T < 128 ? T : 128, T})
          if (!check<T, NW, false>(lim, 128 * ((T + 127) / 128 + more), blocks)) return false;
    }
  return true;
}

int main() {
  if (!check_all<256, 8>() || !check_all<128, 8>() || !check_all<64, 8>() || !check_all<128, 4>() || !check_all<64, 4>() || !check_all<32, 4>()) return 1;
  printf("float8_loader ok %lld\n", g_checked);
  return 0;
}
