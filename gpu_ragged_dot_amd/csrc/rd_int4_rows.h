// Which rows a work-group of a product on 4-bit weights computes, worked out by each wave from group_sizes.
#pragma once
#include "rd_int4.h"
#include "rd_lookup.h"

namespace rd {

// What a group's size counts behind `before` rows: negative ones nothing, and none more than the rows that are left.  So the sum
// of 64 groups and of what lies before them stays below 64 m, and 32 bits hold it (kInt4MaxRows).
__host__ __device__ __forceinline__ int counted_rows(int size, int before, int m) { return imin(imax(size, 0), m - before); }

// The groups as the waves of a launch see them: sizes that are negative count as 0 and groups end at row m.  kLookupGroups at a
// time, four per lane: f(chunk of 64 groups, first row and row behind the last one of lane's group) until it returns true.
template <class F>
__device__ __forceinline__ void scan_groups(const int32_t* __restrict__ gs, int g, int m, F&& f) {
  const int lane = threadIdx.x & 63;
  int rows_before = 0;
  for (int base = 0; base < g; base += kLookupGroups) {
    int size[kLookupChunks];
#pragma unroll
    for (int c = 0; c < kLookupChunks; ++c) {
      const int e = base + 64 * c + lane;
      size[c] = e < g ? gs[e] : 0;
    }
#pragma unroll
    for (int c = 0; c < kLookupChunks; ++c) {
      if (base + 64 * c >= g) break;
      const int end = imin(rows_before + wave_inclusive_sum(counted_rows(size[c], rows_before, m)), m);
      const int first = __builtin_amdgcn_update_dpp(rows_before, end, 0x138, 0xf, 0xf, false);  // the lane below's end: wave_shr:1
      if (f(base + 64 * c, first, end)) return;
      rows_before = __builtin_amdgcn_readlane(end, 63);
    }
  }
}

struct RowTile {
  int group, first, rows;  // rows 0: none
};

// Tile t of BM rows of the groups that the weights hold, in order, counting those of at least `least` and at most `most` rows.
template <int BM>
__device__ __forceinline__ RowTile find_row_tile(const Int4Problem& p, int least, int most, int t) {
  RowTile found = {0, 0, 0};
  int tiles_before = 0;
  const int lane = threadIdx.x & 63;
  scan_groups(p.group_sizes, p.g, p.m, [&](int base, int first, int end) {
    const int e = base + lane - p.g_first, rows = end - first;
    const int own = e >= 0 && e < p.g_local && rows >= least && rows <= most ? (rows + BM - 1) / BM : 0;
    const int tiles = tiles_before + wave_inclusive_sum(own);
    const unsigned long long past = __ballot(tiles > t);
    if (past) {
      const int l = __ffsll(past) - 1;
      const int at = (t - (__builtin_amdgcn_readlane(tiles, l) - __builtin_amdgcn_readlane(own, l))) * BM;
      const int f = __builtin_amdgcn_readlane(first, l), n = __builtin_amdgcn_readlane(rows, l);
      found = {base + l, f + at, imin(BM, n - at)};
      return true;
    }
    tiles_before = __builtin_amdgcn_readlane(tiles, 63);
    return false;
  });
  return found;
}

// The rows of the groups that the weights hold: [first, second); all others are zero.
__device__ __forceinline__ void held_rows(const Int4Problem& p, int* first_row, int* end_row) {
  int a = p.g_first == 0 ? 0 : -1, b = -1;
  scan_groups(p.group_sizes, p.g, p.m, [&](int base, int first, int end) {
    const int la = p.g_first - base, lb = p.g_first + p.g_local - 1 - base;
    if (la >= 0 && la < 64) a = __builtin_amdgcn_readlane(first, la);
    if (lb >= 0 && lb < 64) b = __builtin_amdgcn_readlane(end, lb);
    return lb < 64;
  });
  *first_row = a; *end_row = b;
}

// Row tiles in all, counted as find_row_tile() counts them.
template <int BM>
__device__ __forceinline__ int count_row_tiles(const Int4Problem& p, int least, int most) {
  int tiles = 0;
  const int lane = threadIdx.x & 63;
  scan_groups(p.group_sizes, p.g, p.m, [&](int base, int first, int end) {
    const int e = base + lane - p.g_first, rows = end - first;
    const int own = e >= 0 && e < p.g_local && rows >= least && rows <= most ? (rows + BM - 1) / BM : 0;
    tiles += __builtin_amdgcn_readlane(wave_inclusive_sum(own), 63);
    return false;
  });
  return tiles;
}

// Position `at` of a walk over all row tiles times `columns` column tiles: group after group, in a group bands of BAND row tiles,
// in a band column after column.  Returns the row tile and its column.
template <int BM, int BAND>
__device__ __forceinline__ RowTile find_in_walk(const Int4Problem& p, int least, int most, int columns, int at, int* column) {
  RowTile found = {0, 0, 0};
  int tiles_before = 0;
  const int lane = threadIdx.x & 63;
  scan_groups(p.group_sizes, p.g, p.m, [&](int base, int first, int end) {
    const int e = base + lane - p.g_first, rows = end - first;
    const int own = e >= 0 && e < p.g_local && rows >= least && rows <= most ? (rows + BM - 1) / BM : 0;
    const int tiles = tiles_before + wave_inclusive_sum(own);
    const int t = at / columns;
    const unsigned long long past = __ballot(tiles > t);
    if (past) {
      const int l = __ffsll(past) - 1;
      const int height = __builtin_amdgcn_readlane(own, l);
      const int local = at - (__builtin_amdgcn_readlane(tiles, l) - height) * columns;
      const int band = local / (BAND * columns), in_band = local - band * BAND * columns, tall = imin(BAND, height - band * BAND);
      *column = in_band / tall;
      const int row = (band * BAND + in_band % tall) * BM;
      found = {base + l, __builtin_amdgcn_readlane(first, l) + row, imin(BM, __builtin_amdgcn_readlane(rows, l) - row)};
      return true;
    }
    tiles_before = __builtin_amdgcn_readlane(tiles, 63);
    return false;
  });
  return found;
}

}  // namespace rd
