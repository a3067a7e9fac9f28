// The ragged product on 4-bit weights: launchers (rd_int4.hip) and the layout that they share.
//
// A weight is scale * (q - zero), q in 0 .. 15, one scale and one zero (8 where none are given) per `block` contraction indices
// (32, 64 or 128) of an output column.  In memory, with runs of 128 contraction indices and strips of 16 columns:
//   codes  [g][ceil(n / 16)][ceil(k / 128)][4][16][4] words: word j of piece (h, c) of a strip's run holds the eight codes of
//          column c and indices 32 j + 8 h + i, i = 0 .. 7, code i at bits 4 (i >> 1) + 16 (i & 1); codes past k and n are 8
//   scales [g][ceil(k / 128)][n][128 / block], bfloat16 or float16, 0 past k;  zeros the same in bytes
//
// A wave's load of 16 bytes per lane is then 1 KB of consecutive memory, and lane 16 h + c holds four fragments of a 16x16x32
// matrix-core instruction, whose lane group h wants the indices 8 h .. 8 h + 7 of a step of 32; a step lies within one block
// whatever the block.  In a word, the codes of a pair of neighbours are 16 bits apart: a shift and an and-or make both, as the
// 16-bit numbers 1 + q / 16.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rd {

constexpr int kInt4Run = 128, kInt4Strip = 16;
constexpr int kInt4MaxRows = (1 << 25) - 1;  // 64 times as many fit 32 bits (counted_rows() in rd_int4_rows.h)

struct Int4Problem {
  const void* x;            // [m][k], bfloat16 or float16
  const uint32_t* codes;
  const void* scales;
  const uint8_t* zeros;     // or null
  const int32_t* group_sizes;
  void* y;                  // [m][n]
  int m, k, n, g;
  int g_first, g_local;     // the groups that the weights hold
  int block;
  bool scale_half;          // scales are float16, else bfloat16
  bool half;                // x and y are float16
  int kernel;               // RD_INT4_*
  float* partials;          // kInt4Slots tiles of 256 x 256, or null: no tile is cut along k
  int32_t* counters;        // kInt4Slots, behind them
};

constexpr int kInt4Slots = 256;  // work-groups of the tile kernel that run at a time, one per compute unit
constexpr size_t kInt4PartialBytes = (size_t)kInt4Slots * 256 * 256 * sizeof(float);
// The tile kernel's weights are of the rows' type, and float16 does not have the range of bfloat16 scales.
inline bool int4_tiles_hold(bool half, bool scale_half) { return !half || scale_half; }
// Of the whole workspace, where the tiles hold the weights; 0: no launch of these sizes is cut.
size_t int4_workspace_bytes(int m, int k, int n, int g, int g_local, int kernel);

__host__ __device__ inline int int4_runs(int k) { return (k + kInt4Run - 1) / kInt4Run; }
__host__ __device__ inline int int4_strips(int n) { return (n + kInt4Strip - 1) / kInt4Strip; }

// Groups of at least `least` rows, by 256-column tiles (rd_int4_tile.hip; one object per instance).
template <bool HALF, int BLOCK>
int launch_int4_tiles(hipStream_t s, const Int4Problem& p, int least);

bool int4_grid_fits(const Int4Problem& p);  // a launch holds its work-groups
int launch_int4_pack(hipStream_t s, const uint8_t* q, uint32_t* codes, int g, int k, int n, bool trans_rhs);
int launch_gmm_int4(hipStream_t s, const Int4Problem& p);

}  // namespace rd
