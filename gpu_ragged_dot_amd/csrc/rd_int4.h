// The ragged product on 4-bit weights: launchers (rd_int4.hip) and the layout that they share.
//
// A weight is scale * (q - zero), q in 0 .. 15, one scale and one zero (8 where none are given) per `block` contraction indices
// (32, 64 or 128) of an output column.  In memory:
//   codes  [g][n][ceil(k / 128)][4][4] words: word j of piece h of a run of 128 indices holds the eight codes of the indices
//          32 j + 8 h + i, i = 0 .. 7, code i at bits 4 (i >> 1) + 16 (i & 1); codes past k are 8
//   scales [g][ceil(k / block)][n], bfloat16, float16 or float32;  zeros the same in bytes
//
// A lane's 16-byte load (a piece) is then four fragments of a 16x16x32 matrix-core instruction, whose lane group h = lane / 16
// wants the indices 8 h .. 8 h + 7 of a step of 32, and a step lies within one block whatever the block.  In a word, the codes
// of a 16-bit pair of neighbours are 16 bits apart: a shift and an and-or make both, as the 16-bit numbers 1 + q / 16.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rd {

constexpr int kInt4Run = 128;                // contraction indices per run
constexpr int kInt4MaxRows = (1 << 25) - 1;  // the sum of 64 groups' rows, each cut off at m, fits 32 bits

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
  int scale_elem;           // 0 bfloat16, 1 float32, 2 float16
  bool half;                // x and y are float16
};

__host__ __device__ inline int int4_runs(int k) { return (k + kInt4Run - 1) / kInt4Run; }

bool int4_grid_fits(const Int4Problem& p);  // a launch holds its work-groups
int launch_int4_pack(hipStream_t s, const uint8_t* q, uint32_t* codes, int g, int k, int n, bool trans_rhs);
int launch_gmm_int4(hipStream_t s, const Int4Problem& p);

}  // namespace rd
