// Rows and weights held as float8 e4m3fn with a scale for each block of 128, and the ragged product on them: launchers and layout.
//
// A block is 128 neighbours of a row (rows of x) or 128 x 128 of an expert's matrix (weights), the last ones short.  With
//   s = max(largest magnitude of the block, 2^-80) / 448, a float32; with pow2 the next power of two; NaN where the block holds a
//       NaN or an infinity
//   q = e4m3(x / s), the quotient a float32, both roundings to nearest even
// a block stands for q s.  448 is the largest e4m3fn number; below 2^-80 scales stop falling, so that neither they nor quotients
// get near the least numbers of 32 bits.  In memory (the block counts of k and n are ceil(k / 128) and ceil(n / 128)):
//   rows     codes [m][128 blocks], scales float32 [m][float8_scale_pitch(k)]
//   weights  codes [g][128 blocks(a)][128 blocks(b)], scales float32 [g][blocks(a)][blocks(b)]; [a, b] is [k, n], or [n, k]
// Codes of the padding are 0, NaN in a block that is NaN.  So every row of codes starts on a line of 128 bytes and no contraction has a tail.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rd {

constexpr int kF8Block = 128;
__host__ __device__ inline int float8_blocks(int k) { return (k + kF8Block - 1) / kF8Block; }
__host__ __device__ inline int float8_pitch(int k) { return float8_blocks(k) * kF8Block; }
__host__ __device__ inline int float8_scale_pitch(int k) { return (float8_blocks(k) + 3) & ~3; }  // whole 16-byte pieces of a row's scales

constexpr int kF8MaxRows = (1 << 25) - 1;  // 64 times as many fit 32 bits (counted_rows() in rd_int4_rows.h)
constexpr int kF8MaxDim = 1 << 22;         // 256 rows of codes stay below 2 GiB

// elem: 0 bfloat16, 1 float32, 2 float16
int launch_float8_rows(hipStream_t s, const void* x, void* codes, float* scales, long long rows, int k, bool swiglu, bool pow2, int elem);
int launch_float8_dispatch(hipStream_t s, const void* h, const int32_t* row_of_slot, const int32_t* slot_of_row, void* codes, float* scales,
                           int tokens, int top_k, int d, bool pow2, int elem);
int launch_float8_weights(hipStream_t s, const void* A, void* codes, float* scales, int g, int a, int b, bool pow2, int elem);
// rows (height 1, g = 1) or weights (height 128) back to numbers
int launch_float8_values(hipStream_t s, const void* codes, const float* scales, void* out, int g, int a, int b, int height, int elem);

struct F8Problem {
  const uint8_t* x;         // codes and scales of the rows
  const float* x_scales;
  const uint8_t* w;         // and of the weights
  const float* w_scales;
  const int32_t* group_sizes;
  void* y;                  // [m][n]
  int m, k, n, g;
  int g_first, g_local;     // the groups that the weights hold
  bool trans_rhs;
  int elem;                 // of y
};
int launch_gmm_float8(hipStream_t s, const F8Problem& p);
bool float8_grid_fits(const F8Problem& p);  // a launch holds its work-groups

}  // namespace rd
