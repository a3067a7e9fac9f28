// Host-side launcher of the Newton-Schulz iteration (rd_ortho.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rd {

constexpr int kOrthoMaxSteps = 32;
// Roundings of X in 15 bits, of 256 x 512 of rank 2, grown by 485 (five steps of a = 3.4445): 1.9e-3 of the result, by 1670: 7.6e-3, by
// 19816: 8.7e-2.
constexpr double kOrthoMostGrown = 2048;
constexpr int kOrthoPad = 64;  // matrices are padded to multiples of this inside

struct OrthoProblem {
  const void* G;  // [g][k][n]
  void* out;
  int g, k, n;
  int elem;  // 0 bfloat16, 1 float32, 2 float16
  int steps;
  const double* coefficients;  // [steps][3], on the host
  double eps, scale;
  void* workspace;
};

size_t ortho_workspace_bytes(int g, int k, int n, bool two);
// whether numbers are held in two float16 numbers: not those of bfloat16 matrices, unless their roundings grow too far
bool ortho_in_two(int elem, int steps, const double* coefficients);
bool ortho_grid_fits(int g, int k, int n);
// the largest singular value that the iteration can lead to from values up to 1
double ortho_growth(int steps, const double* coefficients);
int launch_orthogonalize(hipStream_t s, const OrthoProblem& p);

}  // namespace rd
