// Ragged product on 4-bit weights, for few rows per group: a stream over the codes (layout in rd_int4.h).
//
//   y[t, c] = sum_b scale[b, c] (sum_{kk in b} x[t, kk] q[kk, c] - zero[b, c] sum_{kk in b} x[t, kk])
//
// A code becomes the 16-bit number v = 1 + q / 16, exactly, by a shift and an and-or for two of them; the matrix cores sum
// x v over a block, and x itself against ones; then  y += 16 scale (sum x v) - scale (16 + zero) (sum x).  So products are
// exact, sums are fp32, and nothing is rounded to 16 bits before the result.
#include "rd_elem.h"
#include "rd_int4.h"
#include "rd_lookup.h"

namespace rd {

namespace {

// ---- the row tile that a work-group computes -----------------------------------------------------------------------------
struct RowTile {
  int group;  // -1: none; g: rows behind the last group
  int first, rows;
};

// Row tile t of the groups in order, each cut into tiles of BM rows, then of the rows behind them.  Groups end at row m.
template <int BM>
__device__ __forceinline__ RowTile find_row_tile(const int32_t* __restrict__ gs, int g, int m, int t) {
  const int lane = threadIdx.x & 63;
  int rows_before = 0, tiles_before = 0;
  for (int base = 0; base < g; base += kLookupGroups) {
    int size[kLookupChunks];
#pragma unroll
    for (int c = 0; c < kLookupChunks; ++c) {
      const int e = base + 64 * c + lane;
      size[c] = e < g ? imin(imax(gs[e], 0), m) : 0;
    }
#pragma unroll
    for (int c = 0; c < kLookupChunks; ++c) {
      if (base + 64 * c >= g) break;
      const int end = imin(rows_before + wave_inclusive_sum(size[c]), m);
      const int before = __builtin_amdgcn_update_dpp(rows_before, end, 0x138, 0xf, 0xf, false);  // the lane below's: wave_shr:1
      const int rows = end - before, tiles_own = (rows + BM - 1) / BM;
      const int tiles = tiles_before + wave_inclusive_sum(tiles_own);
      const unsigned long long past = __ballot(tiles > t);
      if (past) {
        const int l = __ffsll(past) - 1;
        const int at = t - (__builtin_amdgcn_readlane(tiles, l) - __builtin_amdgcn_readlane(tiles_own, l));
        const int first = __builtin_amdgcn_readlane(before, l) + at * BM;
        return {base + 64 * c + l, first, imin(BM, __builtin_amdgcn_readlane(end, l) - first)};
      }
      rows_before = __builtin_amdgcn_readlane(end, 63);
      tiles_before = __builtin_amdgcn_readlane(tiles, 63);
    }
  }
  const int first = rows_before + (t - tiles_before) * BM;
  return {first < m ? g : -1, first, imin(BM, m - first)};
}

int row_tile_bound(int m, int g, int bm) { return m / bm + imin(g, m) + 1; }

// ---- arithmetic ----------------------------------------------------------------------------------------------------------
template <bool HALF>
__device__ __forceinline__ f32x4_t mfma_16x16x32(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight codes of a word as 1 + q / 16: a code goes to the four highest bits of the fraction, under the exponent of one.
template <bool HALF>
__device__ __forceinline__ u32x4_t codes_plus_one(uint32_t w) {
  constexpr int AT = HALF ? 6 : 3;  // of 10 and of 7 fraction bits
  constexpr uint32_t MASK = 0x000f000fu << AT, ONE = HALF ? 0x3c003c00u : 0x3f803f80u;
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((4 * i <= AT ? w << (AT - 4 * i) : w >> (4 * i - AT)) & MASK) | ONE;
  return v;
}
template <bool HALF>
__device__ __forceinline__ u32x4_t ones() {
  constexpr uint32_t ONE = HALF ? 0x3c003c00u : 0x3f803f80u;
  return u32x4_t{ONE, ONE, ONE, ONE};
}

__device__ __forceinline__ float load_scale(const void* p, size_t at, int elem) {
  return elem == 1 ? static_cast<const float*>(p)[at]
       : elem == 2 ? (float)static_cast<const f16_t*>(p)[at] : bf16_to_f32(static_cast<const bf16_bits*>(p)[at]);
}

// ---- streaming kernel ------------------------------------------------------------------------------------------------------
constexpr int kInt4Threads = 256, kInt4Waves = 4, kInt4Cols = 64;

// Eight consecutive elements of a row of x from index kk on, zeros from index k on.
__device__ __forceinline__ u32x4_t load_x(const uint16_t* row, int kk, int k) {
  if (kk + 8 <= k) return load_any<u32x4_t>(row + kk);
  alignas(16) uint16_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = kk + i < k ? row[kk + i] : 0;
  return *reinterpret_cast<u32x4_t*>(e);
}

// 16 rows x 64 columns; the four waves take every fourth run of 128 contraction indices and add up their sums in LDS.
template <bool HALF, int BLOCK>
__global__ __launch_bounds__(kInt4Threads) void gmm_int4_stream_kernel(Int4Problem p, int col_tiles) {
  __shared__ float sums[kInt4Waves][16][kInt4Cols];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowTile tile = find_row_tile<16>(p.group_sizes, p.g, p.m, blockIdx.x / col_tiles);
  if (tile.group < 0) return;
  const int c0 = blockIdx.x % col_tiles * kInt4Cols, cols = imin(kInt4Cols, p.n - c0);
  const int e = tile.group - p.g_first;
  const bool held = tile.group < p.g && e >= 0 && e < p.g_local;  // otherwise the rows are zero
  const int q4 = lane & 15, h = lane >> 4;
  const int runs = int4_runs(p.k), blocks = (p.k + BLOCK - 1) / BLOCK;
  f32x4_t y[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) y[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (held) {
    const uint16_t* xrow = static_cast<const uint16_t*>(p.x) + (size_t)(tile.first + imin(q4, tile.rows - 1)) * p.k;
    const uint32_t* codes = p.codes + (size_t)e * p.n * runs * 16;
    const size_t scale0 = (size_t)e * blocks * p.n;
    int col[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) col[c] = c0 + imin(16 * c + q4, cols - 1);
    for (int r = wave; r < runs; r += kInt4Waves) {
      u32x4_t w[4], x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const u32x4_t*>(codes + ((size_t)col[c] * runs + r) * 16 + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = load_x(xrow, r * kInt4Run + 32 * j + 8 * h, p.k);
      constexpr int STEPS = BLOCK / 32;
#pragma unroll
      for (int b = 0; b < 4 / STEPS; ++b) {
        const int kb = r * (kInt4Run / BLOCK) + b;
        if (kb >= blocks) break;
        f32x4_t xs = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < STEPS; ++j) xs = mfma_16x16x32<HALF>(x[b * STEPS + j], ones<HALF>(), xs);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < STEPS; ++j) v = mfma_16x16x32<HALF>(x[b * STEPS + j], codes_plus_one<HALF>(w[c][b * STEPS + j]), v);
          const size_t at = scale0 + (size_t)kb * p.n + col[c];
          const float s = load_scale(p.scales, at, p.scale_elem);
          const float z = p.zeros ? (float)p.zeros[at] : 8.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[c][i] = __builtin_fmaf(16.f * s, v[i], __builtin_fmaf(-s * (16.f + z), xs[i], y[c][i]));
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][4 * h + i][16 * c + q4] = y[c][i];
  __syncthreads();
  for (int at = threadIdx.x; at < tile.rows * kInt4Cols; at += kInt4Threads) {
    const int r = at / kInt4Cols, c = at % kInt4Cols;
    if (c >= cols) continue;
    const float v = sums[0][r][c] + sums[1][r][c] + sums[2][r][c] + sums[3][r][c];
    uint16_t* out = static_cast<uint16_t*>(p.y) + (size_t)(tile.first + r) * p.n + c0 + c;
    if constexpr (HALF) *reinterpret_cast<f16_t*>(out) = (f16_t)v;
    else *out = f32_to_bf16(v);
  }
}

// ---- laying out the weights --------------------------------------------------------------------------------------------------
// One word of eight codes per thread.
__global__ __launch_bounds__(256) void int4_pack_kernel(const uint8_t* __restrict__ q, uint32_t* __restrict__ codes, long long words,
                                                        int k, int n, bool trans_rhs) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= words) return;
  const int j = (int)(at & 3), h = (int)(at >> 2 & 3), runs = int4_runs(k);
  const long long column = (at >> 4) / runs;
  const int r = (int)((at >> 4) - column * runs);
  const long long e = column / n, c = column - e * n;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int kk = r * kInt4Run + 32 * j + 8 * h + i;
    const uint32_t v = kk < k ? q[trans_rhs ? column * k + kk : (e * k + kk) * n + c] & 15u : 8u;
    w |= v << (4 * (i >> 1) + 16 * (i & 1));
  }
  codes[at] = w;
}

template <bool HALF>
int stream(hipStream_t s, const Int4Problem& p) {
  const int col_tiles = (p.n + kInt4Cols - 1) / kInt4Cols;
  const dim3 grid((unsigned)row_tile_bound(p.m, p.g, 16) * (unsigned)col_tiles);
  if (p.block == 32) hipLaunchKernelGGL((gmm_int4_stream_kernel<HALF, 32>), grid, dim3(kInt4Threads), 0, s, p, col_tiles);
  else if (p.block == 64) hipLaunchKernelGGL((gmm_int4_stream_kernel<HALF, 64>), grid, dim3(kInt4Threads), 0, s, p, col_tiles);
  else hipLaunchKernelGGL((gmm_int4_stream_kernel<HALF, 128>), grid, dim3(kInt4Threads), 0, s, p, col_tiles);
  return (int)hipGetLastError();
}

}  // namespace

int launch_int4_pack(hipStream_t s, const uint8_t* q, uint32_t* codes, int g, int k, int n, bool trans_rhs) {
  const long long words = (long long)g * n * int4_runs(k) * 16;
  hipLaunchKernelGGL(int4_pack_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, q, codes, words, k, n, trans_rhs);
  return (int)hipGetLastError();
}

bool int4_grid_fits(const Int4Problem& p) {
  return (long long)row_tile_bound(p.m, p.g, 16) * ((p.n + kInt4Cols - 1) / kInt4Cols) < (1ll << 31) / kInt4Threads;
}

int launch_gmm_int4(hipStream_t s, const Int4Problem& p) {
  if (p.m == 0 || p.n == 0) return hipSuccess;
  return p.half ? stream<true>(s, p) : stream<false>(s, p);
}

}  // namespace rd
