// Ragged product on 4-bit weights, for few rows per group: a stream over the codes (layout in rd_int4.h).
//
//   y[t, c] = sum_b scale[b, c] (sum_{kk in b} x[t, kk] q[kk, c] - zero[b, c] sum_{kk in b} x[t, kk])
//
// A code becomes the 16-bit number v = 1 + q / 16, exactly, by a shift and an and-or for two of them; the matrix cores sum
// x v over a block, and x itself against ones; then  y += 16 scale (sum x v) - scale (16 + zero) (sum x).  So products are
// exact, sums are fp32, and nothing is rounded to 16 bits before the result.
#include "../../include/ragged_dot_hip.h"
#include "rd_elem.h"
#include "rd_int4_rows.h"
#include "rd_int4_tile.h"

namespace rd {

namespace {

using int4_detail::load_at;
using int4_detail::scalar_base;
using int4_detail::scale_to_f32;

// ---- arithmetic ----------------------------------------------------------------------------------------------------------
template <bool HALF>
__device__ __forceinline__ f32x4_t mfma_16x16x32(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight codes of a word as 1 + q / 16: a code goes to the four highest bits of the fraction, under the exponent of one.  (The
// exponent sits in a vector register and the mask in a scalar one: as literals they would take an instruction each.)
template <bool HALF>
__device__ __forceinline__ u32x4_t codes_plus_one(uint32_t w) {
  constexpr int AT = HALF ? 6 : 3;  // of 10 and of 7 fraction bits
  uint32_t mask = 0x000f000fu << AT, one = HALF ? 0x3c003c00u : 0x3f803f80u;
  asm("" : "+s"(mask));
  asm("" : "+v"(one));
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((4 * i <= AT ? w << (AT - 4 * i) : w >> (4 * i - AT)) & mask) | one;
  return v;
}
template <bool HALF>
__device__ __forceinline__ u32x4_t ones() {
  constexpr uint32_t ONE = HALF ? 0x3c003c00u : 0x3f803f80u;
  return u32x4_t{ONE, ONE, ONE, ONE};
}

// Element i of eight of 16 bits, 0 before, set to e.
__device__ __forceinline__ u32x4_t insert_element(u32x4_t v, int i, uint32_t e) {
#pragma unroll
  for (int w = 0; w < 4; ++w) v[w] |= i >> 1 == w ? e << (16 * (i & 1)) : 0u;
  return v;
}

// ---- streaming kernel ------------------------------------------------------------------------------------------------------
// A work-group computes up to 32 rows of a group x 64 columns.  Its four waves take every fourth run of 128 contraction indices
// and add up their sums in LDS; a wave has the next run's loads in flight while it multiplies the present one.
//
// What bounds few rows is the stream over the codes, what bounds more of them the addresses that a compute unit's loads touch, one
// piece of a row of memory per cycle.  A fragment's lanes want 16 bytes of 16 rows of x, 64 pieces a load: read like that, x took
// 512 of the 640 pieces of a run of 32 rows (texture addresser busy 82 % of the time, matrix cores 20 %).  So x comes in whole
// rows, 16 lanes to a row's 256 bytes of a run (the tile's last row again for those that it does not have), and goes to the
// fragments through LDS, a wave's own part of it; and 64 columns' scales come in one load and to their lanes by a permutation.
constexpr int kInt4Threads = 256, kInt4Waves = 4, kInt4Cols = 64, kInt4Rows = 32, kInt4Strips = kInt4Cols / kInt4Strip;
constexpr int kInt4RowBytes = 2 * kInt4Run;  // of x in a run

template <int BLOCK>
struct Int4Run {
  static constexpr int PER = kInt4Run / BLOCK;
  typedef typename int4_detail::Bits<2 * PER>::type Scales;
  typedef typename int4_detail::Bits<PER>::type Zeros;
  u32x4_t codes[kInt4Strips];
  Scales scales;  // of column `lane`
  Zeros zeros;
};

__device__ __forceinline__ uint32_t from_column(uint32_t v, int lane4) { return (uint32_t)__builtin_amdgcn_ds_bpermute(lane4, (int)v); }
__device__ __forceinline__ uint64_t from_column(uint64_t v, int lane4) {
  return (uint64_t)from_column((uint32_t)v, lane4) | (uint64_t)from_column((uint32_t)(v >> 32), lane4) << 32;
}

// NT: row tiles of 16
template <bool HALF, int BLOCK, bool ZEROS, int NT>
__device__ __forceinline__ void int4_stream_tile(const Int4Problem& p, const RowTile& tile, int c0, unsigned char* smem) {
  typedef Int4Run<BLOCK> Run;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane & 15, h = lane >> 4, cols = imin(kInt4Cols, p.n - c0);
  const int runs = int4_runs(p.k), strips = int4_strips(p.n), e = tile.group - p.g_first;
  // Every address is a base that all lanes share and an offset of 32 bits.
  const size_t codes0 = ((size_t)e * strips + c0 / kInt4Strip) * runs * 1024, scales0 = (size_t)e * runs * p.n + c0;
  const uint32_t column = (uint32_t)imin(lane, cols - 1);
  auto load = [&](int r) {
    Run d;
    const size_t at = scales0 + (size_t)r * p.n;
    d.scales = load_at<typename Run::Scales>(scalar_base(p.scales, at * sizeof(typename Run::Scales)), column * (uint32_t)sizeof(typename Run::Scales));
    if constexpr (ZEROS) d.zeros = load_at<typename Run::Zeros, 1>(scalar_base(p.zeros, at * sizeof(typename Run::Zeros)), column * (uint32_t)sizeof(typename Run::Zeros));
#pragma unroll
    for (int c = 0; c < kInt4Strips; ++c) {
      const size_t strip = (size_t)imin(c, (cols - 1) / kInt4Strip) * runs + r;
      d.codes[c] = load_at<u32x4_t>(scalar_base(p.codes, codes0 + strip * 1024), lane * 16u);
    }
    return d;
  };
  // x: load i is rows 4 i + h, 16 bytes (chunk q) of each to a lane.  In LDS a row's chunks are permuted by its number, so that the 16
  // rows of a fragment read lie in different banks.
  constexpr int XL = 4 * NT;
  unsigned char* mine = smem + wave * (NT * 16 * kInt4RowBytes);
  const char* x0 = static_cast<const char*>(p.x) + (size_t)tile.first * p.k * 2;
  const uint32_t four_rows = (uint32_t)p.k * 8u, row0 = (uint32_t)h * (uint32_t)p.k * 2u + 16u * q, row_last = (uint32_t)(tile.rows - 1) * (uint32_t)p.k * 2u + 16u * q;
  auto fetch_x = [&](int r, u32x4_t (&d)[XL]) {
    const char* base = scalar_base(x0, (size_t)r * kInt4RowBytes);
#pragma unroll
    for (int i = 0; i < XL; ++i) d[i] = load_at<u32x4_t>(base, umin(row0 + (uint32_t)i * four_rows, row_last));
  };
  // Of the run that holds index k: zeros from there on.  A chunk that would run past it is read from before it and shifted down.
  auto fetch_x_tail = [&](int r, u32x4_t (&d)[XL]) {
    const int past = imax(r * kInt4Run + 8 * q + 8 - p.k, 0);  // elements
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const char* at = x0 + (size_t)r * kInt4RowBytes + umin(row0 + (uint32_t)i * four_rows, row_last);
      if (p.k >= 8) {
        d[i] = shift_down(load_any<u32x4_t>(at - 2 * past), 2 * imin(past, 8));
      } else {
        d[i] = u32x4_t{0, 0, 0, 0};
#pragma unroll 1
        for (int n = 0; n < 8 - past; ++n) d[i] = insert_element(d[i], n, *reinterpret_cast<const uint16_t*>(at + 2 * n));
      }
    }
  };
  auto stage_x = [&](const u32x4_t (&d)[XL]) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < XL; ++i)
      *reinterpret_cast<u32x4_t*>(mine + (4 * i + h) * kInt4RowBytes + ((q ^ ((4 * i + h) & 15)) << 4)) = d[i];
    __builtin_amdgcn_wave_barrier();
  };
  auto fragment = [&](int t, int j) { return *reinterpret_cast<const u32x4_t*>(mine + (16 * t + q) * kInt4RowBytes + (((4 * j + h) ^ q) << 4)); };

  f32x4_t y[NT][kInt4Strips];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < kInt4Strips; ++c) y[t][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // A run's blocks, two strips at a time.
  auto multiply = [&](const Run& d) {
    constexpr int STEPS = BLOCK / 32, U = 2;
#pragma unroll
    for (int b = 0; b < Run::PER; ++b) {
      f32x4_t xs[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) xs[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kInt4Strips; c += U) {
        f32x4_t v[U][NT];
#pragma unroll
        for (int j = b * STEPS; j < (b + 1) * STEPS; ++j) {
          u32x4_t w[U];
#pragma unroll
          for (int u = 0; u < U; ++u) w[u] = codes_plus_one<HALF>(d.codes[c + u][j]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const u32x4_t x = fragment(t, j);
            if (c == 0) xs[t] = mfma_16x16x32<HALF>(x, ones<HALF>(), xs[t]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
              v[u][t] = mfma_16x16x32<HALF>(x, w[u], j == b * STEPS ? zero : v[u][t]);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int from = (kInt4Strip * (c + u) + q) * 4;
          typedef typename std::conditional<sizeof(typename Run::Scales) == 8, uint64_t, uint32_t>::type Word;
          const float s = scale_to_f32((uint32_t)(from_column((Word)d.scales, from) >> (16 * b)) & 0xffff, p.scale_half);
          float plus = 24.f;  // 16 + zero
          if constexpr (ZEROS) plus = 16.f + (float)((from_column((uint32_t)d.zeros, from) >> (8 * b)) & 0xff);
          const float s16 = 16.f * s, sz = -s * plus;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[t][c + u][i] = __builtin_fmaf(s16, v[u][t][i], __builtin_fmaf(sz, xs[t][i], y[t][c + u][i]));
        }
      }
    }
  };
  const int whole = p.k / kInt4Run, own = (whole - wave + kInt4Waves - 1) / kInt4Waves;  // whole runs; this wave's
  u32x4_t xr[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) xr[i] = u32x4_t{0, 0, 0, 0};
  if (own > 0) {
    // Work-groups begin at runs of their own: strips lie runs x 1 KB apart, a multiple of 4 KB for most k, and all in step they
    // would ask a few memory channels at a time.  Two runs in turn, so that nothing that is still on its way is moved from one
    // register to another.
    int i = (int)(blockIdx.x % (uint32_t)own);
    auto turn = [&]() { i = i + 1 < own ? i + 1 : 0; return wave + i * kInt4Waves; };
    fetch_x(wave + i * kInt4Waves, xr);
    Run even = load(wave + i * kInt4Waves), odd;
    int left = own;
    for (; left >= 2; left -= 2) {
      stage_x(xr);
      const int second = turn();
      fetch_x(second, xr);
      odd = load(second);
      __builtin_amdgcn_sched_barrier(0);  // (the compiler would put these loads off until they are needed)
      multiply(even);
      stage_x(xr);
      const int third = turn();  // (behind the last run the first one again, for nothing)
      fetch_x(third, xr);
      even = load(third);
      __builtin_amdgcn_sched_barrier(0);
      multiply(odd);
    }
    if (left) {
      stage_x(xr);
      multiply(even);
    }
  }
  if (whole < runs && whole % kInt4Waves == wave) {
    const Run last = load(whole);
    fetch_x_tail(whole, xr);
    stage_x(xr);
    multiply(last);
  }
  float (*sums)[16][kInt4Cols] = reinterpret_cast<float (*)[16][kInt4Cols]>(smem);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (16 * t >= tile.rows) break;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kInt4Strips; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][4 * h + i][kInt4Strip * c + q] = y[t][c][i];
    __syncthreads();
    for (int cell = threadIdx.x; cell < imin(16, tile.rows - 16 * t) * kInt4Cols; cell += kInt4Threads) {
      const int r = cell / kInt4Cols, c = cell % kInt4Cols;
      if (c >= cols) continue;
      const float v = sums[0][r][c] + sums[1][r][c] + sums[2][r][c] + sums[3][r][c];
      uint16_t* out = static_cast<uint16_t*>(p.y) + (size_t)(tile.first + 16 * t + r) * p.n + c0 + c;
      if constexpr (HALF) *reinterpret_cast<f16_t*>(out) = (f16_t)v;
      else *out = f32_to_bf16(v);
    }
  }
}

// Work-groups [0, tiles * col_tiles): a row tile and 64 of its columns; those behind them: 64 rows, of which they zero what is
// no row of a group that the weights hold.
// ROWS: of a row tile, 16 or 32.
template <bool HALF, int BLOCK, bool ZEROS, int ROWS>
__global__ __launch_bounds__(kInt4Threads, ROWS == 16 ? 3 : 2) void gmm_int4_stream_kernel(Int4Problem p, int tiles, int col_tiles, int most) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[kInt4Waves * ROWS * kInt4RowBytes];
  if ((int)blockIdx.x >= tiles * col_tiles) {
    int first, end;
    held_rows(p, &first, &end);
    if (p.partials && (int)blockIdx.x == tiles * col_tiles && threadIdx.x < kInt4Slots) p.counters[threadIdx.x] = 0;  // of the tile kernel behind this one
    const int r0 = ((int)blockIdx.x - tiles * col_tiles) * kInt4Rows;
    for (int r = r0; r < imin(r0 + kInt4Rows, p.m); ++r)
      if (r < first || r >= end)
        for (int c = threadIdx.x; c < p.n; c += kInt4Threads) static_cast<uint16_t*>(p.y)[(size_t)r * p.n + c] = 0;
    return;
  }
  const RowTile tile = find_row_tile<ROWS>(p, 1, most, blockIdx.x / col_tiles);
  if (tile.rows == 0) return;
  const int c0 = blockIdx.x % col_tiles * kInt4Cols;
  int4_stream_tile<HALF, BLOCK, ZEROS, ROWS / 16>(p, tile, c0, smem);
}

// ---- laying out the weights --------------------------------------------------------------------------------------------------
// One word of eight codes per thread; from [g, n, k] its bytes in one load, 470 MB in 166 us (byte by byte 803).
__global__ __launch_bounds__(256) void int4_pack_kernel(const uint8_t* __restrict__ q, uint32_t* __restrict__ codes, long long words,
                                                        int k, int n, bool trans_rhs) {
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < words; at += (long long)gridDim.x * 256) {
    const int j = (int)(at & 3), c16 = (int)(at >> 2 & 15), h = (int)(at >> 6 & 3);
    const int runs = int4_runs(k), strips = int4_strips(n);
    const long long strip = (at >> 8) / runs;
    const int r = (int)((at >> 8) - strip * runs);
    const long long e = strip / strips, c = (strip - e * strips) * kInt4Strip + c16;
    const int k0 = r * kInt4Run + 32 * j + 8 * h;
    uint32_t w = 0;
    if (trans_rhs && k0 + 8 <= k && c < n) {
      const u32x2_t v = load_any<u32x2_t>(q + (e * n + c) * k + k0);
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= (v[i >> 2] >> (8 * (i & 3)) & 15u) << (4 * (i >> 1) + 16 * (i & 1));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v = k0 + i < k && c < n ? q[trans_rhs ? (e * n + c) * k + k0 + i : (e * k + k0 + i) * n + c] & 15u : 8u;
        w |= v << (4 * (i >> 1) + 16 * (i & 1));
      }
    }
    codes[at] = w;
  }
}

struct StreamGrid {
  int rows, tiles, col_tiles;  // rows of a tile; tiles at most, of groups with at most `most` rows
  long long blocks;
};
StreamGrid stream_grid(const Int4Problem& p, int most) {
  StreamGrid s;
  s.rows = p.m <= 8 * p.g ? 16 : kInt4Rows;
  const int groups = imin(p.g_local, p.m);
  const long long of_few = (long long)groups * ((most + s.rows - 1) / s.rows), of_any = p.m / s.rows + groups;
  s.tiles = (int)(of_few < of_any ? of_few : of_any);
  s.col_tiles = (p.n + kInt4Cols - 1) / kInt4Cols;
  s.blocks = (long long)s.tiles * s.col_tiles + (p.m + kInt4Rows - 1) / kInt4Rows;
  return s;
}

template <bool HALF, int BLOCK, bool ZEROS>
int stream(hipStream_t s, const Int4Problem& p, int most) {
  const StreamGrid g = stream_grid(p, most);
  const dim3 grid((unsigned)g.blocks);
  if (g.rows == 16) hipLaunchKernelGGL((gmm_int4_stream_kernel<HALF, BLOCK, ZEROS, 16>), grid, dim3(kInt4Threads), 0, s, p, g.tiles, g.col_tiles, most);
  else hipLaunchKernelGGL((gmm_int4_stream_kernel<HALF, BLOCK, ZEROS, kInt4Rows>), grid, dim3(kInt4Threads), 0, s, p, g.tiles, g.col_tiles, most);
  return (int)hipGetLastError();
}

// Whether groups of more rows than kInt4FewRows are left to the tile kernel, a launch of its own.  The sizes are on the device; the
// rule takes them to be equal, and what each kernel needs for that, us, from rounds of what the device holds at a time: 512
// work-groups of 32 rows x 64 columns of the streaming kernel at 1 and 4 per 1024 indices, 256 tiles of the other at 1.1 .. 2.0 a slab
// of 64 by their height.  bf16, blocks of 128, streaming | tiles: 32 groups of 64 x 7168 x 2048 168 | 135, 128 of 64 x 2048 x 768 85 |
// 81, 8 of 64 x 4096 x 14336 106 | 138, 32 of 128 x 2048 x 768 35 | 47, 17 of 96 x 328 x 3080 (blocks of 64, zeros) 35 | 24, where
// the rule is wrong.  Over 216 calls of random and of equal sizes it costs 0.7 % on the faster of the two, 35 % at worst (8 of 64 x
// 4096 x 14336) and more than 12 % in 8 of them.  Where the streaming kernel is long at work, groups of very different sizes pay for the other launch, a few us, whatever their mean.
constexpr int kInt4FewRows = 48;

// `held`: the groups that the weights hold, which is what either kernel multiplies, of the g that the m rows are spread over.
bool uses_tiles(int m, int k, int n, int g, int held, int kernel) {
  if (m <= kInt4FewRows || k < 8 || k > (1 << 22) || kernel == RD_INT4_STREAM) return false;
  if (kernel == RD_INT4_TILES) return true;
  const double rows = (double)((m + g - 1) / g), cols64 = (n + 63) / 64, cols256 = (n + 255) / 256;
  const double streaming = 6 + held * ceil(rows / 32) * cols64 / 512 * (1 + k * 0.004);
  if (streaming > 100) return true;
  if (rows <= kInt4FewRows) return false;
  const double last = rows - 256 * floor(rows / 256), height = last == 0 ? 0 : last <= 64 ? 1.1 : last <= 128 ? 1.3 : last <= 192 ? 1.65 : 2;
  const double work = held * cols256 * (2 * floor(rows / 256) + height) / 256, least = rows >= 256 ? 2 : height;
  return 12 + k / 64 * (work > least ? work : least) < streaming;
}

// Rows of the largest groups that the streaming kernel multiplies.
int most_streamed(const Int4Problem& p) {
  return int4_tiles_hold(p.half, p.scale_half) && uses_tiles(p.m, p.k, p.n, p.g, p.g_local, p.kernel) ? kInt4FewRows : p.m;
}

template <bool HALF, int BLOCK>
int gmm_int4(hipStream_t s, const Int4Problem& p) {
  const int most = most_streamed(p);
  const int rc = p.zeros ? stream<HALF, BLOCK, true>(s, p, most) : stream<HALF, BLOCK, false>(s, p, most);
  return rc != hipSuccess || most == p.m ? rc : launch_int4_tiles<HALF, BLOCK>(s, p, most + 1);
}
template <bool HALF>
int gmm_int4(hipStream_t s, const Int4Problem& p) {
  return p.block == 32 ? gmm_int4<HALF, 32>(s, p) : p.block == 64 ? gmm_int4<HALF, 64>(s, p) : gmm_int4<HALF, 128>(s, p);
}

}  // namespace

int launch_int4_pack(hipStream_t s, const uint8_t* q, uint32_t* codes, int g, int k, int n, bool trans_rhs) {
  const long long words = (long long)g * int4_strips(n) * int4_runs(k) * 256;
  hipLaunchKernelGGL(int4_pack_kernel, dim3((unsigned)(words < (1ll << 24) ? (words + 255) / 256 : 1 << 16)), dim3(256), 0, s, q, codes, words, k, n, trans_rhs);
  return (int)hipGetLastError();
}

size_t int4_workspace_bytes(int m, int k, int n, int g, int g_local, int kernel) {
  return uses_tiles(m, k, n, g, g_local, kernel) && n > 0 ? kInt4PartialBytes + kInt4Slots * sizeof(int32_t) : 0;
}

// (The tile kernel's work-groups are fewer than rows / 256 and groups come to, times the columns.)
bool int4_grid_fits(const Int4Problem& p) {
  const long long tiles = (p.m / 256 + imin(p.g_local, p.m)) * (long long)((p.n + 255) / 256);
  return stream_grid(p, most_streamed(p)).blocks < (1ll << 31) / kInt4Threads && tiles < (1ll << 31) / kInt4Threads;
}

int launch_gmm_int4(hipStream_t s, const Int4Problem& p) {
  return p.half ? gmm_int4<true>(s, p) : gmm_int4<false>(s, p);
}

}  // namespace rd
