// The ragged product on float8 rows and weights with a scale for each block of 128: which work-group computes which tile.
#include "rd_elem.h"
#include "rd_float8_tile.h"
#include "rd_int4_rows.h"

#include <math.h>

namespace rd {

namespace {

constexpr int kF8ZeroRows = 64;  // rows that a work-group looks after which multiplies nothing
constexpr int kF8Band = 8;       // row tiles of a band of the walk

constexpr int larger(int a, int b) { return a > b ? a : b; }

// Rows of a tile and columns; a tile of fewer rows runs on the least of the heights that holds it.
template <bool B_KMAJOR>
struct F8Tall {
  static constexpr int BM = 256, BN = 256, NT = 512, WAVES = 2;
  typedef F8TileCfg<256, 256, 2, 4, 2, B_KMAJOR> C256;
  typedef F8TileCfg<128, 256, 2, 4, 3, B_KMAJOR> C128;
  typedef F8TileCfg<64, 256, 2, 4, 3, B_KMAJOR> C64;
  static constexpr int LDS_BYTES = larger(C256::LDS_BYTES, larger(C128::LDS_BYTES, C64::LDS_BYTES));
  static __device__ __forceinline__ void run(const F8Tile& t, void* y, int ldy, int elem, unsigned char* smem) {
    const bool again = t.rows <= 64 ? float8_tile<C64>(t, y, ldy, elem, smem) : t.rows <= 128 ? float8_tile<C128>(t, y, ldy, elem, smem)
                                                                                             : float8_tile<C256>(t, y, ldy, elem, smem);
    if (again) float8_tile_any_scale<C64>(t, y, ldy, elem, smem);
  }
};
template <bool B_KMAJOR>
struct F8Middle {
  static constexpr int BM = 128, BN = 128, NT = 256, WAVES = 2;
  typedef F8TileCfg<128, 128, 2, 2, 2, B_KMAJOR> C128;
  typedef F8TileCfg<64, 128, 1, 4, 3, B_KMAJOR> C64;
  typedef F8TileCfg<32, 128, 1, 4, 3, B_KMAJOR> C32;
  static constexpr int LDS_BYTES = larger(C128::LDS_BYTES, larger(C64::LDS_BYTES, C32::LDS_BYTES));
  static __device__ __forceinline__ void run(const F8Tile& t, void* y, int ldy, int elem, unsigned char* smem) {
    const bool again = t.rows <= 32 ? float8_tile<C32>(t, y, ldy, elem, smem) : t.rows <= 64 ? float8_tile<C64>(t, y, ldy, elem, smem)
                                                                                            : float8_tile<C128>(t, y, ldy, elem, smem);
    if (again) float8_tile_any_scale<C32>(t, y, ldy, elem, smem);
  }
};
template <bool B_KMAJOR>
struct F8Few {
  static constexpr int BM = 64, BN = 128, NT = 256, WAVES = 2;
  typedef F8TileCfg<64, 128, 1, 4, 3, B_KMAJOR> C64;
  typedef F8TileCfg<32, 128, 1, 4, 3, B_KMAJOR> C32;
  static constexpr int LDS_BYTES = larger(C64::LDS_BYTES, C32::LDS_BYTES);
  static __device__ __forceinline__ void run(const F8Tile& t, void* y, int ldy, int elem, unsigned char* smem) {
    const bool again = t.rows <= 32 ? float8_tile<C32>(t, y, ldy, elem, smem) : float8_tile<C64>(t, y, ldy, elem, smem);
    if (again) float8_tile_any_scale<C32>(t, y, ldy, elem, smem);
  }
};
template <bool B_KMAJOR>
struct F8Narrow {  // a compute unit's LDS full of slabs on their way
  static constexpr int BM = 64, BN = 64, NT = 256, WAVES = 1;
  typedef F8TileCfg<64, 64, 1, 4, 8, B_KMAJOR> C64;
  typedef F8TileCfg<32, 64, 1, 4, 10, B_KMAJOR> C32;
  static constexpr int LDS_BYTES = larger(C64::LDS_BYTES, C32::LDS_BYTES);
  static __device__ __forceinline__ void run(const F8Tile& t, void* y, int ldy, int elem, unsigned char* smem) {
    const bool again = t.rows <= 32 ? float8_tile<C32>(t, y, ldy, elem, smem) : float8_tile<C64>(t, y, ldy, elem, smem);
    if (again) float8_tile_any_scale<C32>(t, y, ldy, elem, smem);
  }
};

// Work-groups [0, whole): a tile each; those behind them: rows, of which they zero what is no row of a group that the weights hold.
template <class S, bool B_KMAJOR>
__global__ __launch_bounds__(S::NT, S::WAVES) void gmm_float8_kernel(F8Problem p, int col_tiles, int whole) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int size = p.elem == 1 ? 4 : 2;
  if ((int)blockIdx.x >= whole) {
    int first, end;
    held_rows(p, &first, &end);
    const int r0 = ((int)blockIdx.x - whole) * kF8ZeroRows;
    for (int r = r0; r < imin(r0 + kF8ZeroRows, p.m); ++r)
      if (r < first || r >= end)
        for (int c = threadIdx.x; c < p.n; c += S::NT) {
          if (p.elem == 1) static_cast<float*>(p.y)[(size_t)r * p.n + c] = 0.f;
          else static_cast<uint16_t*>(p.y)[(size_t)r * p.n + c] = 0;
        }
    return;
  }
  const int positions = count_row_tiles<S::BM>(p, 1, p.m) * col_tiles;
  if ((int)(blockIdx.x >> 3) >= (positions + 7) / 8) return;  // (the launch holds as many work-groups as there may be tiles)
  const int at = xcd_contiguous_id(blockIdx.x, positions);
  if (at < 0) return;
  int column = 0;
  RowTile tile = find_in_walk<S::BM, kF8Band>(p, 1, p.m, col_tiles, at, &column);
  // the same in all lanes, and so in scalar registers: buffer descriptors made of others are read lane by lane in a loop around every load
  tile.group = __builtin_amdgcn_readfirstlane(tile.group);
  tile.first = __builtin_amdgcn_readfirstlane(tile.first);
  tile.rows = __builtin_amdgcn_readfirstlane(tile.rows);
  column = __builtin_amdgcn_readfirstlane(column);
  const int c0 = column * S::BN, kb = float8_blocks(p.k), nb = float8_blocks(p.n);
  const size_t e = tile.group - p.g_first;
  F8Tile t;
  t.lda = kb * kF8Block;
  t.ldb = B_KMAJOR ? t.lda : nb * kF8Block;
  t.ldas = float8_scale_pitch(p.k);
  t.a = p.x + (size_t)tile.first * t.lda;
  t.a_scales = p.x_scales + (size_t)tile.first * t.ldas;
  t.b = p.w + e * kb * nb * (kF8Block * kF8Block) + (size_t)c0 * (B_KMAJOR ? t.lda : 1);
  t.b_block = B_KMAJOR ? 1 : nb;
  t.b_column = B_KMAJOR ? kb : 1;
  t.b_scales = p.w_scales + e * kb * nb + (size_t)(c0 / kF8Block) * t.b_column;
  t.rows = tile.rows;
  t.cols = imin(S::BN, p.n - c0);
  t.blocks = kb;
  t.columns = B_KMAJOR ? t.cols : imin(S::BN, t.ldb - c0);
  S::run(t, static_cast<char*>(p.y) + ((size_t)tile.first * p.n + c0) * size, p.n, p.elem, smem);
}

// Which tiles, by rounds of what the device holds, if the rows are spread evenly and each of several groups has half a tile over: 256 tiles of
// 256 x 256 take 1 (of at most 128 rows 0.65), 512 of 128 x 128, two to a compute unit, 0.75, and 512 of 64 x 128 0.5; half a round of
// those 0.6 of it.  Groups of 32 rows and less have the least tiles, which run on 32 rows.
//
// us of 64 | 128 | 256 rows, trans_rhs, of rows dealt out at random: 8 groups of 128 x 2048 x 2048 17 | 19 | 33; of 256 rows 28 | 23 | 35; of
// 512 40 | 37 | 36; of 1024 66 | 56 | 67; 1 of 500 x 4096 x 4096 22 | 30 | 59; 128 of 64 x 2048 x 768 44 | 44 | 49; 32 of 256 x 1024 x
// 1024 26 | 25 | 23; 32 of 128 x 7168 x 2048 165 | 164 | 124; 8 of 256 x 4096 x 14336 230 | 197 | 196; 4 of 1024 x 4096 x 4096 115 | 100 | 120.
int height_for(const F8Problem& p) {
  const double rows = (double)p.m / p.g;
  if (rows <= 32) return 64;
  const auto time = [&](int h, int bn, int held, double round) {
    const double per_group = p.g == 1 ? ceil(rows / h) : rows / h + 0.5, tiles = p.g_local * (per_group > 1 ? per_group : 1) * ((p.n + bn - 1) / bn);
    const double whole = floor(tiles / held), rest = tiles - whole * held;
    return round * (whole + (rest <= 0 ? 0 : rest <= 256 && held > 256 ? 0.6 : 1));
  };
  const double tall = time(256, 256, 256, rows <= 128 ? 0.65 : 1), middle = time(128, 128, 512, 0.75), few = time(64, 128, 512, 0.5);
  return tall <= middle && tall <= few ? 256 : middle <= few ? 128 : 64;
}

// Launches of at most so many tiles of 64 x 128 take 64 columns: more work-groups, and as many slabs on their way as LDS holds.  us, 128 | 64
// columns, trans_rhs: 1 x 4096 x 4096 19.5 | 16.2; 33 rows in 4 groups x 7168 x 2048 31.4 | 26.4; 8 in 256 x 7168 x 2048 33.7 | 29.3 (without
// trans_rhs 46.9 | 41.8).  Of more tiles 64 columns have twice the rounds: 32 rows in 128 x 2048 x 768 11.6 | 19.5 (before tiles looked
// at their scales).
constexpr int kF8FewTiles = 128;
struct F8Grid {
  int height, width, col_tiles;
  long long whole, all;
};
F8Grid grid_of(const F8Problem& p) {
  F8Grid g;
  g.height = height_for(p);
  const auto tiles = [&] {
    g.col_tiles = (p.n + g.width - 1) / g.width;
    g.whole = ((p.m / g.height + imin(p.g_local, p.m)) * (long long)g.col_tiles + 7) / 8 * 8;
  };
  g.width = g.height == 256 ? 256 : 128;
  tiles();
  if (g.height == 64 && g.whole <= kF8FewTiles) {
    g.width = 64;
    tiles();
  }
  g.all = g.whole + (p.m + kF8ZeroRows - 1) / kF8ZeroRows;
  return g;
}

template <template <bool> class S, bool B_KMAJOR>
int launch_t(hipStream_t s, const F8Problem& p, const F8Grid& g) {
  auto kern = gmm_float8_kernel<S<B_KMAJOR>, B_KMAJOR>;
  if (S<B_KMAJOR>::LDS_BYTES > 64 * 1024) {
    const int rc = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, S<B_KMAJOR>::LDS_BYTES);
    if (rc != hipSuccess) return rc;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)g.all), dim3(S<B_KMAJOR>::NT), S<B_KMAJOR>::LDS_BYTES, s, p, g.col_tiles, (int)g.whole);
  return (int)hipGetLastError();
}

}  // namespace

bool float8_grid_fits(const F8Problem& p) { return grid_of(p).all < (1ll << 31) / 512; }

int launch_gmm_float8(hipStream_t s, const F8Problem& p) {
  const F8Grid g = grid_of(p);
  if (g.width == 64) return p.trans_rhs ? launch_t<F8Narrow, true>(s, p, g) : launch_t<F8Narrow, false>(s, p, g);
  if (g.height == 64) return p.trans_rhs ? launch_t<F8Few, true>(s, p, g) : launch_t<F8Few, false>(s, p, g);
  if (g.height == 128) return p.trans_rhs ? launch_t<F8Middle, true>(s, p, g) : launch_t<F8Middle, false>(s, p, g);
  return p.trans_rhs ? launch_t<F8Tall, true>(s, p, g) : launch_t<F8Tall, false>(s, p, g);
}

}  // namespace rd
