// The tile kernel of the ragged product on 4-bit weights, one instance per object: -DRD_INT4_HALF=0|1 -DRD_INT4_BLOCK=32|64|128.
#include "rd_int4_rows.h"
#include "rd_int4_tile.h"

namespace rd {

namespace {

constexpr int kTileRows = 256, kTileCols = 256;
// Row tiles of a band: a band's rows times a few columns run on one XCD at a time, 32 tiles of which 4 x 8 fetch the least (x has
// four times the bytes of the codes per index, and a tile as many rows as columns).
constexpr int kTileBand = 4;

template <bool HALF, int BLOCK, int BM>
__device__ __forceinline__ void tile_of(const Int4Problem& p, const RowTile& tile, const Int4Columns& b, unsigned char* smem) {
  typedef Int4TileCfg<BM, HALF, BLOCK> C;
  int4_tile<C>(static_cast<const uint16_t*>(p.x) + (size_t)tile.first * p.k, p.k, tile.rows, b, p.k,
               static_cast<uint16_t*>(p.y) + (size_t)tile.first * p.n + b.first, smem);
}

template <bool HALF, int BLOCK>
__global__ __launch_bounds__(256, 1) void gmm_int4_tile_kernel(Int4Problem p, int least, int col_tiles) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[Int4TileCfg<kTileRows, HALF, BLOCK>::LDS_BYTES];
  const int positions = count_row_tiles<kTileRows>(p, least, p.m) * col_tiles;
  if ((int)(blockIdx.x >> 3) >= (positions + 7) / 8) return;  // (the launch holds as many work-groups as there may be positions)
  const int at = xcd_contiguous_id(blockIdx.x, positions);
  if (at < 0) return;
  int column = 0;
  const RowTile tile = find_in_walk<kTileRows, kTileBand>(p, least, p.m, col_tiles, at, &column);
  const int runs = int4_runs(p.k), e = tile.group - p.g_first, c0 = column * kTileCols;
  constexpr int PER = kInt4Run / BLOCK;
  const size_t factors = (size_t)e * runs * p.n * PER;
  Int4Columns b;
  b.codes = reinterpret_cast<const char*>(p.codes) + ((size_t)e * int4_strips(p.n) + c0 / kInt4Strip) * runs * 1024;
  b.scales = static_cast<const char*>(p.scales) + factors * 2;
  b.zeros = p.zeros ? reinterpret_cast<const char*>(p.zeros) + factors : b.scales;
  b.first = c0; b.n = p.n; b.runs = runs;
  b.has_zeros = p.zeros != nullptr; b.scale_half = p.scale_half;
  // the least of the heights that holds the tile
  if (tile.rows <= 64) tile_of<HALF, BLOCK, 64>(p, tile, b, smem);
  else if (tile.rows <= 128) tile_of<HALF, BLOCK, 128>(p, tile, b, smem);
  else tile_of<HALF, BLOCK, 256>(p, tile, b, smem);
}

}  // namespace

template <bool HALF, int BLOCK>
int launch_int4_tiles(hipStream_t s, const Int4Problem& p, int least) {
  const int col_tiles = (p.n + kTileCols - 1) / kTileCols;
  const long long tiles = (p.m / kTileRows + imin(p.g, p.m / least)) * (long long)col_tiles;
  hipLaunchKernelGGL((gmm_int4_tile_kernel<HALF, BLOCK>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(256), 0, s, p, least, col_tiles);
  return (int)hipGetLastError();
}

template int launch_int4_tiles<RD_INT4_HALF != 0, RD_INT4_BLOCK>(hipStream_t, const Int4Problem&, int);

}  // namespace rd
