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
__device__ __forceinline__ void tile_of(const Int4Problem& p, const RowTile& tile, int run, const Int4Columns& b, const SplitK& sk, unsigned char* smem) {
  typedef Int4TileCfg<BM, HALF, BLOCK> C;
  const int k0 = run * kInt4Run;
  int4_tile<C>(static_cast<const uint16_t*>(p.x) + (size_t)tile.first * p.k + k0, p.k, tile.rows, b, imin(p.k - k0, b.runs * kInt4Run),
               static_cast<uint16_t*>(p.y) + (size_t)tile.first * p.n + b.first, smem, sk);
}

// One work-group runs on a compute unit at a time, so the launch proceeds in rounds of kInt4Slots tiles.  `tiles` of them in the
// last round, which is not full: over how many work-groups each is cut along k.  us, as measured: a slab of 64 indices 2.0; what a
// cut costs, 28, and 0.09 for every piece's 256 KB of partial sums through memory and back.  A launch uncut | as cut so: 16 tiles of
// 2048 indices 58 | 45, of 4096 100 | 58, of 14336 310 | 87; 100 tiles 62 | 62, 105 | 90, 331 | 228; 128 tiles 63 | 63, 103 | 101, 338 |
// 254; 288 tiles, of which 32 are in the last round, 128 | 117, 225 | 195, 710 | 538.
__device__ __forceinline__ int split_parts(int tiles, int runs) {
  int best = 1;
  float least = 4.0f * runs;
  for (int p = 2; p <= 8 && p * tiles <= kInt4Slots && p * 4 <= runs; ++p) {
    const float t = 4.0f * ((runs + p - 1) / p) + 28.f + 0.09f * p * tiles;
    if (t < least) { least = t; best = p; }
  }
  return best;
}

// Work-groups [0, whole): whole tiles; kInt4Slots behind them: pieces of the last round's.
template <bool HALF, int BLOCK>
__global__ __launch_bounds__(256, 1) void gmm_int4_tile_kernel(Int4Problem p, int least, int col_tiles, int whole) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[Int4TileCfg<kTileRows, HALF, BLOCK>::LDS_BYTES];
  const int positions = count_row_tiles<kTileRows>(p, least, p.m) * col_tiles, runs = int4_runs(p.k);
  const int in_last = positions % kInt4Slots, parts = p.partials && in_last ? split_parts(in_last, runs) : 1;
  const int uncut = parts > 1 ? positions - in_last : positions;
  int at, run = 0, own_runs = runs;
  SplitK sk;
  if ((int)blockIdx.x < whole) {
    if ((int)(blockIdx.x >> 3) >= (uncut + 7) / 8) return;  // (the launch holds as many work-groups as there may be tiles)
    at = xcd_contiguous_id(blockIdx.x, uncut);
    if (at < 0) return;
  } else {
    // numbered by range of k first, so that neighbours at work at the same time share rows and columns
    const int piece = (int)blockIdx.x - whole;
    if (parts == 1 || piece >= parts * in_last) return;
    sk.parts = parts;
    sk.part = piece / in_last;
    const int tile = piece % in_last;
    at = uncut + tile;
    sk.partials = p.partials + (size_t)tile * parts * (kTileRows * kTileCols);
    sk.counter = p.counters + tile;
    run = (int)((long long)runs * sk.part / parts);
    own_runs = (int)((long long)runs * (sk.part + 1) / parts) - run;
  }
  int column = 0;
  const RowTile tile = find_in_walk<kTileRows, kTileBand>(p, least, p.m, col_tiles, at, &column);
  const int e = tile.group - p.g_first, c0 = column * kTileCols;
  constexpr int PER = kInt4Run / BLOCK;
  const size_t factors = ((size_t)e * runs + run) * p.n * PER;
  Int4Columns b;
  b.codes = reinterpret_cast<const char*>(p.codes) + (((size_t)e * int4_strips(p.n) + c0 / kInt4Strip) * runs + run) * 1024;
  b.scales = static_cast<const char*>(p.scales) + factors * 2;
  b.zeros = p.zeros ? reinterpret_cast<const char*>(p.zeros) + factors : b.scales;
  b.first = c0; b.n = p.n; b.runs = own_runs; b.stride = runs;
  b.has_zeros = p.zeros != nullptr; b.scale_half = p.scale_half;
  // the least of the heights that holds the tile
  if (tile.rows <= 64) tile_of<HALF, BLOCK, 64>(p, tile, run, b, sk, smem);
  else if (tile.rows <= 128) tile_of<HALF, BLOCK, 128>(p, tile, run, b, sk, smem);
  else if (tile.rows <= 192) tile_of<HALF, BLOCK, 192>(p, tile, run, b, sk, smem);
  else tile_of<HALF, BLOCK, 256>(p, tile, run, b, sk, smem);
}

}  // namespace

template <bool HALF, int BLOCK>
int launch_int4_tiles(hipStream_t s, const Int4Problem& p, int least) {
  const int col_tiles = (p.n + kTileCols - 1) / kTileCols;
  const long long tiles = (p.m / kTileRows + imin(p.g_local, p.m / least)) * (long long)col_tiles;
  const int whole = (int)((tiles + 7) / 8 * 8);
  hipLaunchKernelGGL((gmm_int4_tile_kernel<HALF, BLOCK>), dim3((unsigned)(whole + (p.partials ? kInt4Slots : 0))), dim3(256), 0, s, p, least, col_tiles, whole);
  return (int)hipGetLastError();
}

template int launch_int4_tiles<RD_INT4_HALF != 0, RD_INT4_BLOCK>(hipStream_t, const Int4Problem&, int);

}  // namespace rd
