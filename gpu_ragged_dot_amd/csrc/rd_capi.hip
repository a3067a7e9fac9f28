// extern "C" entry points declared in include/ragged_dot_hip.h: argument checking, plan resolution, workspace
// carving, and the launches.  Nothing here allocates device memory or waits for the device.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "../../include/ragged_dot_hip.h"
#include <atomic>
#include <cstring>

#include "rd_decode.h"
#include "rd_int4.h"
#include "rd_moe.h"
#include "rd_kernels.h"
#include "rd_lookup.h"
#include "rd_sched.h"

// One getter per compiled tile shape; the list is generated by the Makefile.
#define RD_VARIANT(name) extern "C" const rd::TileVariant* rd_variant_##name();
#include "rd_variant_list.inc"
#undef RD_VARIANT

namespace {

typedef const rd::TileVariant* (*variant_getter)();
const variant_getter kVariantGetters[] = {
#define RD_VARIANT(name) &rd_variant_##name,
#include "rd_variant_list.inc"
#undef RD_VARIANT
};
constexpr int kNumVariants = (int)(sizeof(kVariantGetters) / sizeof(kVariantGetters[0]));

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int hip_fail(int rc, const char* what) {
  return fail(RD_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString((hipError_t)rc), rc);
}

inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
inline int cdiv(int a, int b) { return (a + b - 1) / b; }
inline int imin_host(int a, int b) { return a < b ? a : b; }

constexpr int kMinTileM = 16;  // bound used to size workspaces independently of the variant

// K-split of a gmm launch's last round: one slot (arrival counter + fp32 tile of partial sums) per piece, at most as
// many pieces as the device runs 160 KB work-groups at a time.  (Four times as many slots for the float32 tiles, so that more
// than half a round of tiles is cut too, gained 7 % on 512 x 4096 x 4096 in 3 groups and lost 5-18 % on 3000 x 1111 x 2222 in 5.)
constexpr int kSplitSlots = 256;

// The direct-to-LDS core addresses one tile's operand window through a 32-bit byte count.  gmm (op 0, 1): the
// window of a weight tile spans up to all of one expert's k x n matrix, that of an activation tile 256 rows.  tgmm
// (op 2): both windows span a group's rows, up to all m, at the row pitch of x (k) or dy (n).  The epilogue addresses the
// output tile the same way: up to 256 rows at the output's row pitch (n).
bool dlds_fits(int op, int m, int k, int n) {
  const long long lim = 1ll << 31;
  if (op == 2) return 2ll * m * (k > n ? k : n) < lim && 2ll * 256 * n < lim;
  return 2ll * k * n < lim && 2ll * 256 * (k > n ? k : n) < lim;
}

// The any-pitch core of rd_gemm_rs.h: the rows it reads along hold at least one 16-byte piece, and 256 rows of an operand or
// of the output stay within 32-bit byte offsets.
bool any_pitch_core_fits(int dtype, int k, int n) {
  const long long elem = dtype == RD_DTYPE_F32_BF16 || dtype == RD_DTYPE_F32 ? 4 : 2;
  return k >= 8 && n >= 8 && 256ll * elem * (k > n ? k : n) < (1ll << 31);
}

int find_variant(int bm, int bn, int vec, bool allow_dlds) {
  for (int i = 0; i < kNumVariants; ++i) {
    const rd::TileVariant* v = kVariantGetters[i]();
    if (v->bm == bm && v->bn == bn && v->vec == vec && v->dtype == RD_DTYPE_BF16 && (allow_dlds || !v->dlds)) return i;
  }
  return -1;
}

int first_variant_with_vec(int vec) {
  for (int i = 0; i < kNumVariants; ++i)
    if (kVariantGetters[i]()->vec == vec && kVariantGetters[i]()->dtype == RD_DTYPE_BF16) return i;
  return -1;
}

int first_variant_of_dtype(int dtype) {
  for (int i = 0; i < kNumVariants; ++i)
    if (kVariantGetters[i]()->dtype == dtype) return i;
  return -1;
}

int variant_by_name(const char* name);
long long est_tiles_256(int m, int n, int g);
int small_tile_variant(int op, int m, int k, int n, int g);

// 16-bit elements at pitches or addresses that the direct-to-LDS cores do not take: the 256 x 256 or the 128 x 128 form of the any-pitch core (rd_gemm_rs.h), or -1 where the 64 x 64 register-staged tile is the
// better one.  Measured, us, 256 | 128 | 64 (m x k x n in g groups):
//   bf16 fwd     8191 x 2047 x 4095 in 16: 218 | 286 | 521      8192 x 767 x 769 in 128: 58 | 67 | 92
//                4099 x 1001 x 1515 in 12: 42 | 33 | 63         1000 x 2047 x 767 in 64: 53 | 59 | 64
//                512 x 2047 x 2049 in 8: 42 | 29 | 41           700 x 333 x 777 in 7: 18 | 12 | 10
//   bf16 tgmm    8192 x 4094 x 4094 in 8: 338 | 459 | 722       4096 x 2047 x 2047 in 32: 171 | 197 | 221
//                30000 x 1001 x 1515 in 12 (zipf): 315 | 200 | 333      8192 x 513 x 513 in 64: 58 | 41 | 36
// So for gmm: the 256 x 256 tile, whose launch takes short groups' tiles at their own height, once it gives the compute
// units about a round of tiles (half a round for short groups with a long contraction) and does not pad n by more than a third (20996 x 2116 x 523 in 11: 129 | 112); the 64 x 64 one for launches that leave most compute units without a 128 x 128 tile, and for short groups,
// with a short contraction, whose tiles are over before the pipeline of the larger ones is full (128 x 128 over 64 x 64 on the 2603 calls that
// this left to the latter for its tiles alone, by contraction: 64 to 512 1.02-1.07, 512 to 1024 0.93 from 64 tiles on, 1024 to 2048 0.77 from 32 on, 2048 to 4096 0.74, more 0.54; 10273 x 250 x 1029 in 203:
// 69 | - | 63; 2306 x 77 x 2330 in 78: 33 | - | 24; 2731 x 289 x 140 in 153: - | 15 | 11).  tgmm, whose tiles take
// as long as their group has rows, wants four rounds of the large tile (or a single group), so that a long group's do not end
// the launch alone, and k and n that do not pad it by more than a fifth.  The 128 x 128 tile from 256 rows on with 96 of them or more
// and 96 indices each way; with fewer or narrower ones the longer the groups.  Over the 64 x 64 one, by rows of a group times tiles, launched one behind the other (1100 random calls that
// the 96 kept from it): 1024 rows and more 0.76 from 24000 to 32000, 0.65 beyond; 512 to 1024 rows 0.97-1.03 up to 50000, 0.82-0.87 beyond; 256 to 512 rows 1.3 under 24000, 0.90-1.04 up to
// 200000 (one in ten over 1.2), 0.77 beyond.  (Groups of 128 to 256 rows 0.9-1.1 whatever the tiles.)
//
// 16-bit elements also have a 128 x 256 tile, eight waves, one to a compute unit: three quarters of the 128 x 128 tile's loads per
// product, which are what bounds it (every 16 bytes at an odd address are an access of their own, the texture addresser is
// busy 81 % of a work-group's time, 74 % under the wider tile: profiles/any_pitch_core.md), and finer rounds than the 256 x 256 tile's.  gmm takes it where its expected tiles fill their rounds: one to
// 57 %, two, of groups long enough for the estimate to hold, to 78 %,
// with a contraction that is worth the fill.  Over the choice without it (profiles/default_rules_random_calls.md), contractions of 700 and
// more, by tiles: 110 to 130 1.21; 130 to 145 0.99 (one in ten over 1.33); 145 to 160 0.95; 160 to 180 0.90; 180 to 262 0.86; 262 to 400 1.0-1.03; groups of 400 rows and more
// 262 to 400 1.03-1.10, 400 to 512 0.95-0.97.  us: 4099 x 1001 x 1515 in 12: 33 | 27, trans_rhs 43 |
// 27 (256 x 256: 41, 40); 4181 x 4074 x 1675 in 2, trans_rhs: 98 | 80.  tgmm, whose tiles are as long as their groups, was level at best.
// Where the 256 x 256 tile would be taken, the 128 x 256 one is the better one up to four rounds of its tiles: 0.89-0.94 times up to three, 0.98 up to
// four; 0.98-1.0 beyond.  Not from contractions of 5000 on, whose last round is cut along K (up to 1.33).
constexpr int kFewTiles128x256 = 1000;
bool fills_rounds_128x256(long long rows, int k, int n, long long tiles) {
  if (n <= 128) return false;
  if (tiles <= 262) return tiles >= 145 && k >= 700;
  return rows >= 400 && k >= 300 && tiles >= 400 && tiles <= 512;
}

int any_pitch_variant(int dtype, int op, int m, int k, int n, int g) {
  const long long g_live = g < m ? g : m;
  if (g_live < 1 || !any_pitch_core_fits(dtype, k, n)) return -1;  // (no rows or no groups: a plan is asked for all the same)
  int tile = 0;
  if (op == 2) {
    const long long t128 = (long long)g * cdiv(k, 128) * cdiv(n, 128), t256 = (long long)g * cdiv(k, 256) * cdiv(n, 256);
    const long long rows = m / g;
    if (rows >= 64 && t256 >= (g == 1 ? 256 : 1024) && 20 * t256 <= 6 * t128) tile = 256;
    else if (rows >= 256 && ((t128 >= 96 && k >= 96 && n >= 96) ||
                             (k >= 56 && n >= 56 && rows * t128 >= (rows >= 1024 ? 24000 : rows >= 512 ? 60000 : 200000)))) tile = 128;
  } else if (n >= 96) {
    const long long t128 = (cdiv(m, 128) + g_live / 2) * cdiv(n, 128), t256 = est_tiles_256(m, n, g);
    const bool short_groups = (long long)m < 96 * g_live;
    if (short_groups && k < 300) tile = 0;
    else if (n >= 192 && t256 >= (short_groups && k >= 1500 ? 100 : 250) && 100ll * 256 * cdiv(n, 256) <= 135ll * n) tile = 256;
    else if (t128 >= 128 && (!short_groups || k >= 768)) tile = 128;
    else if (k >= 2048 || (k >= 512 && t128 >= (k >= 1024 ? 32 : 64))) tile = 128;
    if (tile == 256 && k < 5000 && (cdiv(m, 128) + g_live / 2) * cdiv(n, 256) <= kFewTiles128x256)
      return variant_by_name(dtype == RD_DTYPE_F16 ? "hr128x256x64_w2x4" : "r128x256x64_w2x4");
    if (!short_groups && fills_rounds_128x256(m / g_live, k, n, (cdiv(m, 128) + g_live / 2) * cdiv(n, 256)))
      return variant_by_name(dtype == RD_DTYPE_F16 ? "hr128x256x64_w2x4" : "r128x256x64_w2x4");
  }
  if (tile == 0) return -1;
  if (dtype == RD_DTYPE_BF16) return variant_by_name(tile == 256 ? "r256x256x64_w2x2" : "r128x128x64_w2x2");
  return variant_by_name(tile == 256 ? "hr256x256x64_w2x2" : "hr128x128x64_w2x2");
}

// What a launch on a tile is expected to take, in units of one that its callers share: t tiles of which the device holds `at_once` take
// t / at_once + `more` rounds (one, where they fit in one; a group's partial last tile counts as half), each as long as `weight` times
// the contraction - of tgmm: a group's rows - and `fill` indices more for the pipeline's fill and the stores.
struct ExpectedTile { int bm, bn, at_once; double weight, fill, more; };

double expected_time(const ExpectedTile& t, int op, int m, int k, int n, int g) {
  const int g_live = g < m ? g : m;
  const long long row_tiles = cdiv(m, t.bm) + g_live / 2;
  const double tiles = op == 2 ? (double)g * cdiv(k, t.bm) * cdiv(n, t.bn) : (double)(row_tiles > g_live ? row_tiles : g_live) * cdiv(n, t.bn);
  const double rounds = tiles / t.at_once;
  return t.weight * (rounds > 1 ? rounds + t.more : 1) * ((op == 2 ? (double)m / g : k) + t.fill);
}

// float32 rounded to bf16: up to how many 64 x 64 tiles a launch stays on them, as they are over before the any-pitch core's pipeline is
// full.  Time of kernels launched one behind the other, 128 x 128 over 64 x 64, by contraction (tgmm: rows of a group) and 64 x 64 tiles (23000
// random calls; through the Python entry points such launches look level, their 5 to 10 us are under what a call takes there):
//   gmm, 16-byte pitches   32 to 130: to 256 tiles 1.03-1.09, 256 to 512 0.93-0.96, 1024 to 2048 0.70-0.77;   130 to 200: to 256 0.95-1.02;   400 to 600: 0.83-0.93
//        others            16 to 32: to 256 1.14-1.32, 256 to 512 1.18, 1024 to 2048 0.70-0.77, over 4096 1.4-1.6;   32 to 65: to 256 1.12-1.21, to 512 1.07,
//                          over 4096 1.18-1.23;   65 to 130: 1.12-1.18, 1.06, 1.0;   130 to 260: to 256 1.01-1.14, 256 to 512 0.95-1.01;   260 to 400: 0.98-1.04, 0.88
//   tgmm, 16-byte pitches  16 to 32: to 768 1.12-1.27, to 1024 1.04, 1024 to 2048 0.99;   32 to 65: to 512 1.14-1.26, to 768 1.05, to 1024 0.99;   65 to 130: to 256
//                          1.12-1.18, to 512 1.02, to 768 0.94;   130 to 200: to 128 1.06-1.11, to 512 0.92
//         others           65 to 130: to 512 1.19-1.34, to 1024 1.13, 1024 to 2048 0.98;   130 to 160: to 512 1.16-1.24, to 1024 0.98;   160 to 260: to 128
//                          1.04-1.20, to 512 0.83-1.06;   260 to 320: to 128 1.04-1.08, to 512 0.84-0.91
long long brief_64x64_tiles(int op, double length, bool vec) {
  if (op == 2) return vec ? (length < 32 ? 1024 : length < 65 ? 768 : length < 130 ? 512 : length < 200 ? 128 : 0) : length < 130 ? 1024 : length < 160 ? 512 : length < 260 ? 128 : 0;
  return vec ? (length < 130 ? 256 : 0) : length < 130 ? 512 : length < 260 ? 256 : 0;
}

// float32 rounded to bf16 (compute_dtype = bfloat16).  The 64 x 64 tile of rd_gemm_tile.h for brief launches (above), and where tiles are little more than their
// stores: tgmm over groups of under 8 rows on average (16 with two to eight rounds of 128 x 128 tiles, 64 where k or n is no more; 64 at pitches of no whole
// 16 bytes), gmm of under 48 indices there with more than 4096 tiles, under 56 columns (of 57 to 63, 128 x 128 0.84 times, 52 calls), at most 64 indices and columns (level, and
// the core's plans ask for a workspace); the core's 128 x 128 tile for what gives under 96 of its 256 x 256 ones.  Its time over
// 256 x 256, by that one's expected tiles: gmm 32 to 64 0.71 | 0.84 at other pitches, 64 to 128 0.93 | 0.93, 128 to 256 1.05 | 0.98.
// Beyond, the tile that the launch is expected to be over with first (expected_time()).  Two lines beside that: gmm contractions of 6400 and more, whose last round is cut along K, take
// the 256 x 256 tile (up to 1.46 times without), and tgmm of several groups takes it from three rounds on, so that a long group's tiles
// do not end the launch alone (at 16-byte pitches mean 0.848 | 0.854 without | with the line, 98 in a hundred under 1.21 | 1.04), and from 32 rows
// (below, 128 x 128 0.97 times, and up to half on a few groups of large k and n).
// From 28759 random calls: 8 - 32768 rows, k and n of 9 - 16384, 1 - 256 groups of equal, softmax and Zipf shares.
// us, 256 x 256 | 128 x 128 | 64 x 64:
//   gmm   8192 x 4096 x 4096 in 8: 380 | 598 | 1597    26422 x 2400 x 672 in 34 (zipf): 179 | 245 | 419
//         10656 x 272 x 704 in 95: 30 | 26 | 41        879 x 448 x 2400 in 2: 17.5 | 12.7 | 20
//   tgmm  8192 x 4096 x 4096 in 8: 342 | 461 | 942     2322 x 1856 x 1264 in 49: 111 | 107 | 191
//         397 x 2560 x 1424 in 24: 88 | 74 | 102       982 x 512 x 496 in 32 (zipf): 20 | 13 | 17
int default_f32_bf16_variant(int op, int m, int k, int n, int g, bool vec) {
  static const ExpectedTile gmm_tiles[2][2] = {{{256, 256, 256, 1.0, 456, 0.54}, {128, 128, 512, 1.04, 113, 0.70}},
                                               {{256, 256, 256, 1.0, 189, 0.37}, {128, 128, 512, 1.0, 182, 0.18}}};
  static const ExpectedTile tgmm_tiles[2][2] = {{{256, 256, 256, 1.0, 582, 0.55}, {128, 128, 512, 0.776, 255, 0.48}},
                                                {{256, 256, 256, 1.0, 244, 0.68}, {128, 128, 512, 0.988, 143, 0.01}}};
  const double rows = (double)m / (g > 0 ? g : 1);
  const long long t128 = (long long)g * cdiv(k, 128) * cdiv(n, 128);  // tgmm's
  const bool few_rows = vec ? rows < (k <= 64 || n <= 64 ? 64 : t128 >= 1024 && t128 < 4096 ? 16 : 8) : rows < 64;
  const int g_live = g < m ? g : m;
  const long long row_tiles = cdiv(m, 64) + g_live / 2;
  const long long t64 = (op == 2 ? (long long)g * cdiv(k, 64) : row_tiles > g_live ? row_tiles : g_live) * cdiv(n, 64);
  if (!any_pitch_core_fits(RD_DTYPE_F32_BF16, k, n) || t64 <= brief_64x64_tiles(op, op == 2 ? rows : k, vec) ||
      (op == 2 ? few_rows : n < 56 || (k <= 64 && n <= 64) || (!vec && k < 48 && t64 > 4096)))
    return variant_by_name("c64x64x32_w2x2");
  const ExpectedTile* tiles = op == 2 ? tgmm_tiles[vec] : gmm_tiles[vec];
  bool tall = expected_time(tiles[0], op, m, k, n, g) < expected_time(tiles[1], op, m, k, n, g);
  if (op == 2) {
    tall = tall && rows >= 32 && (g == 1 || (long long)g * cdiv(k, 256) * cdiv(n, 256) >= 768);
  } else {
    tall = est_tiles_256(m, n, g) >= 96 && (tall || (k >= 6400 && n >= 192 && 100ll * 256 * cdiv(n, 256) <= 135ll * n));
  }
  if (vec) return variant_by_name(tall ? "cr256x256x32_w2x4" : "cr128x128x32_w2x2");
  return variant_by_name(tall ? "cs256x256x32_w2x4" : "cs128x128x32_w2x2");
}

// Arrays that are widened to bf16 on their way into LDS (float8; float32 rounded to bf16 and odd pitches above), float16 on register-staged tiles: the 128 x 128 tile when
// the groups are tall enough for it and it fills the device, else the 64-row tile of 256 columns where one is
// compiled (16-byte pitches), else the any-shape 64 x 64 one.
int default_variant(int op, int m, int k, int n, int g, bool vec);

// float16 at 16-byte pitches: the tile that bf16 arrays of this shape run on, compiled with the float16 instruction, but for the lines
// below, which are fitted to float16 times of 5260 random calls (256 - 32768 rows, k and n of 256 - 16384, 2 - 256 groups, equal,
// softmax-sized and skewed).  Time over that on the tiles float16 had before - the four-wave core for every 256 x 256 tile,
// v128x128x32 for d128x128x32, the 64 x 256 register-staged tile for the 64 x 64 one:
//   tgmm  64 x 64 0.82 (46 calls, 1.01 at worst);   128 x 128, three work-groups to a unit 0.82 in groups under 64 rows on average with
//         1600 tiles or more, 0.93 with 800, level below that; under 32 rows 0.84-0.97 whatever the tiles; over 64 rows up to 1.7 where groups are skewed;
//         eight-wave 256 x 256 0.86 (64 to 128 rows), 0.91, 0.93, 0.97 (512 to 1024), 1.01 beyond
//   trans_rhs  eight-wave 256 x 256 0.966 (0.88 in groups of 64 to 128 rows);  128 x 256 ping-pong 0.77-0.96 (6 calls, both layouts)
//   gmm   eight-wave 256 x 256, weights of 256 MB and more: 0.956 in groups under 128 rows, level from 128 to 160, 0.97 to 800, level beyond;
//         less weights: 1.01-1.04.
int float16_variant(int op, int m, int k, int n, int g, int as_bf16) {
  const rd::TileVariant* b = kVariantGetters[as_bf16]();
  const int g_live = op == 2 || g < m ? g : m;
  const double rows = (double)m / g_live, weight_mb = 2e-6 * (double)g_live * k * n;
  const char* name = b->name;
  if (b->dlds && b->bm == 256) {
    const bool eight = op == 2 ? rows < 1000 : b->split_rings && (op == 1 || (weight_mb >= 256 && (rows < 128 || (rows >= 160 && rows < 800))));
    if (!eight) name = "w256x256x32_w2x2_s5";
  } else if (std::strcmp(name, "d128x128x32_w2x2_s3") == 0) {
    const long long t128 = (long long)g * cdiv(k, 128) * cdiv(n, 128);
    if (op != 2 || rows >= 64 || (rows >= 32 && t128 < 800)) name = "v128x128x32_w2x2_s5";
  }
  char half_name[64];
  snprintf(half_name, sizeof(half_name), "h%s", name);
  return variant_by_name(half_name);  // (none for the register-staged tiles of other sizes)
}

int default_cvt_variant(int dtype, int op, int m, int k, int n, int g, bool vec) {
  if (dtype == RD_DTYPE_F32_BF16) return default_f32_bf16_variant(op, m, k, n, g, vec);
  if (dtype == RD_DTYPE_F16 && !vec) {
    const int any = any_pitch_variant(dtype, op, m, k, n, g);
    if (any >= 0) return any;
  }
  int big = -1, wide = -1, small_ = -1;
  if (dtype == RD_DTYPE_F16 && vec) {
    const int h = float16_variant(op, m, k, n, g, default_variant(op, m, k, n, g, vec));
    if (h >= 0) return h;
  }
  if (vec && dtype == RD_DTYPE_F8E4M3_BF16 && k % 16 == 0 && (op == 1 || n % 16 == 0) && dlds_fits(op, m, k, n)) {
    // float8 with 16-byte row pitches: the direct-to-LDS core on the float8 matrix-core instruction.  tgmm has its 256 x 256 tile, from about half a
    // round of tiles on; gmm the tile that the launch is expected to be over with first: 256 x 256, 128 x 256 with two work-groups to
    // a compute unit, so that one's epilogue hides behind the other's K loop, or 64 x 256.  Fitted to half of 2098 random calls (256 - 32768
    // rows, k and n of 256 - 16384, 2 - 256 groups); on the other half 1.019 (trans_rhs 1.035) times the best tile's time, 1.088 (1.102) before, by
    // counts of tiles; on 10585 others from 8 rows and 64 columns on, over the time before: under 256 rows 0.97 (trans_rhs 0.93), groups averaging
    // under 32 0.92 (0.92), 32 to 128 0.91 (0.89), more 0.96 (0.94).  Not 128 x 256 up to one round of 64 x 256 tiles: over that one's time, launched one behind
    // the other (14000 random calls), 1.11-1.28 up to 128 tiles, 1.16-1.20 up to 256, 0.79-0.93 up to 512 (trans_rhs 1.1-1.2, 1.05-1.15, 0.72-0.89).  us, 256 x 256 | 128 x 256 | 64 x 256:
    //   gmm  2283 x 1680 x 3152 in 7 25 | 32 | 43, 908 x 624 x 960 in 71 (zipf) 13 | 12 | 17, 292 x 272 x 2336 in 219 40 | 30 | 40;  trans_rhs  8329 x 7808 x
    //   1792 in 101 (zipf) 275 | 336 | 419, 3221 x 400 x 6624 in 100 102 | 69 | 94, 2121 x 7152 x 352 in 94 81 | 68 | 61
    static const ExpectedTile tiles[2][3] = {{{256, 256, 256, 1.0, 390, 0.30}, {128, 256, 512, 1.393, 60, 0.70}, {64, 256, 256, 0.788, 299, 0.38}},
                                             {{256, 256, 256, 1.0, 415, 0.09}, {128, 256, 512, 1.340, 92, 0.70}, {64, 256, 256, 1.025, 238, 0.13}}};
    static const char* const names[3] = {"x256x256x64_w2x4_s4", "x128x256x64_w2x4_s3", "x64x256x64_w1x4_s8"};
    if (op == 2) {
      if (k >= 256 && n >= 256 && (long long)g * cdiv(k, 256) * cdiv(n, 256) >= 128) return variant_by_name(names[0]);
    } else if (n >= 64) {
      const int g_live = g < m ? g : m;
      const long long row_tiles = cdiv(m, 64) + g_live / 2;
      const bool one_round = (row_tiles > g_live ? row_tiles : g_live) * cdiv(n, 256) <= 256;
      int best = 0;
      for (int i = one_round ? 2 : 1; i < 3; ++i)
        if (expected_time(tiles[op][i], op, m, k, n, g) < expected_time(tiles[op][best], op, m, k, n, g)) best = i;
      return variant_by_name(names[best]);
    }
  }
  for (int i = 0; i < kNumVariants; ++i) {
    const rd::TileVariant* v = kVariantGetters[i]();
    if (v->dtype != dtype || v->dlds || v->any_pitch_core) continue;  // (the direct-to-LDS float8 shapes serve one product only: chosen above)
    if (v->vec && v->bm >= 128 && big < 0) big = i;
    if (v->vec && v->bm < 128 && wide < 0) wide = i;
    if (!v->vec && small_ < 0) small_ = i;
  }
  if (!vec) return small_;
  const long long out_rows = op == 2 ? (long long)g * k : m;
  const long long rows_per_group = op == 2 ? k : (g > 0 ? m / g : m);
  const long long tiles = (out_rows / 128) * ((n + 127) / 128);
  if (big >= 0 && rows_per_group >= 96 && n >= 96 && tiles >= 128) return big;
  if (wide >= 0 && n >= 192) return wide;
  return small_ >= 0 ? small_ : big;
}

// float32 default: the tile that a launch of this size is expected to be over with first.  t tiles of which the device holds
// `at_once` take t / at_once + 0.365 rounds (a last round is seldom full), each as long as `weight` times the contraction and
// `fill` indices more for the pipeline's; a last round that will be cut along K (split_plan()) takes a `parts`-th of that and
// `piece` more for every piece.  In units of the 128 x 256 tile's time per contraction index (about 0.045 us).
//   gmm: three tiles of bf16 terms (rd_gemm_rs.h) and, for few small tiles, the 64 x 64 one on the float32 instruction, 64 columns
//   wide and three to a compute unit.  The 128 x 256 tile computes its last round in halves of its columns, which are 128 x 128
//   tiles, within that one's workspace: plans name the 128 x 128 tile for both, and a launch that is left to the library (no variant, or
//   split_k = 0) takes two columns of tiles to a work-group where that is the shorter way (pairs_f32_tiles()).
//   tgmm: a tile's contraction is its group's rows, nothing is cut, and groups of a few dozen rows are over before the other
//   tiles' pipelines are full: there the plain tile of rd_gemm_f32.h.
// Fitted to sizes of 256 - 32768 rows, k and n of 57 - 16384, 1 - 256 groups.  Outside them: gmm of under 57 columns keeps the tile of 64 (1.05-1.12 times as
// long with the fit, 112 random calls; now 1.00 over 3253), of under 64 indices the ones of 64 rows (those of 128 took 1.0-1.10 times the time before the terms, 91
// calls; now 0.98 over the 1128 whose tile is another one than then).
// On fresh calls of that range the choice takes 1.035 (gmm, 1742 calls) and 1.035 times (tgmm, 892) the best tile's time, those on the float32 instruction alone 1.30 and
// 1.22 (profiles/default_rules_random_calls.md).  us, 128 x 256 | 128 x 128 | 64 x 128 of terms | 64 x 64 | plain 64 x 64:
//   gmm   8192 x 2048 x 2048 in 16 groups: 391 | 446 | 472 | 580 | 719     4096 x 2048 x 2048 in 4: 210 | 224 | 231 | 332 | -
//         2692 x 336 x 1488 in 7: 34 | 43 | 39 | 47 | 49                   1334 x 7584 x 768 in 5: 117 | 118 | 229 | 175 | 442
//         27488 x 640 x 384 in 50: 97 | 96 | 115 | 130 | 158               883 x 2134 x 1492 in 16: 86 | 91 | 78 | 91 | 153
//         777 x 333 x 421 in 5: 29 | 20 | 17 | 14 | -
//   tgmm  8192 x 2048 x 2048 in 16: 380 | 440 | - | 613 | 680              14520 x 1488 x 1008 in 225: 572 | 681 | - | 812 | 704
//         27488 x 640 x 384 in 50: 184 | 145 | - | 170 | 257               1190 x 560 x 624 in 110: 73 | 85 | - | 80 | 33
struct F32Tile {
  const rd::TileVariant* v;
  int id, at_once;
  double weight, fill, piece;
  F32Tile(const char* name, int at_once_, double weight_, double fill_, double piece_)
      : v(kVariantGetters[variant_by_name(name)]()), id(variant_by_name(name)), at_once(at_once_), weight(weight_), fill(fill_), piece(piece_) {}
};
struct F32Tiles {
  F32Tile gmm[4] = {{"ft128x256x32_w2x4", 256, 1.0, 160, 0}, {"ft128x128x32_w2x4", 256, 0.66, 260, 91},
                    {"ft64x128x32_w2x2", 512, 0.80, 153, 46}, {"fr64x64x32_w2x2", 768, 0.71, 145, 38}};
  F32Tile tgmm[4] = {{"ft128x256x32_w2x4", 256, 1.0, 175, 0}, {"ft128x128x32_w2x4", 256, 0.575, 170, 0},
                     {"fr64x64x32_w2x2", 768, 0.575, 135, 0}, {"f64x64x16_w2x2", 1024, 1.42, 24, 0}};
  const F32Tile &pair = gmm[0], &single = gmm[1], &plain = tgmm[3];
};
const F32Tiles& f32_tiles() {
  static const F32Tiles tiles;  // (looked up by name once)
  return tiles;
}

// How many pieces split_plan() makes of each last tile of a launch of `tiles`, for a plan that leaves it to the library (1: none are cut).
int split_parts_for(const rd::TileVariant* v, long long tiles, int k) {
  const rd::SplitRule cut{k, (int)((long long)k * v->split_quarters / 4), v->split_min_k, v->splitk ? kSplitSlots : 0, kSplitSlots, 0, v->split_by_gain != 0};
  const int live = (int)(tiles < kSplitSlots ? tiles : kSplitSlots + tiles % kSplitSlots);  // (one whole round or several: the same)
  return rd::split_plan(live, cut, v->split_bn < v->bn ? 2 : 1).parts;
}

// cut: whether the launch may compute its last round in halves and pieces (a default plan assumes so).
double f32_gmm_cost(const F32Tile& t, int m, int k, int n, int g, bool cut) {
  const rd::TileVariant* v = t.v;
  const int g_live = g < m ? g : m;
  const long long row_tiles = cdiv(m, v->bm) + g_live / 2, tiles = (row_tiles > g_live ? row_tiles : g_live) * cdiv(n, v->bn);
  const long long last = tiles % kSplitSlots, full = tiles - last;
  const double whole = k + t.fill;
  if (cut && v->split_bn < v->bn) {
    const F32Tile& half = f32_tiles().single;
    const int parts = split_parts_for(v, last, k);
    const double halves = half.weight * ((double)k / parts + half.fill + (parts > 1 ? half.piece * parts : 0));
    return (double)full / t.at_once * whole + (last == 0 ? 0 : 2 * last <= kSplitSlots ? halves : whole);
  }
  const int parts = cut ? split_parts_for(v, last, k) : 1;
  const double rounds = (double)tiles / t.at_once, pieces = (double)last * parts / t.at_once;
  if (parts < 2) return t.weight * (rounds > 1 ? rounds + 0.365 : 1) * whole;
  return t.weight * ((double)full / t.at_once * whole + (double)k / parts * (pieces > 1 ? pieces : 1) + t.fill + t.piece * parts);
}

bool pairs_f32_tiles(int m, int k, int n, int g, bool cut) {
  const F32Tiles& tiles = f32_tiles();
  return f32_gmm_cost(tiles.pair, m, k, n, g, cut) < f32_gmm_cost(tiles.single, m, k, n, g, cut);
}

int default_f32_variant(int op, int m, int k, int n, int g) {
  const F32Tiles& tiles = f32_tiles();
  if (!any_pitch_core_fits(RD_DTYPE_F32, k, n)) return tiles.plain.id;
  if (op != 2 && n < 57) return tiles.gmm[3].id;
  const F32Tile* best = nullptr;
  double least = 0;
  for (const F32Tile& t : op == 2 ? tiles.tgmm : tiles.gmm) {
    if (op != 2 && k < 64 && t.v->bm == 128) continue;
    const double rounds = (double)g * cdiv(k, t.v->bm) * cdiv(n, t.v->bn) / t.at_once;
    const double cost = op == 2 ? t.weight * (rounds > 1 ? rounds + 0.114 : 1) * ((double)m / (g > 0 ? g : 1) + t.fill)
                                : f32_gmm_cost(t, m, k, n, g, true);
    if (!best || cost < least) { best = &t; least = cost; }
  }
  return op != 2 && best == &tiles.pair ? tiles.single.id : best->id;
}

// bytes of one element of the output
size_t out_elem_bytes(int dtype) { return dtype == RD_DTYPE_F32 || dtype == RD_DTYPE_F32_BF16 ? 4 : 2; }

bool vec_ok(const void* a, const void* b, const void* c, int k, int n) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  return k % 8 == 0 && n % 8 == 0 && al(a) && al(b) && al(c);
}

int variant_by_name(const char* name) {
  for (int i = 0; i < kNumVariants; ++i)
    if (std::strcmp(kVariantGetters[i]()->name, name) == 0) return i;
  return -1;
}

// Expected number of 256 x 256 tiles of a gmm launch: a group's partial last tile counts as half a tile.
long long est_tiles_256(int m, int n, int g) {
  const long long g_live = g < m ? g : m;
  return (cdiv(m, 256) + g_live / 2) * cdiv(n, 256);
}

// Default tile walk of gmm: bands of 2 row tiles in blocks of 8 while the launch has only a few rounds of tiles (small
// blocks spread them evenly over the XCDs), bands of 4 in blocks of 32 - what an XCD runs at a time - beyond that.
// 64 x 64 tiles: blocks of 16 (a block of 8 of them is 128 rows x 256 columns - too little shared between its tiles:
// 36 against 27 us on 1024 x 2048 x 512 in 4 groups with trans_rhs).
void default_walk(int m, int k, int n, int g, const rd::TileVariant* v, int* group_m, int* group_n) {
  if (v->bm <= 64 && v->bn <= 64) { *group_m = 4; *group_n = 4; return; }
  // The eight-wave core with short routines, many groups of about one row tile: bands of one row tile, so that a block does not
  // alternate between a group's whole tile and its short last one.  us, bands of two or four | one: 24576 x 3072 x 1024 in 96 221 | 204,
  // 16384 x 2048 x 3584 in 64 315 | 297, trans_rhs 24458 x 880 x 1248 in 91 121 | 112, 31929 x 880 x 3072 in 125 311 | 293 (equal
  // groups; softmax-sized and skewed ones are level).  0.99 times on 91 calls of this range, 1.02 at worst.  Blocks of 32 gain more on
  // equal groups (trans_rhs 32768 x 768 x 2048 in 128 171 | 163) and lose up to 5 % on skewed ones.  Outside the range blocks of 32
  // lost up to 14 % (21140 x 7792 x 1136 in 71: 533 | 606), blocks of 8 were not measured.
  if (v->split_rings && k <= 3072 && n <= 3584 && g >= 64 && (long long)m >= 192ll * g && (long long)m <= 384ll * g) { *group_m = 1; *group_n = 8; return; }
  // Groups that average at most half a tile's height have one row tile each, so a band is one row of tiles and a block
  // of 8 positions is 8 column tiles of one group; blocks of 32 then span four groups' weights (DeepSeek-V3 shapes, both
  // projections, and softmax-sized groups of 128 rows on average: 1.5-5 % for 2 x 4 over 4 x 8).
  const bool few = est_tiles_256(m, n, g) < 1536 || (long long)m <= 128ll * g;
  *group_m = few ? 2 : 4;
  *group_n = few ? 4 : 8;
}

// Groups whose row tiles want the streaming routines of the four-wave 256 x 256 core: below a quarter of its height, and up to half
// of it (forward: 100 rows) where the weights are more than the last-level cache holds.  Streamed past the cache they lie in, the
// others' cost 4 to 15 % (trans_rhs 64 to 128 rows, 250 calls: 0.90 times on the tiles this leaves them to, forward 64 to 100, 51 calls: 0.90).
bool wants_stream(int op, double rows, double weight_mb) { return rows < 64 || (rows < (op == 1 ? 128 : 100) && weight_mb >= 256); }

// bfloat16 and float16 at 16-byte pitches: the tile of the core of rd_gemm_ws.h that computes the product, or -1 where another
// core is the better one.  The lines are fitted to bfloat16 times of random calls (256 - 32768 rows, k and n of 256 - 16384, 2 - 256
// groups); float16 follows them.  On others of that range what the whole rule picks is 4 % (gmm), 6 % (trans_rhs) and 4 % (tgmm) from
// the best variant of each call, float16 4, 6 and 10 % before float16_variant() had lines of its own, and takes 0.78, 0.73 and 0.80 times what the rules before this core took, 0.61,
// 0.61 and 0.78 (geometric means; profiles/default_rules_random_calls.md).  us, before | now:
//                                   gmm         trans_rhs   tgmm
//   259 x 10432 x 336 in 3          83 | 23     134 | 24    8 | 8
//   512 x 4096 x 4096 in 2          60 | 32     56 | 30     33 | 31
//   2048 x 2048 x 2048 in 4         39 | 28     36 | 28     23 | 23
//   4096 x 1000 x 1512 in 12        28 | 23     45 | 37     42 | 29
//   13785 x 960 x 400 in 24 (zipf)  24 | 20     28 | 23     82 | 41
// gmm: the smaller the launch, the smaller the tile.  64-wide slabs and a deep ring (one work-group to a compute unit) where a
// work-group has the unit to itself anyway and the contraction is long, 32-wide slabs with two to a unit where tiles are many
// and short.  From about two thirds of a round of 256 x 256 tiles on those move fewer bytes per tile, and groups well below
// their height want the streaming routines of the four-wave core.  tgmm pads k and n instead of rows; its tiles are as long as
// the groups: 128 x 256 with two work-groups to a unit, so that one's stores run behind the other's loop; 128 x 128 where the
// longest groups would otherwise end the launch alone; three work-groups of d128x128x32 to a unit where a tile is little more
// than its stores; 256 x 256 for long groups (four waves) and where x is large: below 100 MB the 128 x 256 tiles take 0.90 times what
// those take (2800 random calls, three sets of operands in turn; 32768 x 768 x 2048 in 128 groups 211 | 173 us), from there on the
// smaller tiles read it more often than the last-level cache makes up for: 0.97 to 200 MB, 0.99 to 300, 1.01 beyond (2860 calls; 8192 x 7168
// x 2048 in 32 groups 338 | 365, 26305 x 9856 x 960 in 104 749 | 815).
int small_tile_variant(int op, int m, int k, int n, int g) {
  const long long g_live = g < m ? g : m;
  const double rows = (double)m / (op == 2 ? g : g_live);  // of a group, on average
  const double x_mb = 2e-6 * m * k, weight_mb = 2e-6 * (double)g_live * k * n;
  const char* name = nullptr;
  if (op == 2) {
    const long long t256 = (long long)g * cdiv(k, 256) * cdiv(n, 256), t128 = (long long)g * cdiv(k, 128) * cdiv(n, 128);
    const long long t64x64 = (long long)g * cdiv(k, 64) * cdiv(n, 64);
    const bool padded = 256ll * cdiv(n, 256) * 100 > 107ll * n;  // 256-column tiles pad n by more than 7 %
    if (k < 128 || n < 128 || (t128 < 64 && rows < 600)) return -1;
    if (t64x64 < 2190) {
      if (rows < 113) return -1;
      name = "v128x128x32_w2x2_s5";
    } else if ((rows >= 1900 && t256 >= 170) || (n % 64 == 0 && (rows <= 64 || (rows <= 128 && t256 >= 16384)))) {
      return -1;  // (level: 3072 x 3072 x 3072 in 48 193 | 183, 16384 x 2048 x 4096 in 128 563 | 537)
    } else if (x_mb < 0.7 || (x_mb >= 100 && rows >= 128) || (padded && (rows < 145 ? t256 < 7000 : x_mb >= 41))) {
      return -1;
    } else {
      name = "v128x256x32_w2x2_s3";
    }
    return variant_by_name(name);
  }
  if (n < 128 || m < 64) return -1;
  // expected tiles: a group's partial last one counts as half
  const double part = 0.5 * (double)g_live;
  const double t64 = (cdiv(m, 64) + part) * cdiv(n, 128), t64x64 = (cdiv(m, 64) + part) * cdiv(n, 64);
  const double t128 = (cdiv(m, 128) + part) * cdiv(n, 128), t256 = (cdiv(m, 256) + part) * cdiv(n, 256);
  const bool round_and_a_bit = t256 > 262 && t256 < 400 && k < 5000;  // of 256 x 256 tiles
  if (op == 0) {
    if (t64 < 530) {
      if (t64x64 <= 520 && k <= 2000) name = "v64x64x64_w2x2_s5";
      else if (x_mb < 7.7) {
        if (t128 < 100) name = k < 5540 ? "v64x64x64_w2x2_s5" : "v64x128x64_w2x2_s6";
        else if (rows < 171) name = k < 3200 ? "v64x128x32_w2x2_s6" : "v64x128x64_w2x2_s6";
        else name = k < 752 ? "v128x128x32_w2x2_s5" : "v128x128x64_w2x2_s5";
      } else if (t128 < 254) {
        name = rows < 75 || t64 < 136 ? "v64x128x64_w2x2_s6" : weight_mb < 121 ? "v128x128x64_w2x2_s5" : "v128x256x64_w2x2_s3";
      } else {
        name = rows < 26 ? "v64x128x64_w2x2_s6" : "v128x256x64_w2x2_s3";
      }
    } else if (k < 888) {
      name = "v128x256x32_w2x2_s3";
    } else if (t256 < 170) {
      if (t128 >= 499) return -1;
      name = "v128x256x64_w2x2_s3";
    } else {
      if (wants_stream(op, rows, weight_mb) || !round_and_a_bit) return -1;
      name = k < 1300 ? "v128x256x32_w2x2_s3" : "v128x256x64_w2x2_s3";
    }
    return variant_by_name(name);
  }
  if (g_live == 1 && k >= 6144 && t256 >= 48 && t256 < 96) return -1;  // one group: the eight-wave 256 x 256 core, all of whose tiles are cut along K
  if (n <= 256 && rows >= 256 && t128 < 160) {
    name = "v64x64x64_w2x2_s5";
  } else if (t128 < 237) {
    if (k < 5480) name = t64 >= 290 ? "v128x128x64_w2x2_s5" : k < 456 ? "v64x128x32_w2x2_s6" : "v64x64x64_w2x2_s5";
    else if (t64x64 < 420) name = x_mb < 11.5 ? "v64x128x64_w2x2_s6" : "v128x128x64_w2x2_s5";
    else name = "v128x256x64_w2x2_s3";
  } else if (t256 < 127) {
    name = k >= 500 ? "v128x256x64_w2x2_s3" : "v128x256x32_w2x2_s3";
  } else if (k < 616) {
    if (k >= 440 && weight_mb >= 107 && rows < 200) return -1;
    name = "v128x256x32_w2x2_s3";
  } else {
    if (wants_stream(op, rows, weight_mb)) return -1;
    // Rounds of 256 x 256 tiles: up to two thirds of one, and a round and a bit, leave those cores' last round mostly empty.
    // From two thirds on (1.10 times the four-wave core's time on 681 calls of 200 to 262 tiles), and of many rounds (1.05 on 1727 of 400
    // to 800), they are ahead, but for groups of a tile's height and a bit with k < 4500, half of whose tall tiles are nearly
    // empty (level: equal groups 0.96, skewed ones 1.04).
    const bool narrow = t256 < 170 || (t256 > 262 && t256 < 400) || (t256 >= 400 && t256 < 800 && k < 4500 && rows >= 250 && rows < 330);
    if (round_and_a_bit) name = k < 1300 ? "v128x256x32_w2x2_s3" : "v128x256x64_w2x2_s3";
    else if ((k >= 1792 && rows < 400 && narrow) || (t256 < 170 && rows < 128)) name = "v128x256x64_w2x2_s3";
    else return -1;
  }
  return variant_by_name(name);
}

// Shape-only default: the largest tile that still gives the 256 compute units enough tiles, from a sweep of all
// compiled variants over a spread of shapes.  One 160 KB work-group of a 256 x 256 core runs per compute unit, so that
// core wants several rounds of tiles or a long contraction; the 128 x 256 ping-pong core (two work-groups per compute
// unit) and the 128 x 128 direct-to-LDS core (three) take over below that, the register-staged tiles for what is smaller still.  A group's expected
// partial tile counts as half a tile.
//
// Where small_tile_variant() names a tile of rd_gemm_ws.h, that one runs.
int default_variant(int op, int m, int k, int n, int g, bool vec) {
  if (!vec) {
    const int any = any_pitch_variant(RD_DTYPE_BF16, op, m, k, n, g);
    return any >= 0 ? any : first_variant_with_vec(0);
  }
  const bool allow_dlds = dlds_fits(op, m, k, n);
  if (allow_dlds) {
    // Among the 256 x 256 cores (all within a few per cent of each other on most shapes): the four-wave core when the
    // launch has many tiles or the groups are much shorter than the tile (only it has the streaming routines for their
    // row tiles); with few tiles its single wave per SIMD hides less, and the eight-wave cores are ahead.  tgmm: the
    // four-wave core when the groups (its contraction) are long.
    const long long g_live = g < m ? g : m;
    int pick = -1;
    const int small_tile = small_tile_variant(op, m, k, n, g);
    if (small_tile >= 0) return small_tile;
    if (op == 2) {
      const long long t256 = (long long)g * cdiv(k, 256) * cdiv(n, 256), t128 = (long long)g * cdiv(k, 128) * cdiv(n, 128);
      if (k >= 256 && n >= 256 && t256 >= 170 && (long long)m >= 1900ll * g) pick = variant_by_name("w256x256x32_w2x2_s5");
      else if (k >= 256 && n >= 256 && (long long)m > 64ll * g && (t256 >= 16384 || (m >= 128ll * g && t256 >= 170))) pick = variant_by_name("p256x256x32_w2x4_s4");
      else if (k >= 128 && n >= 128 && t128 >= 64) pick = variant_by_name("d128x128x32_w2x2_s3");
    } else {
      // k is the contraction length here
      const long long t256 = est_tiles_256(m, n, g), rows128 = cdiv(m, 128) + g_live / 2;
      const long long t128x256 = rows128 * cdiv(n, 256), t128 = rows128 * cdiv(n, 128);
      const bool big = (t256 >= 127 && k >= (op == 1 ? 440 : 888)) ||   // half a round of tiles with a contraction that amortises them (small_tile_variant() has taken what is not)
                       (t256 >= 96 && k >= 3072) ||    // long contraction
                       (t256 >= 128 && (long long)m <= 64ll * g);  // groups far shorter than any tile: the tall tile costs nothing
      const double rows = (double)m / g_live, weight_mb = 2e-6 * (double)g_live * k * n;
      if (n >= 256 && m >= 256 && big) {
        // the four-wave core for groups that need the streaming routines; else gmm: the eight-wave one with a ring per operand, up
        // to 10 % ahead on a round or more of tiles, unless the weights are few (38 MB: 5 %); trans_rhs: the four-wave core's
        // register-staged form from a contraction of 1792 on, the eight-wave one below (10 %)
        const bool w4 = wants_stream(op, rows, weight_mb) ||
                        (op == 1 ? k >= 1792
                                 : (t256 >= 170 && weight_mb < 38) || (t256 >= 100 && t256 < 170 && m >= 1024 && rows >= 400));
        // trans_rhs, groups of under 16 rows on average: the 64 x 64 tile of rd_gemm_ws.h, five slabs of 64 to a work-group and four times the work-groups, where
        // the weights' pitch does not make its tiles start in the same memory channels (kRotatePitch: only the streaming routines spread their
        // starts).  Time over theirs on weights from HBM 0.945 (2876 random calls, nine in ten under 1.03), 0.79-0.86 on weights in the last-level cache; at
        // those pitches 1.01, of 16 to 32 rows 1.01, of 32 to 64 1.13.  us: 835 x 3440 x 832 in 73 groups 150 | 82 (in cache).
        if (op == 1 && rows < 16 && k % rd::kRotatePitch != 0) pick = variant_by_name("v64x64x64_w2x2_s5");
        else pick = variant_by_name(w4 ? "w256x256x32_w2x2_s5" : "q256x256x32_w2x4");
      } else if (op == 1 && n >= 256 && m >= 256 && t256 >= 48 && k >= 6144) {
        // trans_rhs, a long contraction and less than a round of 256 x 256 tiles: the eight-wave core, whose tiles are all
        // cut along K (512 x 8192 x 8192 in one group: 99 us against 125-134 for the 128-row cores)
        pick = variant_by_name("p256x256x32_w2x4_s4");
      } else if (n >= 256 && m >= 128 && t128x256 >= 96) pick = variant_by_name("p128x256x32_w2x4_s3");
      else if (n >= 128 && m >= 128 && t128 >= 96) pick = variant_by_name("d128x128x32_w2x2_s3");
    }
    if (pick >= 0) return pick;
  }
  // Register-staged tiles, largest first: the first that is no taller than a group's slab calls for and still gives
  // about one tile per compute unit; failing that, the one with the most tiles.
  const int out_rows = op == 2 ? k : (g > 0 ? m / g : m);  // rows of one group's output slab
  const int bm_pref = out_rows >= 96 ? 128 : out_rows >= 48 ? 64 : 32;
  const int bn_pref = n >= 192 ? 256 : n >= 96 ? 128 : 64;
  static const int shapes[][2] = {{128, 256}, {128, 128}, {64, 256}, {32, 256}, {64, 64}};
  int most = -1;
  long long most_tiles = -1;
  for (const auto& sh : shapes) {
    if (sh[0] > bm_pref || sh[1] > bn_pref) continue;
    const int id = find_variant(sh[0], sh[1], 1, false);
    if (id < 0) continue;
    const long long row_tiles = op == 2 ? (long long)g * cdiv(k, sh[0]) : cdiv(m, sh[0]) + (g < m ? g : m) / 2;
    const long long tiles = row_tiles * cdiv(n, sh[1]);
    if (tiles >= 200) return id;
    if (tiles > most_tiles) { most_tiles = tiles; most = id; }
  }
  if (most >= 0) return most;
  for (int i = 0; i < kNumVariants; ++i)
    if (kVariantGetters[i]()->vec == 1 && !kVariantGetters[i]()->dlds && kVariantGetters[i]()->dtype == RD_DTYPE_BF16) return i;
  return first_variant_with_vec(0);
}

// a, b, c: the three tensors of the call with their element counts na, nb, nc; a tensor without elements may be null.
int check_common(const void* a, long long na, const void* b, long long nb, const void* c, long long nc,
                 const int32_t* gs, int m, int k, int n, int g, int dtype) {
  if (m < 0 || k < 0 || n < 0 || g < 1) return fail(RD_ERR_INVALID_ARGUMENT, "bad shape m=%d k=%d n=%d g=%d", m, k, n, g);
  if (dtype < RD_DTYPE_BF16 || dtype > RD_DTYPE_F16) return fail(RD_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (first_variant_of_dtype(dtype) < 0) return fail(RD_ERR_UNSUPPORTED, "no kernel for dtype %d compiled in", dtype);
  // the float32 tile routines address one slab with 32-bit element offsets: up to 128 rows of pitch k or n
  if (dtype != RD_DTYPE_BF16 && (k >= (1 << 24) || n >= (1 << 24)))
    return fail(RD_ERR_UNSUPPORTED, "float32: k=%d or n=%d beyond 2^24", k, n);
  if (!gs || (!a && na > 0) || (!b && nb > 0) || (!c && nc > 0)) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if ((long long)g * k * n >= (1ll << 40)) return fail(RD_ERR_INVALID_ARGUMENT, "g*k*n too large");
  return RD_OK;
}

// Whether tile shape v computes product op (0 gmm, 1 gmm with trans_rhs, 2 tgmm) of this size.  vec: 16-byte pitches and
// addresses.
int variant_takes(const rd::TileVariant* v, int op, int m, int k, int n, int dtype, bool vec) {
  if (v->dtype != dtype) return fail(RD_ERR_UNSUPPORTED, "variant %s does not take dtype %d", v->name, dtype);
  if (v->vec && !vec) return fail(RD_ERR_UNSUPPORTED, "variant %s needs k %% 8 == 0, n %% 8 == 0 and 16-byte aligned buffers", v->name);
  if (v->any_pitch_core && !any_pitch_core_fits(dtype, k, n)) return fail(RD_ERR_UNSUPPORTED, "variant %s needs k >= 8, n >= 8 and 256 rows within 2 GiB", v->name);
  if (v->dlds && !dlds_fits(op, m, k, n)) return fail(RD_ERR_UNSUPPORTED, "variant %s: operand window of one tile exceeds 2 GiB", v->name);
  if (op == 2 ? !v->tgmm : !(op == 1 ? v->gmm_nt : v->gmm_nn))
    return fail(RD_ERR_UNSUPPORTED, "variant %s has no %s kernel", v->name, op == 2 ? "tgmm" : op == 1 ? "gmm trans_rhs" : "gmm");
  if (v->dlds && dtype == RD_DTYPE_F8E4M3_BF16 && (k % 16 != 0 || (op != 1 && n % 16 != 0)))
    return fail(RD_ERR_UNSUPPORTED, "variant %s needs 16-byte row pitches: k %% 16 == 0 (and n %% 16 == 0 unless the weights are stored [g, n, k])", v->name);
  return RD_OK;
}

struct MapSpace {
  int32_t *group_offsets, *tile2group, *tile2it, *total, *tile2band;
};

size_t map_bytes(int U, int g) { return align_up(((size_t)g + 3 * (size_t)U + 1) * sizeof(int32_t), 256); }

constexpr int kWsCutMinK = 5700;
// Launches of 256 x 256 tiles whose last round may be cut (split_parts_by_gain()) have the map built for contractions of 6400 and more, and
// below where the expected last round would be cut with this many tiles more in it: the sizes decide, and the map is 4 us for
// nothing where they leave it uncut (built for every k from 2500 on: 180 calls of 2500 to 3500 indices with more than 50 tiles in
// the expected last round took 1.02-1.07 times as long as without, 3500 to 6400 with more than 110 1.00-1.05; with fewer 0.90-1.0).
constexpr int kCutDoubt = 16;

// Whether the core of rd_gemm_ws.h reads the weights of groups of one row tile past the caches: where they are more than the 256 MB
// of the last-level cache hold, the groups average less than a tile's 128 rows, and the weights' rows are whole 128-byte lines (a
// line that two tiles share, or the two halves of one that 32-wide slabs of K-major weights read, would be fetched twice; those
// have no such kernel).  Time without over time with, geometric means of 508 random forward and 144 trans_rhs calls that the
// rule takes: 1.07 and 1.07 on weights that were in use, 1.06 and 1.06 on cold ones, 1.18 and 1.10 on weights just written, whose dirty
// lines the cache would have to write back first (0.83 at worst: groups of 96 to 128 rows whose weights are a little more than
// the cache holds).  2048 x 768 x 2048 in 128 groups: 74 | 68, 76 | 71 and 97 | 74 us (the four-wave 256 x 256 core 84, 88 and 91).
// With 200 to 256 MB of weights 0.92, 1.03 and 1.01; forward products with rows of no whole lines 1.00, 0.99 and 1.04, trans_rhs ones 0.94, 0.93
// and 0.88, with 32-wide slabs 0.77, 0.78 and 0.89; groups of 128 to 200 rows level.
constexpr double kStreamWeightBytes = 300e6;
bool streams_weights(int m, int k, int n, int groups, int trans_rhs) {
  return 2.0 * groups * k * n >= kStreamWeightBytes && (long long)m < 128ll * groups && (trans_rhs ? k : n) % 64 == 0;
}
constexpr size_t kBlockOrderBytes = (size_t)64 << 10;
constexpr int kLongGroupRows = 128;  // groups with more rows than this have matrix-core-bound tiles (the streaming routines serve up to 128)
constexpr size_t kDecodePartialBytes = (size_t)64 << 20;  // header + fp32 partial sums of the whole-row streaming kernel
size_t split_bytes(const rd::TileVariant* v) {
  return align_up(kSplitSlots * sizeof(int32_t), 256) + (size_t)kSplitSlots * v->bm * v->split_bn * sizeof(float);
}

// Compute units of the current device, looked up once per device.
int num_compute_units() {
  static std::atomic<int> cached[64];  // zero-initialised; racing threads store the same value
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return kSplitSlots;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = kSplitSlots;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int carve(void* ws, size_t ws_bytes, int U, int g, MapSpace* out) {
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 3) != 0) return fail(RD_ERR_WORKSPACE, "workspace null or misaligned");
  if (ws_bytes < map_bytes(U, g)) return fail(RD_ERR_WORKSPACE, "workspace %zu B < %zu B needed", ws_bytes, map_bytes(U, g));
  int32_t* p = static_cast<int32_t*>(ws);
  out->group_offsets = p;
  out->tile2group = p + g;
  out->tile2it = p + g + U;
  out->total = p + g + 2 * U;
  out->tile2band = p + g + 2 * U + 1;
  return RD_OK;
}

// vec: rows and buffers start on 16-byte boundaries.
int default_plan(int op, int m, int k, int n, int g, int dtype, bool vec, rd_plan* out) {
  if (!out || op < 0 || op > 2) return fail(RD_ERR_INVALID_ARGUMENT, "bad op %d or null plan", op);
  if (dtype < RD_DTYPE_BF16 || dtype > RD_DTYPE_F16) return fail(RD_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  out->variant = dtype == RD_DTYPE_F32 ? default_f32_variant(op, m, k, n, g)
               : dtype >= RD_DTYPE_F32_BF16 ? default_cvt_variant(dtype, op, m, k, n, g, vec) : default_variant(op, m, k, n, g, vec);
  out->group_m = 0;
  out->group_n = 0;
  out->decode_nb = 0;
  out->split_k = 0;
  if (op != 2 && out->variant >= 0) {
    const rd::TileVariant* v = kVariantGetters[out->variant]();
    default_walk(m, k, n, g, v, &out->group_m, &out->group_n);
  }
  const long long few_tiles = (long long)(g < m ? g : m) * cdiv(n, 256) <= 512;
  if (dtype == RD_DTYPE_F8E4M3_BF16) {
    // float8 has the streaming kernel for weights stored [g, n, k] only.  Widening the bytes costs instructions: up to
    // one row per group on average (4 rows per pass) it is ahead of the tile kernels (128 experts of 2048 x 768, m = 64:
    // 20.8 against 27.3 us, m = 128: 26.3 against 33.1), with 8 rows per pass level with them (m = 256: 49.2 against 50.0).
    if (op == 1 && vec && k % 16 == 0 && g > 0 && few_tiles && m <= g && m <= 1024 &&
        rd::gmm_rows_t_fits(m, k, n, g, true) && (long long)k * n < (1ll << 31))
      out->decode_nb = RD_DECODE_ROWS;
  }
  if (dtype != RD_DTYPE_BF16 && dtype != RD_DTYPE_F16)
    return out->variant >= 0 ? RD_OK : fail(RD_ERR_UNSUPPORTED, "no kernel for dtype %d compiled in", dtype);
  // A few rows per group: the streaming kernels.  Whole-row slices (n <= 2048) take 4 rows of a group per pass over its
  // weights up to one row per group on average and 8 rows per pass beyond; with top-8 routing over 128 experts, 4 rows
  // per group on average still leaves every group within one pass (75 us against 76-79 for the tile kernels at
  // m = 512, k = 2048, n = 768; 66 against 72 at m = 256).  The column-strip kernel holds 4 rows per pass.
  // They win where the tile kernels have too few tiles to fill the device - at most two rounds of 256-column tiles of the
  // non-empty groups, of which there are at most min(g, m); with more tiles than that (256 experts of 7168 x 2048: 8 tiles
  // each) the tile kernels' streaming routines run at 7 TB/s and a second pass over any group's weights is what decides.
  if (op == 0 && vec && g > 0 && few_tiles && m <= (n <= 2048 ? 4 * g : g) && m <= 1024 && k <= rd::kDecodeMaxK &&
      (long long)k * n < (1ll << 31))
    out->decode_nb = n <= 2048 ? RD_DECODE_ROWS : 64;
  // the same with weights stored [g, n, k]: the stream is cut along n and needs no workspace
  if (op == 1 && vec && g > 0 && few_tiles && m <= 4 * g && m <= 1024 && rd::gmm_rows_t_fits(m, k, n, g) && (long long)k * n < (1ll << 31))
    out->decode_nb = RD_DECODE_ROWS;
  return out->variant >= 0 ? RD_OK : fail(RD_ERR_UNSUPPORTED, "no tile variant compiled in");
}

}  // namespace

extern "C" {

int rd_abi_version(void) { return RD_ABI_VERSION; }
const char* rd_last_error(void) { return g_err; }
int rd_num_variants(void) { return kNumVariants; }

int rd_get_variant(int id, rd_variant_info* out) {
  if (id < 0 || id >= kNumVariants || !out) return fail(RD_ERR_INVALID_ARGUMENT, "variant id %d out of range", id);
  const rd::TileVariant* v = kVariantGetters[id]();
  memset(out, 0, sizeof(*out));
  out->id = id;
  out->tile_m = v->bm; out->tile_n = v->bn; out->tile_k = v->bk;
  out->waves_m = v->waves_m; out->waves_n = v->waves_n;
  out->vec = v->vec;
  out->dtype = v->dtype;
  out->direct_to_lds = v->dlds;
  out->stages = v->stages;
  strncpy(out->name, v->name, sizeof(out->name) - 1);
  return RD_OK;
}

int rd_variant_takes(int id, int op, int m, int k, int n, int dtype) {
  if (id < 0 || id >= kNumVariants) return fail(RD_ERR_INVALID_ARGUMENT, "variant id %d out of range", id);
  if (op < 0 || op > 2 || m < 0 || k < 0 || n < 0) return fail(RD_ERR_INVALID_ARGUMENT, "bad op %d or shape m=%d k=%d n=%d", op, m, k, n);
  return variant_takes(kVariantGetters[id](), op, m, k, n, dtype, dtype != RD_DTYPE_F32 && k % 8 == 0 && n % 8 == 0);
}

int rd_default_plan(int op, int m, int k, int n, int g, int dtype, rd_plan* out) {
  return default_plan(op, m, k, n, g, dtype, k % 8 == 0 && n % 8 == 0, out);
}

int rd_default_plan_any_address(int op, int m, int k, int n, int g, int dtype, rd_plan* out) {
  return default_plan(op, m, k, n, g, dtype, false, out);
}

int rd_sched_map_len(int m, int g, int chunk_m) {
  if (m < 0 || g < 0 || chunk_m < 1) return fail(RD_ERR_INVALID_ARGUMENT, "bad m=%d g=%d chunk_m=%d", m, g, chunk_m);
  return cdiv(m, chunk_m) + g;
}

int rd_sched_map(void* stream, const int32_t* group_sizes, int g, int m, int chunk_m, int32_t* group_offsets,
                 int32_t* row_it2group, int32_t* row_it2it_in_group, int32_t* total_row_its) {
  if (g < 1 || m < 0 || chunk_m < 1) return fail(RD_ERR_INVALID_ARGUMENT, "bad g=%d m=%d chunk_m=%d", g, m, chunk_m);
  if (!group_sizes || !group_offsets || !row_it2group || !row_it2it_in_group || !total_row_its)
    return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  const int rc = rd::launch_sched_map((hipStream_t)stream, group_sizes, g, m, chunk_m, group_offsets, row_it2group,
                                      row_it2it_in_group, total_row_its);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "sched_map launch");
}

size_t rd_gmm_workspace_bytes(int m, int g, const rd_plan* plan) {
  if (m < 0 || g < 0) return 0;
  // the scheduling map for the smallest tile height, and room for the interleaved order of the walk's blocks (one word
  // per block of tiles; without it the blocks are dealt in walk order)
  const size_t map = map_bytes(cdiv(m, kMinTileM) + g, g) + kBlockOrderBytes;
  if (plan && plan->decode_nb == RD_DECODE_ROWS) return map + kDecodePartialBytes;
  if (plan && (plan->split_k < 0 || plan->decode_nb > 0)) return map;
  // room for the K-split partial sums of the planned variant, or of the largest one when the library is to choose
  size_t split = 0;
  for (int i = 0; i < kNumVariants; ++i) {
    const rd::TileVariant* v = kVariantGetters[i]();
    if (!v->splitk || (plan && plan->variant >= 0 && plan->variant != i)) continue;
    // (a whole tile a slot, also where the pieces are of half a tile and the launch asks for half of it)
    const size_t whole_tiles = split_bytes(v) + (size_t)kSplitSlots * v->bm * (v->bn - v->split_bn) * sizeof(float);
    if (whole_tiles > split) split = whole_tiles;
  }
  return map + split;
}

}  // extern "C"

namespace {

// A holds the g_local groups [g_first, g_first + g_local) of the g groups in group_sizes.  may_cut: false where the workspace
// is not the call's own, so that the K-split stays off whatever its size and the plan say.
int gmm_impl(void* stream, const void* x, const void* A, const int32_t* group_sizes, void* y, int m, int k, int n,
             int g, int g_first, int g_local, int trans_rhs, int dtype, const rd_plan* plan, void* workspace,
             size_t workspace_bytes, bool may_cut = true) {
  int rc = check_common(x, (long long)m * k, A, (long long)(g_local > 0 ? g_local : 0) * k * n, y, (long long)m * n, group_sizes, m, k, n, g, dtype);
  if (rc != RD_OK) return rc;
  if (g_first < 0 || g_local < 1 || (long long)g_first + g_local > g)
    return fail(RD_ERR_INVALID_ARGUMENT, "groups [%d, %d + %d) are not within the %d of group_sizes", g_first, g_first, g_local, g);
  const bool whole = g_first == 0 && g_local == g;
  if (m == 0 || n == 0) return RD_OK;
  hipStream_t s = (hipStream_t)stream;
  if (k == 0) {  // an empty contraction: every output element is zero
    rc = rd::launch_zero_bytes(s, y, (size_t)m * n * out_elem_bytes(dtype));
    return rc == hipSuccess ? RD_OK : hip_fail(rc, "zero fill");
  }
  const bool f8 = dtype == RD_DTYPE_F8E4M3_BF16;
  // bfloat16 and float16 have the streaming kernels, float8 the one for weights stored [g, n, k]; the other types have
  // their own tile shapes
  const bool half = dtype == RD_DTYPE_F16;
  const bool f32 = dtype != RD_DTYPE_BF16 && !half && !(f8 && trans_rhs);
  const bool vec = dtype != RD_DTYPE_F32 && vec_ok(x, A, y, k, n);

  rd_plan pl;
  if (plan) pl = *plan; else { pl.variant = -1; pl.group_m = 0; pl.group_n = 0; pl.decode_nb = 0; pl.split_k = 0; }
  if (!plan) {
    rd_plan d;
    if (rd_default_plan(trans_rhs ? 1 : 0, m, k, n, g, dtype, &d) == RD_OK && vec) pl.decode_nb = d.decode_nb;
  }

  if (f32) pl.decode_nb = 0;
  if (!whole) {  // the streaming kernels serve all groups only
    if (plan && plan->decode_nb != 0) return fail(RD_ERR_UNSUPPORTED, "the streaming kernels take all groups: no group_offset");
    pl.decode_nb = 0;
  }
  if (f8 && pl.decode_nb != 0 && pl.decode_nb != RD_DECODE_ROWS) {
    if (plan && plan->decode_nb != 0) return fail(RD_ERR_UNSUPPORTED, "float8 operands have no column-strip streaming kernel");
    pl.decode_nb = 0;
  }
  if (pl.decode_nb == RD_DECODE_ROWS && trans_rhs) {
    if (!vec || (f8 && k % 16 != 0) || !rd::gmm_rows_t_fits(m, k, n, g, f8) || (long long)k * n >= (1ll << 31))
      return fail(RD_ERR_UNSUPPORTED, "the trans_rhs streaming kernel needs 16-byte pitches, k <= 8192 and k * n < 2^31");
    rd::DecodeArgs a{(const uint16_t*)x, (const uint16_t*)A, (uint16_t*)y, group_sizes, m, k, n, g, half ? 1 : 0};
    rc = rd::launch_gmm_rows_t(s, a, num_compute_units(), f8);
    return rc == hipSuccess ? RD_OK : hip_fail(rc, "gmm_rows_t launch");
  }
  if (pl.decode_nb == RD_DECODE_ROWS) {
    // whole-row slices need room for at least one layer of fp32 partial sums; without it, or for very wide outputs,
    // the column-strip kernel does the job
    const bool fits = vec && !trans_rhs && n <= 2048 && k > 0 && (long long)k * n < (1ll << 31) && workspace &&
                      (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                      workspace_bytes >= rd::gmm_rows_workspace_bytes(m, n, 1);
    if (fits) {
      rd::DecodeArgs a{(const uint16_t*)x, (const uint16_t*)A, (uint16_t*)y, group_sizes, m, k, n, g, half ? 1 : 0};
      rc = rd::launch_gmm_rows(s, a, num_compute_units(), workspace, workspace_bytes);
      return rc == hipSuccess ? RD_OK : hip_fail(rc, "gmm_rows launch");
    }
    pl.decode_nb = 64;
  }
  if (pl.decode_nb > 0) {
    if (trans_rhs) return fail(RD_ERR_UNSUPPORTED, "the column-strip streaming kernel has no trans_rhs form (decode_nb = RD_DECODE_ROWS has)");
    if (!vec || k > rd::kDecodeMaxK || k == 0 || (long long)k * n >= (1ll << 31))
      return fail(RD_ERR_UNSUPPORTED, "streaming kernel needs 16-byte pitches, 0 < k <= %d and k * n < 2^31", rd::kDecodeMaxK);
    rd::DecodeArgs a{(const uint16_t*)x, (const uint16_t*)A, (uint16_t*)y, group_sizes, m, k, n, g, half ? 1 : 0};
    rc = rd::launch_gmm_decode(s, a, pl.decode_nb);
    return rc == hipSuccess ? RD_OK : hip_fail(rc, "gmm_decode launch");
  }

  const int op = trans_rhs ? 1 : 0;
  int vid = pl.variant >= 0 ? pl.variant
          : dtype == RD_DTYPE_F32 ? default_f32_variant(op, m, k, n, g)
          : dtype >= RD_DTYPE_F32_BF16 ? default_cvt_variant(dtype, op, m, k, n, g, vec) : default_variant(op, m, k, n, g, vec);
  if (vid < 0 || vid >= kNumVariants) return fail(RD_ERR_INVALID_ARGUMENT, "variant %d out of range", vid);
  const rd::TileVariant* v = kVariantGetters[vid]();
  rc = variant_takes(v, op, m, k, n, dtype, vec);
  if (rc != RD_OK) return rc;
  if (dtype == RD_DTYPE_F32 && vid == f32_tiles().single.id && (pl.variant < 0 || pl.split_k == 0 || !may_cut)) {
    // the same bits either way, so the workspace may say which; with room for its pieces the launch may cut
    const bool cut = may_cut && pl.split_k >= 0 && workspace_bytes >= map_bytes(cdiv(m, v->bm) + g, g) + split_bytes(v);
    if (pairs_f32_tiles(m, k, n, g, cut)) v = f32_tiles().pair.v;
  }

  const int U = cdiv(m, v->bm) + g;
  MapSpace ms;
  rc = carve(workspace, workspace_bytes, U, g, &ms);
  if (rc != RD_OK) return rc;
  // The K-split is an optimisation: it is used when the variant has it, the plan does not forbid it and the workspace
  // has the room rd_gmm_workspace_bytes() asks for; otherwise every tile is computed whole.
  const size_t map_sz = map_bytes(U, g);
  const bool split = may_cut && v->splitk && pl.split_k >= 0 && workspace_bytes >= map_sz + split_bytes(v) &&
                     (reinterpret_cast<uintptr_t>(workspace) & 15) == 0;
  int32_t* counters = split ? reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + map_sz) : nullptr;
  // The interleaved order of the walk's blocks (long groups' among short groups') is an optimisation too: built when the
  // launch has several rounds of tiles and the workspace has room for it behind what the K-split takes.
  const size_t order_at = map_sz + (split ? split_bytes(v) : 0);
  // tile walk: bands of at most group_m row tiles, blocks of group_m x group_n positions (32 by default: what one XCD
  // runs at a time with one work-group per compute unit)
  const int n_tiles = cdiv(n, v->bn);
  int group_m = 0, group_n = 0;
  default_walk(m, k, n, g, v, &group_m, &group_n);
  if (pl.group_m > 0) { group_m = pl.group_m; group_n = pl.group_n > 0 ? pl.group_n : (32 / group_m > 0 ? 32 / group_m : 1); }
  else if (pl.group_n > 0) group_n = pl.group_n;
  if (group_m > rd::kBandMaxRows || (long long)group_m * group_n > 4096)
    return fail(RD_ERR_INVALID_ARGUMENT, "tile walk group_m=%d (1..%d) x group_n=%d beyond 4096 positions per block", group_m, rd::kBandMaxRows, group_n);
  if ((long long)U * n_tiles + (long long)16 * group_m * group_n + 8 >= (1ll << 30) || U >= (1 << 23))
    return fail(RD_ERR_UNSUPPORTED, "more than 2^30 tile slots (m=%d n=%d g=%d with tile %d x %d)", m, n, g, v->bm, v->bn);
  const long long slots = (long long)U * n_tiles, per_block = (long long)group_m * group_n;
  const long long n_blocks = (slots + per_block - 1) / per_block;
  // (Rounds of expected tiles - a group's partial last one counts as half - not of the slots they may take.  Groups shorter than
  // half a tile come out too few that way, so a launch of up to twice the four rounds may do without.  Over 900 random calls on
  // which the two counts differ the map cost 1.06 times the time without it (groups of equal, softmax and skewed sizes 1.05, 1.06,
  // 1.07; 1.02 where the launch takes 300 us and more), 4 % was the most that the order gained: 5499 x 7376 x 7168 in 25 skewed groups,
  // trans_rhs, 901 | 866.)
  const long long expected = ((long long)cdiv(m, v->bm) + (g < m ? g : m) / 2) * n_tiles;
  const bool interleave = whole && expected >= 4ll * kSplitSlots && n_blocks <= rd::kMaxOrderedBlocks &&
                          workspace_bytes >= order_at + (size_t)(n_blocks + 2) * sizeof(int32_t);
  int32_t* block_order = interleave ? reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + order_at) : nullptr;
  // The cores with streaming routines for short row tiles (the four-wave 256 x 256 ones): when the K-split is on for
  // this contraction length, the scheduling-map kernel may move the short last tiles of long groups into the last round
  // (it decides from the group sizes; launch_sched_map).  The round size and the piece limit are those of split_plan().
  const long long k_cost = (long long)k * v->split_quarters / 4;
  const bool cut_by_k = k_cost >= 6400 || (v->split_by_gain && expected % kSplitSlots > 0 && expected % kSplitSlots + kCutDoubt < kSplitSlots &&
                                           split_parts_for(v, expected + kCutDoubt, k) >= 2);
  const bool defer = split && v->bm == 256 && std::strstr(v->name, "w256x256x32_w2x2") != nullptr &&
                     (pl.split_k > 0 ? pl.split_k >= 2 : cut_by_k) && k >= 2 * 512;
  const int split_cus = imin_host(num_compute_units(), kSplitSlots);
  // The map is built by a kernel of its own where the launch needs more than each work-group can look up for itself
  // (rd_lookup.h): the interleaved block order, cleared K-split counters (may_split: where split_plan() would cut the expected
  // launch, or the caller asks for it), or more groups than a wave scans.  It is built for a plan that says something about the cut
  // itself too, cut or not: so the tests compare the two ways, and read the map out of the workspace.  (No other caller is
  // promised the map, and one that sets split_k to -1 pays the kernel's 4-8 us, rd_gmm_noalloc with a plan among them.)
  // A cut makes at least two pieces of a tile, so with kSplitSlots slots it needs a last round of at most 128 tiles.  The cores
  // of rd_gemm_ws.h are mostly asked for less than a round: with more tiles than that, and a shorter contraction than
  // kWsCutMinK, the map kernel would be for nothing (1166 x 2320 x 1904 in 7: 28 -> 32 us; 6406 x 5744 x 288 in 85: 103 -> 98).
  const bool few = !v->ws_core || k >= kWsCutMinK || expected <= kSplitSlots / 2 + 12;
  const bool may_split = split && (pl.split_k > 0 ? pl.split_k >= 2 : cut_by_k && few) && k >= 2 * v->split_min_k;
  const bool mapped = interleave || may_split || pl.split_k != 0 || g > rd::kLookupGroups;
  const rd::SplitRule cut{k, (int)k_cost, v->split_min_k, may_split ? kSplitSlots : 0, split_cus, pl.split_k > 0 ? pl.split_k : 0, v->split_by_gain != 0};
  if (mapped) {
    rc = rd::launch_sched_map(s, group_sizes, g, m, v->bm, ms.group_offsets, ms.tile2group, ms.tile2it, ms.total,
                              counters, kSplitSlots, ms.tile2band, group_m, block_order, interleave ? (int)n_blocks : 0,
                              (int)per_block, n_tiles, kLongGroupRows, nullptr, 0, 0, defer ? kLongGroupRows : 0, cut);
    if (rc != hipSuccess) return hip_fail(rc, "sched_map launch");
  }

  rd::GmmArgs a;
  a.counters = counters;
  const bool pieces = split && may_split;
  a.partials = pieces ? reinterpret_cast<float*>(static_cast<char*>(workspace) + map_sz + align_up(kSplitSlots * sizeof(int32_t), 256)) : nullptr;
  a.split_slots = pieces || (split && v->split_bn < v->bn) ? kSplitSlots : 0;  // halves of the last round's tiles need no map
  a.max_parts = pl.split_k > 0 ? pl.split_k : 0;
  a.num_cus = split ? split_cus : kSplitSlots;
  a.main_grid = 0;
  a.x = x; a.A = A; a.y = y;
  a.group_sizes = group_sizes; a.group_offsets = ms.group_offsets;
  a.tile2group = ms.tile2group; a.tile2it = ms.tile2it; a.total_tiles = mapped ? ms.total : nullptr; a.tile2band = ms.tile2band;
  a.m = m; a.k = k; a.n = n; a.g = g;
  a.g_first = g_first; a.g_local = g_local;
  a.U = U; a.n_tiles = n_tiles;
  a.group_m = group_m; a.group_n = group_n;
  a.block_order = block_order; a.n_blocks = interleave ? (int)n_blocks : 0;
  const rd::gmm_launch_fn stream_fn = trans_rhs ? v->gmm_nt_stream : v->gmm_nn_stream;
  const bool streams = stream_fn && streams_weights(m, k, n, imin_host(g_local, m), trans_rhs);
  rc = streams ? stream_fn(s, a) : trans_rhs ? v->gmm_nt(s, a) : v->gmm_nn(s, a);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "gmm launch");
}

// Scratch memory of rd_gmm_noalloc(): one copy per device, held until the process ends.  The name below is only a
// host-side handle; the device address is looked up per device with hipGetSymbolAddress() and kept in g_scratch_ptr.
constexpr size_t kScratchBytes = (size_t)4 << 20;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];
constexpr int kMaxDevices = 64;
std::atomic<void*> g_scratch_ptr[kMaxDevices];  // zero-initialised; racing threads store the same address

// Device address of the current device's copy of `scratch`, or null with the error text set.
void* scratch_of_current_device() {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) { hip_fail((int)e, "hipGetDevice"); return nullptr; }
  if (dev < 0 || dev >= kMaxDevices) { fail(RD_ERR_UNSUPPORTED, "device ordinal %d beyond %d", dev, kMaxDevices - 1); return nullptr; }
  void* p = g_scratch_ptr[dev].load(std::memory_order_acquire);
  if (!p) {
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p) { hip_fail((int)e, "hipGetSymbolAddress(scratch)"); return nullptr; }
    g_scratch_ptr[dev].store(p, std::memory_order_release);
  }
  return p;
}

}  // namespace

extern "C" {

int rd_gmm(void* stream, const void* x, const void* A, const int32_t* group_sizes, void* y, int m, int k, int n,
           int g, int trans_rhs, int dtype, const rd_plan* plan, void* workspace, size_t workspace_bytes) {
  return gmm_impl(stream, x, A, group_sizes, y, m, k, n, g, 0, g, trans_rhs, dtype, plan, workspace, workspace_bytes);
}

int rd_gmm_sharded(void* stream, const void* x, const void* A, const int32_t* group_sizes, void* y, int m, int k, int n,
                   int g_total, int group_offset, int g_local, int trans_rhs, int dtype, const rd_plan* plan,
                   void* workspace, size_t workspace_bytes) {
  return gmm_impl(stream, x, A, group_sizes, y, m, k, n, g_total, group_offset, g_local, trans_rhs, dtype, plan, workspace,
                  workspace_bytes);
}

size_t rd_gmm_noalloc_scratch_bytes(void) { return kScratchBytes; }

int rd_gmm_noalloc(void* stream, const void* x, const void* A, const int32_t* group_sizes, void* y, int m, int k, int n,
                   int g, int trans_rhs, int dtype, const rd_plan* plan) {
  if (m < 0 || g < 1) return fail(RD_ERR_INVALID_ARGUMENT, "bad shape m=%d g=%d", m, g);
  // The scheduling map must fit whatever tile height the plan resolves to; the K-split is forbidden - the partial sums of the
  // smallest float32 tile are 4 MiB, about what the scratch holds - and the whole-row streaming kernel takes as many pieces as
  // the scratch has room for.
  rd_plan pl;
  if (plan) pl = *plan; else { pl.variant = -1; pl.group_m = 0; pl.group_n = 0; pl.decode_nb = 0; pl.split_k = 0; }
  pl.split_k = -1;
  const size_t need = rd_gmm_workspace_bytes(m, g, &pl);
  if (need > kScratchBytes && !(pl.decode_nb == RD_DECODE_ROWS && map_bytes(cdiv(m, kMinTileM) + g, g) <= kScratchBytes))
    return fail(RD_ERR_WORKSPACE, "rd_gmm_noalloc: m=%d g=%d needs %zu B of scratch, the built-in buffer has %zu B; use rd_gmm with a workspace",
                m, g, need, kScratchBytes);
  void* ws = scratch_of_current_device();
  if (!ws) return RD_ERR_HIP;
  // a caller without a plan gets the library default (streaming kernel for a few rows per group) like rd_gmm's
  return gmm_impl(stream, x, A, group_sizes, y, m, k, n, g, 0, g, trans_rhs, dtype, plan ? &pl : nullptr, ws, kScratchBytes, /*may_cut*/ false);
}

size_t rd_tgmm_workspace_bytes(int m, int g, const rd_plan* plan) {
  (void)plan; (void)m;
  if (g < 0) return 0;
  // the row offsets, and the order in which the launch visits the groups (a record of four words each; without room
  // for it the groups are visited as they come)
  return map_bytes(g + 1, g) + align_up((size_t)g * 4 * sizeof(int32_t), 256);
}

}  // extern "C"

namespace {

// dA holds the slices of the g_local groups [g_first, g_first + g_local) of the g groups in group_sizes.
int tgmm_impl(void* stream, const void* x, const void* dy, const int32_t* group_sizes, void* dA, int m, int k, int n,
              int g, int g_first, int g_local, int dtype, const rd_plan* plan, void* workspace, size_t workspace_bytes) {
  int rc = check_common(x, (long long)m * k, dy, (long long)m * n, dA, (long long)(g_local > 0 ? g_local : 0) * k * n, group_sizes, m, k, n, g, dtype);
  if (rc != RD_OK) return rc;
  if (g_first < 0 || g_local < 1 || (long long)g_first + g_local > g)
    return fail(RD_ERR_INVALID_ARGUMENT, "groups [%d, %d + %d) are not within the %d of group_sizes", g_first, g_first, g_local, g);
  if (k == 0 || n == 0) return RD_OK;
  hipStream_t s = (hipStream_t)stream;
  if (m == 0) {  // no rows: every group is empty and its slice is zero
    rc = rd::launch_zero_bytes(s, dA, (size_t)g_local * k * n * out_elem_bytes(dtype));
    return rc == hipSuccess ? RD_OK : hip_fail(rc, "zero fill");
  }
  const bool vec = dtype != RD_DTYPE_F32 && vec_ok(x, dy, dA, k, n);
  const int group_m = plan && plan->group_m > 0 ? plan->group_m : 4;  // 4 and 8 are within 1 % on average; 8 has the worse outliers (128 x 128 tiles, 8 tiles along k: +20 %)
  int vid = plan && plan->variant >= 0 ? plan->variant
          : dtype == RD_DTYPE_F32 ? default_f32_variant(2, m, k, n, g_local)
          : dtype >= RD_DTYPE_F32_BF16 ? default_cvt_variant(dtype, 2, m, k, n, g_local, vec) : default_variant(2, m, k, n, g_local, vec);
  if (vid < 0 || vid >= kNumVariants) return fail(RD_ERR_INVALID_ARGUMENT, "variant %d out of range", vid);
  const rd::TileVariant* v = kVariantGetters[vid]();
  rc = variant_takes(v, 2, m, k, n, dtype, vec);
  if (rc != RD_OK) return rc;

  // Only the row offsets are needed: build the map with a single chunk per group.
  const int chunk = m > 0 ? m : 1;
  const int U = cdiv(m, chunk) + g;
  MapSpace ms;
  rc = carve(workspace, workspace_bytes, U, g, &ms);
  if (rc != RD_OK) return rc;
  const size_t map_sz = map_bytes(U, g);
  // Groups visited by falling size class (plan.group_n = 1; -1 = as they come; 0 = by the rule below).  With long
  // groups of uneven length and a few rounds of tiles the longest groups' tiles otherwise start last and end the
  // launch alone (softmax-sized groups: 40 of 1000 rows on average, k = n = 768: 111 -> 82 us; 30 x 1000 rows, k 2048,
  // n 1024: 144 -> 124 us; -2 % on average over the 46 shapes of the default-plan sweep, 21 of them taken by the rule);
  // with groups much shorter than a tile two groups share an XCD and the order they come in mixes long and short tiles
  // better (DeepSeek-V3 shape: a tuned plan asks for it there), and launches of one round or a few tens of microseconds
  // pay for the extra dependent load per tile.
  const int order_pref = plan ? plan->group_n : 0;
  const long long tgmm_tiles = (long long)g_local * cdiv(k, v->bm) * cdiv(n, v->bn);
  const bool by_size = order_pref == 1 || (order_pref == 0 && g_local >= 3 && (long long)m >= 512ll * g && tgmm_tiles > 256 &&
                                           (double)m * k * n >= 8e9);
  int32_t* group_order = by_size && g_local > 1 && workspace_bytes >= map_sz + (size_t)g_local * 4 * sizeof(int32_t)
                             ? reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + map_sz) : nullptr;
  // in the order the groups come, each work-group adds up the sizes before its group itself (rd_lookup.h)
  const bool mapped = group_order || g > 4 * rd::kLookupGroups;
  if (mapped) {
    rc = rd::launch_sched_map(s, group_sizes, g, m, chunk, ms.group_offsets, ms.tile2group, ms.tile2it, ms.total, nullptr, 0,
                              nullptr, 1, nullptr, 0, 1, 1, 0, group_order, g_first, group_order ? g_local : 0);
    if (rc != hipSuccess) return hip_fail(rc, "sched_map launch");
  }

  rd::TgmmArgs a;
  a.x = x; a.dy = dy; a.dA = dA;
  a.group_sizes = group_sizes; a.group_offsets = mapped ? ms.group_offsets : nullptr;
  a.m = m; a.k = k; a.n = n; a.g = g_local;
  a.g_first = g_first;
  a.k_tiles = cdiv(k, v->bm); a.n_tiles = cdiv(n, v->bn);
  a.group_m = group_m;
  const size_t out_bytes = out_elem_bytes(dtype);
  a.edge_lines = (n * out_bytes % 64 != 0 || (reinterpret_cast<uintptr_t>(dA) & 63) != 0) &&
                 m <= (long long)(out_bytes == 4 ? rd::kEdgeLineRowsF32 : rd::kEdgeLineRows) * g;
  a.group_order = group_order;
  rc = v->tgmm(s, a);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "tgmm launch");
}

}  // namespace

extern "C" {

int rd_tgmm(void* stream, const void* x, const void* dy, const int32_t* group_sizes, void* dA, int m, int k,
            int n, int g, int dtype, const rd_plan* plan, void* workspace, size_t workspace_bytes) {
  return tgmm_impl(stream, x, dy, group_sizes, dA, m, k, n, g, 0, g, dtype, plan, workspace, workspace_bytes);
}

int rd_tgmm_sharded(void* stream, const void* x, const void* dy, const int32_t* group_sizes, void* dA, int m, int k, int n,
                    int g_total, int group_offset, int g_local, int dtype, const rd_plan* plan, void* workspace,
                    size_t workspace_bytes) {
  return tgmm_impl(stream, x, dy, group_sizes, dA, m, k, n, g_total, group_offset, g_local, dtype, plan, workspace, workspace_bytes);
}

int rd_probe_stream_read(void* stream, const void* src, size_t bytes, size_t block_bytes, void* sink) {
  if (!src || (reinterpret_cast<uintptr_t>(src) & 15) != 0 || block_bytes < 16)
    return fail(RD_ERR_INVALID_ARGUMENT, "stream probe: src null or not 16-byte aligned, or block_bytes < 16");
  const int rc = rd::launch_stream_read((hipStream_t)stream, src, bytes, block_bytes, sink);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "stream_read launch");
}

// ---- token routing around ragged_dot ----------------------------------------------------------------------------

static int moe_elem(int dtype) { return dtype == RD_DTYPE_F32 ? 1 : dtype == RD_DTYPE_F16 ? 2 : 0; }

static int check_moe(int tokens, int top_k, int d, int dtype) {
  if (tokens < 0 || top_k < 1 || top_k > rd::kMoeMaxTopK || d < 0 || (long long)tokens * top_k >= (1ll << 31))
    return fail(RD_ERR_INVALID_ARGUMENT, "bad routing shape tokens=%d top_k=%d (1..%d) d=%d", tokens, top_k, rd::kMoeMaxTopK, d);
  if (dtype != RD_DTYPE_BF16 && dtype != RD_DTYPE_F32 && dtype != RD_DTYPE_F16)
    return fail(RD_ERR_INVALID_ARGUMENT, "unknown dtype %d for routing (rows are bfloat16, float32 or float16)", dtype);
  return RD_OK;
}

size_t rd_moe_route_workspace_bytes(int tokens, int top_k, int g) {
  if (tokens < 0 || top_k < 1 || g < 1) return 0;
  return align_up(rd::moe_route_workspace_bytes((long long)tokens * top_k, g), 256);
}

int rd_moe_route(void* stream, const int32_t* expert_ids, int tokens, int top_k, int g, int32_t* group_sizes,
                 int32_t* row_of_slot, int32_t* slot_of_row, void* workspace, size_t workspace_bytes) {
  int rc = check_moe(tokens, top_k, 0, RD_DTYPE_BF16);
  if (rc != RD_OK) return rc;
  if (g < 1 || g > rd::kMoeMaxGroups) return fail(RD_ERR_INVALID_ARGUMENT, "g=%d outside 1..%d", g, rd::kMoeMaxGroups);
  const int slots = tokens * top_k;
  if (!group_sizes || (slots > 0 && (!expert_ids || !row_of_slot || !slot_of_row)))
    return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0 ||
      workspace_bytes < rd::moe_route_workspace_bytes(slots, g))
    return fail(RD_ERR_WORKSPACE, "workspace null, misaligned or smaller than %zu B", rd::moe_route_workspace_bytes(slots, g));
  rc = rd::launch_moe_route((hipStream_t)stream, expert_ids, slots, g, group_sizes, row_of_slot, slot_of_row,
                            static_cast<int32_t*>(workspace));
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_route launch");
}

int rd_moe_dispatch(void* stream, const void* h, const int32_t* row_of_slot, const int32_t* slot_of_row,
                    const float* row_scale, void* x, int tokens, int top_k, int d, int dtype) {
  int rc = check_moe(tokens, top_k, d, dtype);
  if (rc != RD_OK) return rc;
  if (tokens == 0 || d == 0) return RD_OK;
  if (!h || !row_of_slot || !slot_of_row || !x) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_moe_dispatch((hipStream_t)stream, h, row_of_slot, slot_of_row, row_scale, x, tokens, top_k, d, moe_elem(dtype));
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_dispatch launch");
}

int rd_moe_combine(void* stream, const void* y, const int32_t* row_of_slot, const float* weights, void* out,
                   int tokens, int top_k, int d, int dtype) {
  int rc = check_moe(tokens, top_k, d, dtype);
  if (rc != RD_OK) return rc;
  if (tokens == 0 || d == 0) return RD_OK;
  if (!y || !row_of_slot || !out) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_moe_combine((hipStream_t)stream, y, row_of_slot, weights, out, tokens, top_k, d, moe_elem(dtype));
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_combine launch");
}

int rd_moe_combine_wgrad(void* stream, const void* y, const void* dout, const int32_t* row_of_slot, float* dw,
                         int tokens, int top_k, int d, int dtype) {
  int rc = check_moe(tokens, top_k, d, dtype);
  if (rc != RD_OK) return rc;
  if (tokens == 0) return RD_OK;
  if (!row_of_slot || !dw || (d > 0 && (!y || !dout))) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_moe_combine_wgrad((hipStream_t)stream, y, dout, row_of_slot, dw, tokens, top_k, d, moe_elem(dtype));
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_combine_wgrad launch");
}

static int check_gate(const void* logits, const int32_t* ids, const float* weights, int tokens, int experts, const rd_gate_spec* spec,
                      int dtype, rd::GateSpec* out) {
  if (!spec) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  const int rc = check_moe(tokens, spec->top_k, 0, dtype);
  if (rc != RD_OK) return rc;
  if (tokens > rd::kGateMaxTokens) return fail(RD_ERR_INVALID_ARGUMENT, "tokens=%d outside 0..%d", tokens, rd::kGateMaxTokens);
  if (experts < 1 || experts > rd::kGateMaxExperts) return fail(RD_ERR_INVALID_ARGUMENT, "experts=%d outside 1..%d", experts, rd::kGateMaxExperts);
  if (spec->clusters < 1 || spec->clusters > 64 || experts % spec->clusters != 0)
    return fail(RD_ERR_INVALID_ARGUMENT, "clusters=%d (1..64) do not divide experts=%d", spec->clusters, experts);
  if (spec->top_clusters < 1 || spec->top_clusters > spec->clusters || spec->top_k > spec->top_clusters * (experts / spec->clusters))
    return fail(RD_ERR_INVALID_ARGUMENT, "top_clusters=%d of %d clusters hold fewer than top_k=%d experts", spec->top_clusters, spec->clusters, spec->top_k);
  if ((spec->flags & ~(RD_GATE_SIGMOID | RD_GATE_TOP2 | RD_GATE_RENORMALIZE)) != 0) return fail(RD_ERR_INVALID_ARGUMENT, "unknown gate flags %d", spec->flags);
  if (!(spec->scale - spec->scale == 0.f) || spec->scale == 0.f) return fail(RD_ERR_INVALID_ARGUMENT, "scale must be finite and not 0");
  if (tokens > 0 && (!logits || !ids || !weights)) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  *out = rd::GateSpec{tokens, experts, spec->top_k, spec->clusters, spec->top_clusters, (spec->flags & RD_GATE_SIGMOID) != 0,
                      (spec->flags & RD_GATE_TOP2) != 0, (spec->flags & RD_GATE_RENORMALIZE) != 0, spec->scale, moe_elem(dtype)};
  return RD_OK;
}

int rd_moe_gate(void* stream, const void* logits, const float* bias, int32_t* expert_ids, float* weights, int tokens,
                int experts, const rd_gate_spec* spec, int dtype) {
  rd::GateSpec p;
  int rc = check_gate(logits, expert_ids, weights, tokens, experts, spec, dtype, &p);
  if (rc != RD_OK || tokens == 0) return rc;
  rc = rd::launch_moe_gate((hipStream_t)stream, logits, bias, expert_ids, weights, p);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_gate launch");
}

int rd_moe_gate_grad(void* stream, const void* logits, const int32_t* expert_ids, const float* weights, const float* dweights,
                     void* dlogits, int tokens, int experts, const rd_gate_spec* spec, int dtype) {
  rd::GateSpec p;
  int rc = check_gate(logits, expert_ids, weights, tokens, experts, spec, dtype, &p);
  if (rc != RD_OK || tokens == 0) return rc;
  if (!dweights || !dlogits) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_moe_gate_grad((hipStream_t)stream, logits, expert_ids, weights, dweights, dlogits, p);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_gate_grad launch");
}

static int check_swiglu(int rows, int f, int dtype) {
  if (rows < 0 || f < 0 || f >= (1 << 30)) return fail(RD_ERR_INVALID_ARGUMENT, "bad shape rows=%d f=%d", rows, f);
  return check_moe(0, 1, 0, dtype);
}

int rd_moe_swiglu(void* stream, const void* y, void* out, int rows, int f, int dtype) {
  int rc = check_swiglu(rows, f, dtype);
  if (rc != RD_OK || rows == 0 || f == 0) return rc;
  if (!y || !out) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_moe_swiglu((hipStream_t)stream, y, out, rows, f, moe_elem(dtype));
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_swiglu launch");
}

int rd_moe_swiglu_grad(void* stream, const void* y, const void* dout, void* dy, int rows, int f, int dtype) {
  int rc = check_swiglu(rows, f, dtype);
  if (rc != RD_OK || rows == 0 || f == 0) return rc;
  if (!y || !dout || !dy) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_moe_swiglu_grad((hipStream_t)stream, y, dout, dy, rows, f, moe_elem(dtype));
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "moe_swiglu_grad launch");
}

size_t rd_int4_codes_bytes(int g, int k, int n) {
  if (g < 0 || k < 0 || n < 0) return 0;
  return (size_t)g * rd::int4_strips(n) * rd::int4_runs(k) * 1024;
}

static int check_int4_weights(const void* codes, int g, int k, int n) {
  if (g < 1 || k < 0 || n < 0 || k > (1 << 24) || n > (1 << 24)) return fail(RD_ERR_INVALID_ARGUMENT, "bad shape g=%d k=%d n=%d", g, k, n);
  if ((long long)g * rd::int4_strips(n) * rd::int4_runs(k) >= (1ll << 29)) return fail(RD_ERR_INVALID_ARGUMENT, "g*k*n too large");
  if (k > 0 && n > 0 && (!codes || (reinterpret_cast<uintptr_t>(codes) & 15) != 0))
    return fail(RD_ERR_INVALID_ARGUMENT, "the codes are null or not 16-byte aligned");
  return RD_OK;
}

int rd_int4_pack(void* stream, const uint8_t* q, void* codes, int g, int k, int n, int trans_rhs) {
  int rc = check_int4_weights(codes, g, k, n);
  if (rc != RD_OK || k == 0 || n == 0) return rc;
  if (!q) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  rc = rd::launch_int4_pack((hipStream_t)stream, q, static_cast<uint32_t*>(codes), g, k, n, trans_rhs != 0);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "int4_pack launch");
}

size_t rd_gmm_int4_workspace_bytes(int m, int k, int n, int g, int kernel) {
  if (m < 0 || k < 0 || n < 0 || g < 1) return 0;
  return align_up(rd::int4_workspace_bytes(m, k, n, g, g, kernel), 256);  // (a slice of the groups needs no more)
}

int rd_gmm_int4(void* stream, const void* x, const void* codes, const void* scales, const uint8_t* zeros,
                const int32_t* group_sizes, void* y, int m, int k, int n, int g_total, int group_offset, int g_local, int block,
                int scale_dtype, int dtype, int kernel, void* workspace, size_t workspace_bytes) {
  int rc = check_int4_weights(codes, g_local, k, n);
  if (rc != RD_OK) return rc;
  if (m < 0 || m > rd::kInt4MaxRows) return fail(RD_ERR_INVALID_ARGUMENT, "m=%d outside 0..%d", m, rd::kInt4MaxRows);
  if (g_total < 1 || group_offset < 0 || group_offset > g_total - g_local)
    return fail(RD_ERR_INVALID_ARGUMENT, "groups [%d, %d + %d) are not within the %d of group_sizes", group_offset, group_offset, g_local, g_total);
  if (block != 32 && block != 64 && block != 128) return fail(RD_ERR_INVALID_ARGUMENT, "block=%d is none of 32, 64, 128", block);
  if (dtype != RD_DTYPE_BF16 && dtype != RD_DTYPE_F16) return fail(RD_ERR_INVALID_ARGUMENT, "dtype %d: rows are bfloat16 or float16", dtype);
  if (scale_dtype != RD_DTYPE_BF16 && scale_dtype != RD_DTYPE_F16)
    return fail(RD_ERR_INVALID_ARGUMENT, "scale dtype %d: scales are bfloat16 or float16", scale_dtype);
  if (kernel < RD_INT4_AUTO || kernel > RD_INT4_TILES) return fail(RD_ERR_INVALID_ARGUMENT, "unknown kernel %d", kernel);
  if (m == 0 || n == 0) return RD_OK;
  if (!group_sizes || !y || (k > 0 && (!x || !scales))) return fail(RD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail(RD_ERR_WORKSPACE, "workspace misaligned");
  const size_t needed = rd::int4_tiles_hold(dtype == RD_DTYPE_F16, scale_dtype == RD_DTYPE_F16) ? rd::int4_workspace_bytes(m, k, n, g_total, g_local, kernel) : 0;
  float* partials = workspace && needed > 0 && workspace_bytes >= needed ? static_cast<float*>(workspace) : nullptr;
  int32_t* counters = partials ? reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + rd::kInt4PartialBytes) : nullptr;
  const rd::Int4Problem p = {x, static_cast<const uint32_t*>(codes), scales, zeros, group_sizes, y, m, k, n, g_total, group_offset, g_local,
                             block, scale_dtype == RD_DTYPE_F16, dtype == RD_DTYPE_F16, kernel, partials, counters};
  if (!rd::int4_grid_fits(p)) return fail(RD_ERR_UNSUPPORTED, "m=%d rows of n=%d in %d groups are more tiles than a launch has", m, n, g_total);
  rc = rd::launch_gmm_int4((hipStream_t)stream, p);
  return rc == hipSuccess ? RD_OK : hip_fail(rc, "gmm_int4 launch");
}

}  // extern "C"
