// Newton-Schulz iteration on a stack of matrices:  X = G / (|G|_F + eps), then `steps` times
//   A = X X',  B = b A + c A A,  X = a X + B X
// with X the smaller side down (G or its transpose), which drives the singular values of X towards one.  Three products of matrices
// per step, of which the first two are symmetric: their tiles on and below the diagonal are computed, and written twice.
//
// Numbers are float16 times a power of two per matrix, step and kind that the growth of the singular values allows (|X|, |A| and |B|
// are bounded by polynomials of it, from |G|_F / (|G|_F + eps) on), so that 2^15 is reached and 2^-29 of it still has all eleven bits.  float16 and not bfloat16:
// eleven bits instead of eight at the same rate.  What the tiles add up is fp32.
//   bfloat16 G: X is held in two numbers, hi + lo, of which the products take hi; A and B in one.  Along the small singular values of X
//              every step multiplies what is there by a = 3.4, the rounding of X included, until after five steps it has grown 485 times:
//              of an update of low rank X in one number left 2 % of noise, in two 0.1 %.  Products of hi alone cost next to nothing of
//              that, since B is small along small singular values.  lo is a byte, the residue times 32 in e4m3: its four bits behind hi's
//              eleven are all that pays (sixteen of them left 0.1 % too), and X is most of what is moved.  X before the last step, whose
//              rounding grows once, has none.
//   float32 G: everything in two numbers and every product in three, lo hi + hi lo + hi hi: 22 bits, as accurate as float32 products.
//   float16 G: as float32 G, for 2.4 times the time of bfloat16: products of eleven bits were off by 1.4e-3 to 2.3e-3, five times what the
//              rounding of the result is.
//   bfloat16 G whose coefficients make the small singular values, and with them the roundings, grow more than 2048 times: as float32 G.  Of 256 x 512 of rank 4 eight steps of a = 3.4445 (19816 times) left 3.4e-2 of noise in the numbers above, ten
//              0.39, in these 5e-4 and 5e-3.
#include "rd_elem.h"
#include "rd_gemm_w4.h"
#include "rd_ortho.h"

#include <math.h>
#include <type_traits>

namespace rd {

namespace {

constexpr int kOrthoThreads = 256;
constexpr int kOrthoChunk = 64 * 1024;  // numbers that a work-group adds up the squares of
typedef uint16_t half_bits;

// ---- norm ----------------------------------------------------------------------------------------------------------------
// Sums of squares in 64 bits: of 14336 x 4096 float32 numbers 32 bits would keep 1e-5 at worst, and squares of 1e-25 nothing.  128 x 2048
// x 768 bf16: 93 us, 4.3 TB/s.
template <class T>
__global__ __launch_bounds__(kOrthoThreads) void ortho_norm_kernel(const T* __restrict__ G, double* __restrict__ partial, long long size, int chunks) {
  __shared__ double sums[kOrthoThreads / 64];
  const long long e = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - e * chunks);
  const long long first = (long long)chunk * kOrthoChunk;
  const int count = (int)(size - first < kOrthoChunk ? size - first : kOrthoChunk);
  const T* p = G + e * size + first;
  double sum = 0;
  constexpr int PER = 16 / sizeof(T);
  const int whole = count / PER;
  for (int i = threadIdx.x; i < whole; i += kOrthoThreads) {
    alignas(16) T v[PER];
    *reinterpret_cast<u32x4_t*>(v) = load_any<u32x4_t>(p + i * PER);
#pragma unroll
    for (int j = 0; j < PER; ++j) { const double d = to_f32<T>(v[j]); sum = fma(d, d, sum); }
  }
  for (int i = whole * PER + threadIdx.x; i < count; i += kOrthoThreads) { const double d = to_f32<T>(p[i]); sum = fma(d, d, sum); }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

__device__ __forceinline__ float half_to_f32(half_bits b) { return (float)__builtin_bit_cast(f16_t, b); }
// Eight numbers as hi, and what hi leaves: as float16 (TWO), or times 32 as e4m3 bytes.  Numbers stay below 2^15, so the residue below 8.
constexpr float kByteUnit = 32.f;
__device__ __forceinline__ u32x4_t high_of(const float (&v)[8], float (&rest)[8]) {
  alignas(16) half_bits h[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const f16_t t = (f16_t)v[q];
    h[q] = __builtin_bit_cast(half_bits, t);
    rest[q] = v[q] - (float)t;
  }
  return *reinterpret_cast<const u32x4_t*>(h);
}
template <bool TWO>
__device__ __forceinline__ void store_low(void* lo, long long cell, const float (&rest)[8]) {
  if constexpr (TWO) {
    float none[8];
    *reinterpret_cast<u32x4_t*>(static_cast<half_bits*>(lo) + cell) = high_of(rest, none);
  } else {
    u32x2_t w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = __builtin_amdgcn_cvt_pk_fp8_f32(rest[4 * h] * kByteUnit, rest[4 * h + 1] * kByteUnit, 0, false);
      w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(rest[4 * h + 2] * kByteUnit, rest[4 * h + 3] * kByteUnit, d, true);
    }
    *reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(lo) + cell) = w;
  }
}
template <bool TWO> struct LowOf { typedef u32x2_t type; };
template <> struct LowOf<true> { typedef u32x4_t type; };
// v += hi + lo, times `by`
__device__ __forceinline__ void add_high(float (&v)[8], u32x4_t hi, float by) {
  alignas(16) half_bits h[8];
  *reinterpret_cast<u32x4_t*>(h) = hi;
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = __builtin_fmaf(half_to_f32(h[q]), by, v[q]);
}
__device__ __forceinline__ void add_low(float (&v)[8], u32x4_t lo, float by) { add_high(v, lo, by); }
__device__ __forceinline__ void add_low(float (&v)[8], u32x2_t lo, float by) {
  by *= 1 / kByteUnit;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo[h], true);
    v[4 * h] = __builtin_fmaf(a[0], by, v[4 * h]); v[4 * h + 1] = __builtin_fmaf(a[1], by, v[4 * h + 1]);
    v[4 * h + 2] = __builtin_fmaf(b[0], by, v[4 * h + 2]); v[4 * h + 3] = __builtin_fmaf(b[1], by, v[4 * h + 3]);
  }
}

// The sum of a matrix's squares, by every wave for itself, in the same order.
__device__ __forceinline__ double sum_of(const double* __restrict__ partial, int chunks) {
  double sum = 0;
  for (int i = threadIdx.x & 63; i < chunks; i += 64) sum += partial[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
  return sum;
}
// 1 / (norm + eps) of a sum of squares; NaN for one that is no number; of zeros, which stay 0 whatever eps, 0.
__device__ __forceinline__ double reciprocal_norm(double sum, double eps) { return sum == 0 ? 0. : 1 / (sqrt(sum) + eps + (sum - sum)); }
// What the singular values of X = G / (norm + eps) are below.
__device__ __forceinline__ double bound_of(double sum, double eps) { return sum > 0 ? sqrt(sum) * reciprocal_norm(sum, eps) : 1; }

// ---- bounds of the singular values ------------------------------------------------------------------------------------------
// A step's coefficients with what the host finds out: the places x where the derivative of q(x) = a x + b x^3 + c x^5 is 0, y of that of
// b y + c y^2, and the magnitudes there (places that there are not: beyond every limit).
struct OrthoTriple {
  double a, b, c, extreme[2], value[2], vertex, vertex_value;
};
struct OrthoTriples {
  OrthoTriple step[kOrthoMaxSteps];
  int steps;
};
__host__ __device__ inline double value_at(const OrthoTriple& t, double x) { return fabs(x * (t.a + x * x * (t.b + x * x * t.c))); }
// The largest |q(x)| for 0 <= x <= limit: at the end or where the derivative is 0; and |b y + c y^2| up to y = limit.
__host__ __device__ inline double largest(const OrthoTriple& t, double limit) {
  const double first = t.extreme[0] <= limit ? t.value[0] : 0, second = t.extreme[1] <= limit ? t.value[1] : 0;
  return fmax(value_at(t, limit), fmax(first, second));
}
__host__ __device__ inline double largest_square(const OrthoTriple& t, double limit) {
  return fmax(fabs(limit * (t.b + limit * t.c)), t.vertex <= limit ? t.vertex_value : 0);
}
// The power of two that takes numbers up to `top` to 2^15 at most, with room for what roundings add; and keeps factors normal numbers.
__host__ __device__ inline int exponent_for(double top) {
  int e;
  frexp(top * 1.01, &e);
  return top > 0 && 15 - e < 100 ? 15 - e : 100;
}
// The roots of a + 3 b y + 5 c y^2, y = x^2, without differences of what is nearly alike: h = -(3 b + sign(b) sqrt(9 b^2 - 20 a c)) gives the
// one as h / (10 c) and the other as 2 a / h, which is the cubic's where c is next to nothing.
OrthoTriple triple_of(double a, double b, double c) {
  OrthoTriple t{a, b, c, {HUGE_VAL, HUGE_VAL}, {0, 0}, HUGE_VAL, 0};
  const double unit = fmax(fmax(fabs(a), fabs(b)), fabs(c));  // (squares of coefficients beyond 1e154)
  const double h = -(3 * (b / unit) + copysign(sqrt(9 * (b / unit) * (b / unit) - 20 * (a / unit) * (c / unit)), b));
  const double y[2] = {h / (10 * (c / unit)), 2 * (a / unit) / h};
  for (int i = 0; i < 2; ++i)
    if (y[i] >= 0) {  // (no roots: y is no number)
      t.extreme[i] = sqrt(y[i]);
      t.value[i] = value_at(t, t.extreme[i]);
    }
  if (-b / (2 * c) >= 0) {
    t.vertex = -b / (2 * c);
    t.vertex_value = fabs(t.vertex * (b / 2));
  }
  return t;
}
OrthoTriples triples_of(int steps, const double* coefficients) {
  OrthoTriples t;
  t.steps = steps;
  for (int i = 0; i < steps; ++i) t.step[i] = triple_of(coefficients[3 * i], coefficients[3 * i + 1], coefficients[3 * i + 2]);
  return t;
}

// What a product multiplies its sums and what it adds by, and the last one its result.
struct OrthoFactors {
  float of_product, of_add, unit, none;
};
// Of the three products of a step whose singular values start below `bound`.
__device__ __forceinline__ void factors_of(const OrthoTriple& t, double bound, bool last, OrthoFactors* __restrict__ to) {
  const int ex = exponent_for(bound), ea = exponent_for(bound * bound), eb = exponent_for(largest_square(t, bound * bound)), en = exponent_for(largest(t, bound));
  to[0] = {(float)ldexp(1., ea - 2 * ex), 0.f, 1.f, 0.f};
  to[1] = {(float)ldexp(t.c, eb - 2 * ea), (float)ldexp(t.b, eb - ea), 1.f, 0.f};
  // (the last one's unit apart: together they would be less than normal numbers where singular values are small)
  to[2] = last ? OrthoFactors{(float)ldexp(1., -eb), (float)t.a, (float)ldexp(1., -ex), 0.f}
               : OrthoFactors{(float)ldexp(1., en - eb - ex), (float)ldexp(t.a, en - ex), 1.f, 0.f};
}

// X = G / (norm + eps), 64 x 64 numbers of the padded X per work-group; `tall`: X is the transpose of G.
// Memory: 128 x 2048 x 768 bf16 192 us, 5.2 TB/s.  The first g work-groups work out the factors of a matrix each, a lane those of a step
// (4 x 256 x 512: 4.5 us; in the first work-group of the matrix's tiles 5.7).
template <class T, bool TWO>
__global__ __launch_bounds__(kOrthoThreads) void ortho_start_kernel(const T* __restrict__ G, const double* __restrict__ partial, int chunks, half_bits* __restrict__ hi,
                                                                    void* __restrict__ lo, int g, int k, int n, int rp, int cp, bool tall, double eps, OrthoTriples triples,
                                                                    OrthoFactors* __restrict__ factors) {
  __shared__ float tile[64][65];
  if ((int)blockIdx.x < g) {
    const double sum = sum_of(partial + (long long)blockIdx.x * chunks, chunks);
    double bound = bound_of(sum, eps), own = bound;
    for (int i = 0; i < triples.steps; ++i) {
      if (i == (int)threadIdx.x) own = bound;
      bound = largest(triples.step[i], bound);
    }
    if ((int)threadIdx.x < triples.steps)
      factors_of(triples.step[threadIdx.x], own, (int)threadIdx.x + 1 == triples.steps, factors + ((long long)blockIdx.x * triples.steps + threadIdx.x) * 3);
    return;
  }
  const int block = (int)blockIdx.x - g, across = cp / 64, down = rp / 64;
  const long long e = block / (across * down);
  const int in_matrix = (int)(block - e * across * down), r0 = in_matrix / across * 64, c0 = in_matrix % across * 64;
  const T* from = G + e * k * n;
  // eight neighbours of a row of G to a thread, twice
  const int gr = tall ? c0 : r0, gc = tall ? r0 : c0, x = threadIdx.x % 8 * 8;
  float v[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = gr + threadIdx.x / 8 + 32 * h, c = gc + x;
    if (r < k && c + 8 <= n) {
      alignas(16) T in[8];
#pragma unroll
      for (int i = 0; i < (int)sizeof(in) / 16; ++i) reinterpret_cast<u32x4_t*>(in)[i] = load_any<u32x4_t>(from + (long long)r * n + c + i * (16 / sizeof(T)));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[h][i] = to_f32<T>(in[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[h][i] = r < k && c + i < n ? to_f32<T>(from[(long long)r * n + c + i]) : 0.f;
    }
  }
  const double sum = sum_of(partial + e * chunks, chunks);
  // a power of two and a number between 1/2 and 1: the factor of small norms is beyond float32
  int power;
  const float by = (float)frexp(ldexp(reciprocal_norm(sum, eps), exponent_for(bound_of(sum, eps))), &power);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int y = threadIdx.x / 8 + 32 * h;
      const float w = __builtin_ldexpf(v[h][i], power) * by;
      if (tall) tile[x + i][y] = w; else tile[y][x + i] = w;
    }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 64 * 8; i += kOrthoThreads) {
    const int r = i / 8, c = i % 8 * 8;
    const long long cell = e * rp * cp + (long long)(r0 + r) * cp + c0 + c;
    float w[8], rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = tile[r][c + j];
    *reinterpret_cast<u32x4_t*>(hi + cell) = high_of(w, rest);
    if (lo) store_low<TWO>(lo, cell, rest);
  }
}

// ---- products --------------------------------------------------------------------------------------------------------------
// Two planes of padded matrices [rows][cols]; no lo: one.
struct Planes {
  half_bits* hi;
  void* lo;
  int rows, cols;
};
enum OrthoKind { kGram, kSquare, kApply, kLast };
struct OrthoStep {
  Planes left, right;  // operands: the product is left right' (kGram, kSquare), or left right
  Planes add, to;      // result = of_product * product + of_add * add (kGram: no second term), of the matrix's factors, kLast: times unit and scale
  const OrthoFactors* factors;  // of the first matrix; those of the next one are `stride` behind it
  int stride;
  float scale;
  int g, tiles_r, tiles_c, per_matrix;
  // kLast: the numbers themselves, [k][n]
  void* out;
  int k, n, elem;
  bool tall;
};

template <class O>
__device__ __forceinline__ void store_last(O* out, int r, int c, int rows, int cols, const float (&v)[8]) {  // row r, columns c ..
  if (r >= rows || c >= cols) return;
  O* to = out + (long long)r * cols + c;
  alignas(16) O o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = from_f32<O>(v[i]);
  if (cols - c >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(o) / 16; ++i) store_any(to + i * (16 / sizeof(O)), reinterpret_cast<const u32x4_t*>(o)[i]);
  } else {
    for (int i = 0; i < cols - c; ++i) to[i] = o[i];
  }
}
__device__ __forceinline__ void store_last(const OrthoStep& p, long long e, int r, int c, const float (&v)[8]) {
  const long long at = e * p.k * p.n;
  if (p.elem == 1) store_last(static_cast<float*>(p.out) + at, r, c, p.k, p.n, v);
  else if (p.elem == 2) store_last(static_cast<f16_t*>(p.out) + at, r, c, p.k, p.n, v);
  else store_last(static_cast<bf16_bits*>(p.out) + at, r, c, p.k, p.n, v);
}

// Tiles of the products.  Of the symmetric ones they are square; of the others, whose contraction is short and whose results are read and
// written in two numbers, large ones are 128 x 256, two work-groups to a compute unit.
template <bool SYMMETRIC>
struct OrthoSmall {  // 64 x 64, a wave 32 x 32 of it, in slabs of 64
  static constexpr bool HALF = true, SMALL = true;
  static constexpr int BM = 64, BN = 64, BK = 64, STAGES = 5, NW = 4, WM = 32, WN = 32, TM = 1, TN = 1;
  static constexpr int A_BYTES = BM * BK * 2, STAGE_BYTES = 2 * A_BYTES, LDS_BYTES = STAGES * STAGE_BYTES;
  typedef DldsLoader<BM, BK, NW, true> LdA;
  typedef DldsLoader<BN, BK, NW, SYMMETRIC> LdB;
  typedef DldsFragReader<BM, BK, TM, true> FragA;
  typedef DldsFragReader<BN, BK, TN, SYMMETRIC> FragB;
};
template <int BM, bool SYMMETRIC>
struct OrthoTile {
  static constexpr int ROWS = !SYMMETRIC && BM == 256 ? 128 : BM, GROUPS = ROWS == 256 ? 1 : 2;
  typedef W4Cfg<ROWS, BM, true, SYMMETRIC, ROWS == 256 ? 5 : BM == 256 ? 3 : 4, true> C;
};
template <bool SYMMETRIC>
struct OrthoTile<64, SYMMETRIC> {
  static constexpr int GROUPS = 2;
  typedef OrthoSmall<SYMMETRIC> C;
};

// The small tile's K loop: what bounds it is how long the first slabs are on their way, so up to four are, and little else.
template <class C>
__device__ __forceinline__ void small_kloop(const half_bits* a, int lda, int rows, const half_bits* b, int ldb, int cols, int klen, unsigned char* smem, int wave, int lane,
                                            f32x16_t (&acc)[1][1]) {
  typename C::LdA la;
  typename C::LdB lb;
  la.init(a, lda, rows, klen, wave, lane);
  lb.init(b, ldb, cols, klen, wave, lane);
  typename C::FragA fra;
  typename C::FragB frb;
  fra.init((wave >> 1) * C::WM, lane);
  frb.init((wave & 1) * C::WN, lane);
  const int nk = klen / C::BK;  // (padded matrices)
  constexpr int L = C::LdA::PER + C::LdB::PER;
  auto issue = [&](int step) {
    unsigned char* st = smem + (step % C::STAGES) * C::STAGE_BYTES;
    __amdgpu_buffer_rsrc_t ra = la.resource(), rb = lb.resource();
#pragma unroll
    for (int q = 0; q < C::LdA::PER; ++q) la.template issue<false>(ra, st, wave, q, 0, 0);
#pragma unroll
    for (int q = 0; q < C::LdB::PER; ++q) lb.template issue<false>(rb, st + C::A_BYTES, wave, q, 0, 0);
    la.advance();
    lb.advance();
  };
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s)
    if (s < nk) issue(s);
  for (int kt = 0; kt < nk; ++kt) {
    if (kt + C::STAGES - 2 < nk) wait_vmcnt<(C::STAGES - 2) * L>(); else wait_vmcnt<0>();
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();  // slab kt is in LDS, and slab kt - 1 is no longer being read
    __builtin_amdgcn_sched_barrier(0);
    if (kt + C::STAGES - 1 < nk) issue(kt + C::STAGES - 1);
    const unsigned char* st = smem + (kt % C::STAGES) * C::STAGE_BYTES;
#pragma unroll
    for (int ks = 0; ks < C::BK / 16; ++ks) acc[0][0] = mfma_32x32x16<true>(frb.read(st + C::A_BYTES, 0, ks), fra.read(st, 0, ks), acc[0][0]);
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();  // the ring is no longer read by any wave
  __builtin_amdgcn_sched_barrier(0);
}

template <int BM, bool SYMMETRIC>
constexpr int ortho_groups = OrthoTile<BM, SYMMETRIC>::GROUPS;

// PLANES 2: lo hi + hi lo + hi hi, the largest last, so that the small ones are added to small sums.  In tiles of 64 and 128 each goes in
// pieces of the contraction whose sums start from zero: one sum of all was rounded once per sixteen indices and product where it was
// largest, and a long contraction of few rows lost more than float32 products do (1 x 32 x 4000: 8.0e-6 of the result, in pieces of 1024
// 1.9e-6, float32 products 2.1e-6; 2048 x 2048: 3.4e-6, 1.0e-6, 3.6e-6).  Pieces of 512 give no more there and cost 5 % of 12 x 1515 x
// 1001 instead of 2.  Tiles of 256 have no registers for a second sum, and enough rows for other roundings to outweigh this one.
//
// 128 x 2048 x 768 bf16, in tiles of 256: X X' 216 us (0.96 PFLOP/s of the six tiles of nine), A A 123 us (0.63: the contraction is
// short, and every tile is read, added and written twice), B X 479 us and the last, whose result is turned on its way out, 513 us (0.65
// and 0.60, 1.36 GB of X in two numbers read and written, 2.8 TB/s: a work-group that has multiplied waits for what it adds, and two to a
// compute unit hide half of that).
constexpr int kOrthoPiece = 1024;
template <int BM, int KIND, int PLANES>
__global__ __launch_bounds__(kOrthoThreads, (ortho_groups<BM, KIND == kGram || KIND == kSquare>)) void ortho_product_kernel(OrthoStep p) {
  constexpr bool SYMMETRIC = KIND == kGram || KIND == kSquare;
  typedef typename OrthoTile<BM, SYMMETRIC>::C C;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int id = xcd_contiguous_id(blockIdx.x, p.g * p.per_matrix);
  if (id < 0) return;
  const long long e = id / p.per_matrix;
  const int t = id - (int)e * p.per_matrix;
  int ti, tj;
  if (SYMMETRIC) {  // tiles on and below the diagonal, row by row
    ti = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
  } else {
    ti = t % p.tiles_r;
    tj = t / p.tiles_r;
  }
  const int r0 = ti * C::BM, c0 = tj * C::BN, klen = p.left.cols;
  const int rows = imin(C::BM, p.left.rows - r0), cols = imin(C::BN, (SYMMETRIC ? p.right.rows : p.right.cols) - c0);
  const long long left = e * p.left.rows * p.left.cols + (long long)r0 * p.left.cols;
  const long long right = e * p.right.rows * p.right.cols + (SYMMETRIC ? (long long)c0 * p.right.cols : c0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
  const bool live = wm * C::WM < rows && wn * C::WN < cols;

  // one to a lane, on their way with the first slabs (a scalar load's result would be waited for in front of them, or behind the K loop)
  const float factors = reinterpret_cast<const float*>(p.factors + e * p.stride)[lane & 3];
  f32x16_t acc[C::TM][C::TN];
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  auto product = [&](const half_bits* a, const half_bits* b, int len) {
    if constexpr (BM == 64) small_kloop<C>(a, p.left.cols, rows, b, p.right.cols, cols, len, smem, wave, lane, acc);
    else if (live) w4_kloop<C, true>(a, p.left.cols, rows, b, p.right.cols, cols, len, smem, wave, lane, acc);
    else w4_kloop<C, false>(a, p.left.cols, rows, b, p.right.cols, cols, len, smem, wave, lane, acc);
  };
  constexpr bool PIECES = PLANES == 2 && BM < 256;
  f32x16_t sum[PIECES ? C::TM : 1][PIECES ? C::TN : 1];
  if constexpr (PIECES) {
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) sum[i][j] = acc[i][j];
  }
#pragma unroll 1
  for (int term = PLANES == 2 ? 0 : 2; term < 3; ++term) {
    const half_bits* a = (term == 0 ? static_cast<const half_bits*>(p.left.lo) : p.left.hi) + left;
    const half_bits* b = (term == 1 ? static_cast<const half_bits*>(p.right.lo) : p.right.hi) + right;
    if constexpr (!PIECES) product(a, b, klen);
    else {
#pragma unroll 1
      for (int at = 0; at < klen; at += kOrthoPiece) {
        product(a + at, b + (SYMMETRIC ? at : (long long)at * p.right.cols), imin(kOrthoPiece, klen - at));
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              sum[i][j][v] += acc[i][j][v];
              acc[i][j][v] = 0.f;
            }
      }
    }
  }
  if constexpr (PIECES) {
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) acc[i][j] = sum[i][j];
  }
  if (!live) return;
  const auto factor = [&](int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, factors), i)); };
  const OrthoFactors by = {factor(0), factor(1), factor(2), 0.f};

  // by way of LDS, 32 rows of the wave's columns at a time, for eight neighbours of a row to a lane, or of a column; what is added is
  // requested before, a piece ahead where registers allow
  constexpr int PITCH = C::WN + 4;
  float* patch = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
  static_assert(C::NW * 32 * PITCH * 4 <= C::LDS_BYTES, "patches");
  constexpr int PER_ROW = C::WN / 8, STEP = 64 / PER_ROW, ITER = 32 / STEP;
  constexpr bool TWO = PLANES == 2, ADDS = KIND != kGram, ADDS_LO = ADDS && (TWO || KIND == kApply);  // (X before the last step has no bytes)
  typedef typename LowOf<TWO>::type Low;
  const bool turned = SYMMETRIC ? ti != tj : KIND == kLast && p.tall;
  const int own_r = lane / PER_ROW, own_c = lane % PER_ROW * 8, pc = c0 + wn * C::WN;
  const bool inside = pc + own_c < p.to.cols;
  const long long matrix = e * p.to.rows * p.to.cols, own = matrix + (long long)(r0 + wm * C::WM + own_r) * p.to.cols + pc + own_c;
  constexpr int AHEAD = SYMMETRIC ? 1 : 0;  // (the sums of the others leave no registers for two; the other work-group fills the wait)
  u32x4_t add_hi[AHEAD + 1][ADDS ? ITER : 1];
  Low add_lo[AHEAD + 1][ADDS_LO ? ITER : 1];
  auto request = [&](int i) {
    if constexpr (ADDS) {
      if (!inside || r0 + wm * C::WM + i * 32 >= p.left.rows) return;
#pragma unroll
      for (int t = 0; t < ITER; ++t) {
        const long long cell = own + (long long)(i * 32 + t * STEP) * p.to.cols;
        add_hi[i & AHEAD][t] = *reinterpret_cast<const u32x4_t*>(p.add.hi + cell);
        if constexpr (ADDS_LO) add_lo[i & AHEAD][t] = *reinterpret_cast<const Low*>(static_cast<const char*>(p.add.lo) + cell * (int)(sizeof(Low) / 8));
      }
    }
  };
  if constexpr (AHEAD > 0) request(0);
#pragma unroll
  for (int i = 0; i < C::TM; ++i) {
    const int pr = r0 + wm * C::WM + i * 32;
    if (pr >= p.left.rows) break;
    if (AHEAD == 0 || i + 1 < C::TM) request(i + AHEAD);
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4_t v;
        v[0] = acc[i][j][4 * g]; v[1] = acc[i][j][4 * g + 1]; v[2] = acc[i][j][4 * g + 2]; v[3] = acc[i][j][4 * g + 3];
        *reinterpret_cast<f32x4_t*>(patch + (lane & 31) * PITCH + j * 32 + 8 * g + 4 * (lane >> 5)) = v;
      }
    __builtin_amdgcn_wave_barrier();
    if (inside) {
#pragma unroll
      for (int t = 0; t < ITER; ++t) {
        float* at = patch + (t * STEP + own_r) * PITCH + own_c;
        float v[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const f32x4_t w = *reinterpret_cast<const f32x4_t*>(at + 4 * q);
          v[4 * q] = w[0] * by.of_product; v[4 * q + 1] = w[1] * by.of_product; v[4 * q + 2] = w[2] * by.of_product; v[4 * q + 3] = w[3] * by.of_product;
        }
        if constexpr (ADDS) {
          add_high(v, add_hi[i & AHEAD][t], by.of_add);
          if constexpr (ADDS_LO) add_low(v, add_lo[i & AHEAD][t], by.of_add);
        }
        if constexpr (KIND == kLast) {  // (one after the other: together they may be less than a normal number)
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = v[q] * by.unit * p.scale;
          if (!p.tall) store_last(p, e, pr + t * STEP + own_r, pc + own_c, v);
        } else {
          const long long cell = own + (long long)(i * 32 + t * STEP) * p.to.cols;
          float rest[8];
          *reinterpret_cast<u32x4_t*>(p.to.hi + cell) = high_of(v, rest);
          if (TWO || (KIND == kApply && p.to.lo)) store_low<TWO>(p.to.lo, cell, rest);
        }
        if (turned) {
#pragma unroll
          for (int q = 0; q < 2; ++q) *reinterpret_cast<f32x4_t*>(at + 4 * q) = f32x4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    if (turned) {
#pragma unroll
      for (int s = 0; s < C::WN; s += 16) {  // sixteen columns, four times eight of their rows
        const int c = s + (lane & 15), r = (lane >> 4) * 8;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = patch[(r + q) * PITCH + c];
        if (pc + c >= p.to.cols) continue;
        if constexpr (KIND == kLast) {
          store_last(p, e, pc + c, pr + r, v);
        } else {
          const long long cell = matrix + (long long)(pc + c) * p.to.cols + pr + r;
          float rest[8];
          *reinterpret_cast<u32x4_t*>(p.to.hi + cell) = high_of(v, rest);
          if constexpr (TWO) store_low<TWO>(p.to.lo, cell, rest);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// no steps: the matrices over their norms
template <class T>
__global__ __launch_bounds__(kOrthoThreads) void ortho_divide_kernel(const T* __restrict__ G, const double* __restrict__ partial, T* __restrict__ out, long long size,
                                                                     int chunks, double eps, double scale) {
  const long long e = blockIdx.x / chunks, first = (blockIdx.x - e * chunks) * (long long)kOrthoChunk;
  const double by = scale * reciprocal_norm(sum_of(partial + e * chunks, chunks), eps);
  for (long long i = first + threadIdx.x; i < size && i < first + kOrthoChunk; i += kOrthoThreads) out[e * size + i] = from_f32<T>((float)(to_f32<T>(G[e * size + i]) * by));
}

// Which tiles: the least time by rounds of what the device holds, 256 compute units of one or two work-groups, in tiles of 128 x 128.  As
// measured, a unit takes 1.35 times as long per number in tiles of 128 x 128, whose operands' reads of LDS bound it, 1.2 times in those of
// 128 x 256, 2.3 times in those of 64 x 64, and a work-group alone on it 0.7 times as long as two.  us, all products in tiles of 64 | 128 |
// 256, bf16: 4 of 256 x 512 83 | 127 | 213; 1 of 768 x 768 141 | 191 | 361; 1 of 2048 x 2048 500 | 343 | 634; 16 of 768 x 2048 817 | 583
// | 653; 12 of 1515 x 1001 872 | 595 | 656; 1 of 4096 x 4096 3266 | 1948 | 1503; 128 of 768 x 2048 7704 | 4963 | 4216.
int tile_for(bool symmetric, int g, int rows, int cols) {
  const auto time = [&](int r, int c, int groups, double slow) {
    const long long down = (rows + r - 1) / r, across = (cols + c - 1) / c, tiles = g * (symmetric ? down * (down + 1) / 2 : down * across);
    const double each = slow * r * c / (128.0 * 128.0);
    const int rest = (int)(tiles % (256 * groups));
    return (tiles / (256 * groups) * groups + (rest == 0 ? 0 : groups == 1 ? 1 : rest <= 256 ? 1.4 : 2)) * each;
  };
  const double large = symmetric ? time(256, 256, 1, 1) : time(128, 256, 2, 1.2), middle = time(128, 128, 2, 1.35), small = time(64, 64, 2, 2.3);
  return large <= middle && large <= small ? 256 : middle <= small ? 128 : 64;
}

template <int BM, int KIND, int PLANES>
int launch_product(hipStream_t s, OrthoStep p) {
  constexpr bool SYMMETRIC = KIND == kGram || KIND == kSquare;
  typedef typename OrthoTile<BM, SYMMETRIC>::C C;
  constexpr int LDS = C::LDS_BYTES;
  auto kern = ortho_product_kernel<BM, KIND, PLANES>;
  if (LDS > 64 * 1024) {
    const int rc = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (rc != hipSuccess) return rc;
  }
  p.tiles_r = (p.left.rows + C::BM - 1) / C::BM;
  p.tiles_c = SYMMETRIC ? p.tiles_r : (p.right.cols + C::BN - 1) / C::BN;
  p.per_matrix = SYMMETRIC ? p.tiles_r * (p.tiles_r + 1) / 2 : p.tiles_r * p.tiles_c;
  hipLaunchKernelGGL(kern, dim3((unsigned)xcd_padded_grid(p.g * p.per_matrix)), dim3(kOrthoThreads), LDS, s, p);
  return (int)hipGetLastError();
}
template <int KIND>
int launch_product(hipStream_t s, const OrthoStep& p, bool two) {
  switch (tile_for(KIND == kGram || KIND == kSquare, p.g, p.left.rows, p.right.cols)) {
    case 256: return two ? launch_product<256, KIND, 2>(s, p) : launch_product<256, KIND, 1>(s, p);
    case 128: return two ? launch_product<128, KIND, 2>(s, p) : launch_product<128, KIND, 1>(s, p);
    default: return two ? launch_product<64, KIND, 2>(s, p) : launch_product<64, KIND, 1>(s, p);
  }
}

struct OrthoSizes {
  int rp, cp, chunks;
  size_t norm, factors, x, bytes, square;  // bytes of the sums of squares, of the products' factors, of one plane of X and one of its bytes, and of one of A
};
size_t up(size_t b) { return (b + 255) / 256 * 256; }
OrthoSizes sizes_of(int g, int k, int n) {
  OrthoSizes z;
  const int r = k < n ? k : n, c = k < n ? n : k;
  z.rp = (r + kOrthoPad - 1) / kOrthoPad * kOrthoPad;
  z.cp = (c + kOrthoPad - 1) / kOrthoPad * kOrthoPad;
  z.chunks = (int)(((long long)k * n + kOrthoChunk - 1) / kOrthoChunk);
  z.norm = up((size_t)g * z.chunks * sizeof(double));
  z.factors = up((size_t)g * kOrthoMaxSteps * 3 * sizeof(OrthoFactors));
  z.x = up((size_t)g * z.rp * z.cp * 2);
  z.bytes = up((size_t)g * z.rp * z.cp);
  z.square = up((size_t)g * z.rp * z.rp * 2);
  return z;
}

template <class T>
int orthogonalize_t(hipStream_t s, const OrthoProblem& p) {
  const OrthoSizes z = sizes_of(p.g, p.k, p.n);
  const bool two = ortho_in_two(p.elem, p.steps, p.coefficients), tall = p.k > p.n;
  char* ws = static_cast<char*>(p.workspace);
  double* partial = reinterpret_cast<double*>(ws);
  ws += z.norm;
  OrthoFactors* factors = reinterpret_cast<OrthoFactors*>(ws);
  ws += z.factors;
  auto planes = [&](int rows, int cols, size_t bytes, size_t lo) {
    Planes q{reinterpret_cast<half_bits*>(ws), lo ? ws + bytes : nullptr, rows, cols};
    ws += bytes + lo;
    return q;
  };
  Planes X[2] = {planes(z.rp, z.cp, z.x, two ? z.x : z.bytes), planes(z.rp, z.cp, z.x, two ? z.x : z.bytes)};
  const Planes A = planes(z.rp, z.rp, z.square, two ? z.square : 0), B = planes(z.rp, z.rp, z.square, two ? z.square : 0);
  const long long size = (long long)p.k * p.n;
  hipLaunchKernelGGL((ortho_norm_kernel<T>), dim3((unsigned)(p.g * z.chunks)), dim3(kOrthoThreads), 0, s, (const T*)p.G, partial, size, z.chunks);
  int rc = (int)hipGetLastError();
  if (rc != hipSuccess) return rc;
  if (p.steps == 0) {
    hipLaunchKernelGGL((ortho_divide_kernel<T>), dim3((unsigned)(p.g * z.chunks)), dim3(kOrthoThreads), 0, s, (const T*)p.G, partial, (T*)p.out, size, z.chunks, p.eps, p.scale);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((two ? ortho_start_kernel<T, true> : ortho_start_kernel<T, !std::is_same<T, bf16_bits>::value>), dim3((unsigned)(p.g + p.g * (z.rp / 64) * (z.cp / 64))), dim3(kOrthoThreads), 0, s,
                     (const T*)p.G, partial, z.chunks, X[0].hi, two || p.steps > 1 ? X[0].lo : nullptr, p.g, p.k, p.n, z.rp, z.cp, tall, p.eps, triples_of(p.steps, p.coefficients), factors);
  if ((rc = (int)hipGetLastError()) != hipSuccess) return rc;
  OrthoStep t{};
  t.g = p.g; t.stride = 3 * p.steps;
  t.out = p.out; t.k = p.k; t.n = p.n; t.elem = p.elem; t.tall = tall; t.scale = (float)p.scale;
  for (int i = 0; i < p.steps; ++i) {
    t.factors = factors + 3 * i;
    t.left = t.right = X[i & 1];
    t.to = A;
    if ((rc = launch_product<kGram>(s, t, two)) != hipSuccess) return rc;
    ++t.factors;
    t.left = t.right = t.add = A;
    t.to = B;
    if ((rc = launch_product<kSquare>(s, t, two)) != hipSuccess) return rc;
    ++t.factors;
    const bool last = i + 1 == p.steps;
    t.left = B;
    t.right = t.add = X[i & 1];
    t.to = X[(i + 1) & 1];
    if (!two && i + 2 == p.steps) t.to.lo = nullptr;
    if ((rc = last ? launch_product<kLast>(s, t, two) : launch_product<kApply>(s, t, two)) != hipSuccess) return rc;
  }
  return hipSuccess;
}

}  // namespace

size_t ortho_workspace_bytes(int g, int k, int n, bool two) {
  const OrthoSizes z = sizes_of(g, k, n);
  return z.norm + z.factors + 2 * z.x + 2 * (two ? z.x : z.bytes) + (two ? 4 : 2) * z.square;
}

bool ortho_in_two(int elem, int steps, const double* coefficients) {
  if (elem != 0) return true;
  double bound = 1, grown = 1;  // the most that what was rounded so far has grown: X by 1 at the start and by its size before each step
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i];
    grown = fmax(grown, bound) * fabs(a);
    bound = largest(triple_of(a, coefficients[3 * i + 1], coefficients[3 * i + 2]), bound);
  }
  return grown > kOrthoMostGrown;
}

bool ortho_grid_fits(int g, int k, int n) {
  const OrthoSizes z = sizes_of(g, k, n);
  const double groups = (double)g * ((double)z.rp / 64 * z.cp / 64 + z.chunks);
  // 32-bit offsets of a tile's operands, and a launch's work-groups
  return groups < (double)(1 << 23) && (double)z.rp * z.cp < (double)(1 << 30);
}

double ortho_growth(int steps, const double* coefficients) {
  double bound = 1, top = 1;
  for (int i = 0; i < steps; ++i) {
    bound = largest(triple_of(coefficients[3 * i], coefficients[3 * i + 1], coefficients[3 * i + 2]), bound);
    top = fmax(top, bound);
  }
  return top;
}

int launch_orthogonalize(hipStream_t s, const OrthoProblem& p) {
  return p.elem == 1 ? orthogonalize_t<float>(s, p) : p.elem == 2 ? orthogonalize_t<f16_t>(s, p) : orthogonalize_t<bf16_bits>(s, p);
}

}  // namespace rd
