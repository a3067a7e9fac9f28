// Numbers to float8 e4m3fn with a scale for each block of 128 and back (rd_float8.h has the definition): rows as they are, rows sorted
// by expert on the way, rows behind the gated activation, and weights in blocks of 128 x 128.
//
// Bound by memory.  Sixteen lanes hold a block of a row, eight neighbours each, so that the largest magnitude is four moves within
// a row of lanes away, and a code is written by whom it was read: 16 bytes in, 8 out, lines of 128 bytes per block.
#include "rd_elem.h"
#include "rd_float8.h"

namespace rd {

namespace {

constexpr int kF8Threads = 256;
constexpr int kF8Per = 8;                        // neighbours of a row that a lane holds
constexpr int kF8Lanes = kF8Block / kF8Per;      // lanes of a block
constexpr int kF8Groups = kF8Threads / kF8Lanes;  // blocks of a work-group at a time
constexpr float kF8Least = 0x1p-80f;

// Eight neighbours at any address, of which `live` are there; the others are 0.
template <class T>
__device__ __forceinline__ void load8(const T* p, int live, float (&v)[kF8Per]) {
  if (live >= kF8Per) {
    alignas(16) T e[kF8Per];
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<u32x4_t*>(e)[i] = load_any<u32x4_t>(p + i * (16 / sizeof(T)));
#pragma unroll
    for (int i = 0; i < kF8Per; ++i) v[i] = to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kF8Per; ++i) v[i] = i < live ? to_f32<T>(p[i]) : 0.f;
  }
}

// Magnitudes compare as their bits, infinity above every number and NaN above that.
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[kF8Per]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kF8Per; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  return top;
}
template <int CTRL>
__device__ __forceinline__ uint32_t max_with(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
  return o > v ? o : v;
}
// over sixteen lanes, for all of them: row_ror:8, 4, 2, 1
__device__ __forceinline__ uint32_t largest_of_row(uint32_t v) {
  return max_with<0x121>(max_with<0x122>(max_with<0x124>(max_with<0x128>(v))));
}

__device__ __forceinline__ float scale_of(uint32_t top, bool pow2) {
  if (top >= 0x7f800000u) return __builtin_bit_cast(float, 0x7fc00000u);
  const float s = fmaxf(__builtin_bit_cast(float, top), kF8Least) / 448.f;
  if (!pow2) return s;
  const uint32_t b = __builtin_bit_cast(uint32_t, s);  // a normal number: the next exponent, unless there is nothing behind the leading bit
  return __builtin_bit_cast(float, (b + 0x7fffffu) & 0x7f800000u);
}

// e4m3(x / s) of eight, `r` = 1 / s.  The quotient that is rounded to e4m3 is the float32 nearest to x / s: ties of e4m3 are frequent
// among rows of few bits, and a unit of 2^-24 to either side would decide them.  x r is off by two units at most, its residue x - q s
// is exact or off in its 25th bit, and q + r residue so the nearest float32, but for quotients within 2^-45 of a border between two.
__device__ __forceinline__ u32x2_t codes_of(const float (&v)[kF8Per], float s, float r) {
  float q[kF8Per];
#pragma unroll
  for (int i = 0; i < kF8Per; ++i) {
    const float q0 = v[i] * r;
    q[i] = __builtin_fmaf(__builtin_fmaf(-q0, s, v[i]), r, q0);
  }
  u32x2_t w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int d = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], d, true);
  }
  return w;
}

// Block `b` of a source row: its eight numbers of this lane.
template <class T, bool SWIGLU>
__device__ __forceinline__ void row_block(const T* __restrict__ row, int k, int c, float (&v)[kF8Per]) {
  load8<T>(row + c, k - c, v);
  if constexpr (SWIGLU) {
    float u[kF8Per];
    load8<T>(row + k + c, k - c, u);
#pragma unroll
    for (int i = 0; i < kF8Per; ++i) {
      float a, b;
      sigmoids<T>(v[i], &a, &b);
      v[i] = v[i] * a * u[i];
    }
  }
}

// A work-group takes kF8Groups neighbouring (row, block) items; blocks past the last one of a row are the padding of its scales.
// 32768 x 7168 and 32768 x 2048 bf16: 175 us together, 5.2 TB/s; behind the gated activation, 32768 x 2048 bf16: 70 us, 4.8 TB/s.
template <class T, bool SWIGLU>
__global__ __launch_bounds__(kF8Threads) void float8_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                                 long long items, int k, bool pow2) {
  const int blocks = float8_blocks(k), per_row = float8_scale_pitch(k), lane = threadIdx.x % kF8Lanes;
  const long long first = (long long)blockIdx.x * kF8Groups, row0 = first / per_row;
  const uint32_t at = (uint32_t)(first - row0 * per_row) + threadIdx.x / kF8Lanes, down = at / per_row;
  if (first + threadIdx.x / kF8Lanes >= items) return;
  const long long row = row0 + down;
  const int b = (int)(at - down * per_row);
  if (b < blocks) {
    float v[kF8Per];
    row_block<T, SWIGLU>(x + row * (SWIGLU ? 2 * (long long)k : k), k, b * kF8Block + lane * kF8Per, v);
    const float s = scale_of(largest_of_row(largest_bits(v)), pow2);
    *reinterpret_cast<u32x2_t*>(codes + (row * blocks + b) * kF8Block + lane * kF8Per) = codes_of(v, s, 1.f / s);
    if (lane == 0) scales[row * per_row + b] = s;
  } else if (lane == 0) {
    scales[row * per_row + b] = 0.f;
  }
}

// The same for a token's row, written to the rows of its slots; and the rows of no slot, as zeros: row i is looked after by token i / top_k.
// 4096 tokens of 7168 bf16 to eight rows each: 74 us, 4.1 TB/s, four fifths of it written.
template <class T>
__global__ __launch_bounds__(kF8Threads) void float8_dispatch_kernel(const T* __restrict__ h, const int32_t* __restrict__ row_of_slot,
                                                                     const int32_t* __restrict__ slot_of_row, uint8_t* __restrict__ codes,
                                                                     float* __restrict__ scales, long long items, int top_k, int d, bool pow2) {
  const int blocks = float8_blocks(d), per_row = float8_scale_pitch(d), lane = threadIdx.x % kF8Lanes;
  const long long first = (long long)blockIdx.x * kF8Groups, token0 = first / per_row;
  const uint32_t at = (uint32_t)(first - token0 * per_row) + threadIdx.x / kF8Lanes, down = at / per_row;
  if (first + threadIdx.x / kF8Lanes >= items) return;
  const long long token = token0 + down;
  const int b = (int)(at - down * per_row);
  float v[kF8Per] = {};
  if (b < blocks) row_block<T, false>(h + token * d, d, b * kF8Block + lane * kF8Per, v);
  const float s = b < blocks ? scale_of(largest_of_row(largest_bits(v)), pow2) : 0.f;
  const u32x2_t w = codes_of(v, s, 1.f / s);
  const float none = b < blocks ? scale_of(0, pow2) : 0.f;
  for (int i = 0; i < top_k; ++i) {
    const long long slot = token * top_k + i;
    const int row = row_of_slot[slot];
    if (row >= 0) {
      if (b < blocks) *reinterpret_cast<u32x2_t*>(codes + ((long long)row * blocks + b) * kF8Block + lane * kF8Per) = w;
      if (lane == 0) scales[(long long)row * per_row + b] = s;
    }
    if (slot_of_row[slot] < 0) {
      if (b < blocks) *reinterpret_cast<u32x2_t*>(codes + (slot * blocks + b) * kF8Block + lane * kF8Per) = u32x2_t{0, 0};
      if (lane == 0) scales[slot * per_row + b] = none;
    }
  }
}

// A work-group to a block of 128 x 128: sixteen lanes to a row, eight rows to a thread.  256 x 7168 x 2048 bf16: 2140 us, 5.3 TB/s.
template <class T>
__global__ __launch_bounds__(kF8Threads) void float8_weights_kernel(const T* __restrict__ A, uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                                    int a, int b, bool pow2) {
  constexpr int ROWS = kF8Block / kF8Groups;
  __shared__ uint32_t tops[kF8Threads / 64];
  const int down = float8_blocks(a), across = float8_blocks(b);
  const long long e = blockIdx.x / ((long long)down * across);
  const int in_matrix = (int)(blockIdx.x - e * down * across), ri = in_matrix / across, ci = in_matrix - ri * across;
  const int r0 = ri * kF8Block + threadIdx.x / kF8Lanes, c = ci * kF8Block + threadIdx.x % kF8Lanes * kF8Per;
  float v[ROWS][kF8Per];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = r0 + i * kF8Groups;
    load8<T>(A + (e * a + r) * b + c, r < a ? b - c : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const uint32_t t = largest_bits(v[i]);
    top = t > top ? t : top;
  }
  top = largest_of_row(top);
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_xor((int)top, o, 64);
    top = t > top ? t : top;
  }
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kF8Threads / 64; ++w) top = tops[w] > top ? tops[w] : top;
  const float s = scale_of(top, pow2), r = 1.f / s;
  const long long pitch = (long long)across * kF8Block;
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    *reinterpret_cast<u32x2_t*>(codes + (e * down * kF8Block + r0 + i * kF8Groups) * pitch + c) = codes_of(v[i], s, r);
  if (threadIdx.x == 0) scales[blockIdx.x] = s;
}

// Eight numbers of a row per thread.  32768 x 7168 to bf16: 152 us, 4.7 TB/s; 32768 x 2048: 37 us, 5.5 TB/s.
template <class T>
__global__ __launch_bounds__(kF8Threads) void float8_values_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ out,
                                                                   long long pieces, int a, int b, int height) {
  const int across = float8_blocks(b), per_row = (b + kF8Per - 1) / kF8Per;
  const int pitch = height == 1 ? float8_scale_pitch(b) : across, down = (a + height - 1) / height;
  const long long first = (long long)blockIdx.x * kF8Threads, row0 = first / per_row;
  if (first + threadIdx.x >= pieces) return;
  const uint32_t at = (uint32_t)(first - row0 * per_row) + threadIdx.x, below = at / per_row;
  const long long row = row0 + below, e = row / a;
  const int r = (int)(row - e * a), c = (int)(at - below * per_row) * kF8Per;
  const u32x2_t w = *reinterpret_cast<const u32x2_t*>(codes + (e * down * height + r) * ((long long)across * kF8Block) + c);
  const float s = scales[(e * down + r / height) * pitch + c / kF8Block];
  alignas(16) T v[kF8Per];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
    v[4 * h] = from_f32<T>(lo[0] * s);
    v[4 * h + 1] = from_f32<T>(lo[1] * s);
    v[4 * h + 2] = from_f32<T>(hi[0] * s);
    v[4 * h + 3] = from_f32<T>(hi[1] * s);
  }
  T* to = out + row * b + c;
  if (b - c >= kF8Per) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(v) / 16; ++i) store_any(to + i * (16 / sizeof(T)), reinterpret_cast<const u32x4_t*>(v)[i]);
  } else {
    for (int i = 0; i < b - c; ++i) to[i] = v[i];
  }
}

unsigned groups_for(long long work, int per_group) { return (unsigned)((work + per_group - 1) / per_group); }

template <class T, bool SWIGLU>
int rows_t(hipStream_t s, const void* x, void* codes, float* scales, long long rows, int k, bool pow2) {
  const long long items = rows * float8_scale_pitch(k);
  hipLaunchKernelGGL((float8_rows_kernel<T, SWIGLU>), dim3(groups_for(items, kF8Groups)), dim3(kF8Threads), 0, s, (const T*)x, (uint8_t*)codes, scales, items, k, pow2);
  return (int)hipGetLastError();
}
template <class T>
int dispatch_t(hipStream_t s, const void* h, const int32_t* row_of_slot, const int32_t* slot_of_row, void* codes, float* scales, int tokens, int top_k,
               int d, bool pow2) {
  const long long items = (long long)tokens * float8_scale_pitch(d);
  hipLaunchKernelGGL((float8_dispatch_kernel<T>), dim3(groups_for(items, kF8Groups)), dim3(kF8Threads), 0, s, (const T*)h, row_of_slot, slot_of_row,
                     (uint8_t*)codes, scales, items, top_k, d, pow2);
  return (int)hipGetLastError();
}
template <class T>
int weights_t(hipStream_t s, const void* A, void* codes, float* scales, int g, int a, int b, bool pow2) {
  const long long blocks = (long long)g * float8_blocks(a) * float8_blocks(b);
  hipLaunchKernelGGL((float8_weights_kernel<T>), dim3((unsigned)blocks), dim3(kF8Threads), 0, s, (const T*)A, (uint8_t*)codes, scales, a, b, pow2);
  return (int)hipGetLastError();
}
template <class T>
int values_t(hipStream_t s, const void* codes, const float* scales, void* out, int g, int a, int b, int height) {
  const long long pieces = (long long)g * a * ((b + kF8Per - 1) / kF8Per);
  hipLaunchKernelGGL((float8_values_kernel<T>), dim3(groups_for(pieces, kF8Threads)), dim3(kF8Threads), 0, s, (const uint8_t*)codes, scales, (T*)out, pieces, a, b, height);
  return (int)hipGetLastError();
}

}  // namespace

int launch_float8_rows(hipStream_t s, const void* x, void* codes, float* scales, long long rows, int k, bool swiglu, bool pow2, int elem) {
  if (swiglu)
    return elem == 1 ? rows_t<float, true>(s, x, codes, scales, rows, k, pow2) : elem == 2 ? rows_t<f16_t, true>(s, x, codes, scales, rows, k, pow2)
                                                                                         : rows_t<bf16_bits, true>(s, x, codes, scales, rows, k, pow2);
  return elem == 1 ? rows_t<float, false>(s, x, codes, scales, rows, k, pow2) : elem == 2 ? rows_t<f16_t, false>(s, x, codes, scales, rows, k, pow2)
                                                                                        : rows_t<bf16_bits, false>(s, x, codes, scales, rows, k, pow2);
}
int launch_float8_dispatch(hipStream_t s, const void* h, const int32_t* row_of_slot, const int32_t* slot_of_row, void* codes, float* scales,
                           int tokens, int top_k, int d, bool pow2, int elem) {
  return elem == 1 ? dispatch_t<float>(s, h, row_of_slot, slot_of_row, codes, scales, tokens, top_k, d, pow2)
       : elem == 2 ? dispatch_t<f16_t>(s, h, row_of_slot, slot_of_row, codes, scales, tokens, top_k, d, pow2)
                   : dispatch_t<bf16_bits>(s, h, row_of_slot, slot_of_row, codes, scales, tokens, top_k, d, pow2);
}
int launch_float8_weights(hipStream_t s, const void* A, void* codes, float* scales, int g, int a, int b, bool pow2, int elem) {
  return elem == 1 ? weights_t<float>(s, A, codes, scales, g, a, b, pow2) : elem == 2 ? weights_t<f16_t>(s, A, codes, scales, g, a, b, pow2)
                                                                                    : weights_t<bf16_bits>(s, A, codes, scales, g, a, b, pow2);
}
int launch_float8_values(hipStream_t s, const void* codes, const float* scales, void* out, int g, int a, int b, int height, int elem) {
  return elem == 1 ? values_t<float>(s, codes, scales, out, g, a, b, height) : elem == 2 ? values_t<f16_t>(s, codes, scales, out, g, a, b, height)
                                                                                       : values_t<bf16_bits>(s, codes, scales, out, g, a, b, height);
}

}  // namespace rd
