// Row elements (bfloat16, float16, float32) as float32 and back, one rounding to nearest even.
#pragma once
#include "rd_common.h"

namespace rd {

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<bf16_bits>(bf16_bits v) { return bf16_to_f32(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<f16_t>(f16_t v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ bf16_bits from_f32<bf16_bits>(float v) { return f32_to_bf16(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float v) { return (f16_t)v; }

// sig(g) and sig(-g), neither by a difference from one, nor of an exponential that overflows.  16-bit results: exponential and
// reciprocal of the hardware, good to 2 units of 2^-23 and the rounding of g log2(e).
template <class T>
__device__ __forceinline__ void sigmoids(float g, float* of, float* of_minus) {
  const float t = sizeof(T) == 2 ? __expf(-fabsf(g)) : expf(-fabsf(g));
  const float r = sizeof(T) == 2 ? __builtin_amdgcn_rcpf(1.f + t) : 1.f / (1.f + t);
  *of = g >= 0.f ? r : t * r;
  *of_minus = g >= 0.f ? t * r : r;
}

}  // namespace rd
