// The gated activation between an expert's two products: rows [gate | up] of 2 f elements -> silu(gate) * up, and its gradient.
//
//   out = g sig(g) u;  dg = dout u sig(g) (1 + g (1 - sig(g)));  du = dout g sig(g)
//
// Bound by memory: 3 f elements of a row forward, 5 f backward, each touched once.
#include "rd_elem.h"
#include "rd_moe.h"

namespace rd {

namespace {

constexpr int kSwigluThreads = 256;

// sig(g) and sig(-g), neither by a difference from one, nor of an exponential that overflows.
template <class T>
__device__ __forceinline__ void sigmoids(float g, float* of, float* of_minus) {
  const float t = sizeof(T) == 2 ? __expf(-fabsf(g)) : expf(-fabsf(g)), r = 1.f / (1.f + t);
  *of = g >= 0.f ? r : t * r;
  *of_minus = g >= 0.f ? t * r : r;
}

template <class T>
__device__ __forceinline__ float swiglu_of(float g, float u) {
  float a, b;
  sigmoids<T>(g, &a, &b);
  return g * a * u;
}
template <class T>
__device__ __forceinline__ void swiglu_grad_of(float g, float u, float d, float* dg, float* du) {
  float a, b;
  sigmoids<T>(g, &a, &b);
  *dg = d * u * a * (1.f + g * b);
  *du = d * g * a;
}

template <class T>
__global__ __launch_bounds__(kSwigluThreads) void moe_swiglu_kernel(const T* __restrict__ y, T* __restrict__ out, long long cells, int f) {
  for (long long i = (long long)blockIdx.x * kSwigluThreads + threadIdx.x; i < cells; i += (long long)gridDim.x * kSwigluThreads) {
    const long long row = i / f, at = row * 2 * f + (i - row * f);
    out[i] = from_f32<T>(swiglu_of<T>(to_f32<T>(y[at]), to_f32<T>(y[at + f])));
  }
}

template <class T>
__global__ __launch_bounds__(kSwigluThreads) void moe_swiglu_grad_kernel(const T* __restrict__ y, const T* __restrict__ dout,
                                                                         T* __restrict__ dy, long long cells, int f) {
  for (long long i = (long long)blockIdx.x * kSwigluThreads + threadIdx.x; i < cells; i += (long long)gridDim.x * kSwigluThreads) {
    const long long row = i / f, at = row * 2 * f + (i - row * f);
    float dg, du;
    swiglu_grad_of<T>(to_f32<T>(y[at]), to_f32<T>(y[at + f]), to_f32<T>(dout[i]), &dg, &du);
    dy[at] = from_f32<T>(dg);
    dy[at + f] = from_f32<T>(du);
  }
}

int blocks_for(long long cells) {
  const long long b = (cells + kSwigluThreads - 1) / kSwigluThreads;
  return (int)(b < 4096 ? b : 4096);
}

template <class T>
int swiglu_t(hipStream_t s, const void* y, void* out, long long rows, int f) {
  hipLaunchKernelGGL(moe_swiglu_kernel<T>, dim3(blocks_for(rows * f)), dim3(kSwigluThreads), 0, s, (const T*)y, (T*)out, rows * f, f);
  return (int)hipGetLastError();
}
template <class T>
int swiglu_grad_t(hipStream_t s, const void* y, const void* dout, void* dy, long long rows, int f) {
  hipLaunchKernelGGL(moe_swiglu_grad_kernel<T>, dim3(blocks_for(rows * f)), dim3(kSwigluThreads), 0, s, (const T*)y, (const T*)dout, (T*)dy, rows * f, f);
  return (int)hipGetLastError();
}

}  // namespace

int launch_moe_swiglu(hipStream_t s, const void* y, void* out, long long rows, int f, int elem) {
  return elem == 1 ? swiglu_t<float>(s, y, out, rows, f) : elem == 2 ? swiglu_t<f16_t>(s, y, out, rows, f) : swiglu_t<bf16_bits>(s, y, out, rows, f);
}
int launch_moe_swiglu_grad(hipStream_t s, const void* y, const void* dout, void* dy, long long rows, int f, int elem) {
  return elem == 1 ? swiglu_grad_t<float>(s, y, dout, dy, rows, f)
       : elem == 2 ? swiglu_grad_t<f16_t>(s, y, dout, dy, rows, f) : swiglu_grad_t<bf16_bits>(s, y, dout, dy, rows, f);
}

}  // namespace rd
