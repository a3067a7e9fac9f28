// The gated activation between an expert's two products: rows [gate | up] of 2 f elements -> silu(gate) * up, and its gradient.
//
//   out = g sig(g) u;  dg = dout u sig(g) (1 + g (1 - sig(g)));  du = dout g sig(g)
//
// Bound by memory: 3 f elements of a row forward, 5 f backward, each touched once.  32768 x 2048 bf16: forward 74 us (5.4 TB/s),
// backward 111 us (6.0 TB/s); a copy reaches 4.9.
#include "rd_elem.h"
#include "rd_moe.h"

namespace rd {

namespace {

constexpr int kSwigluThreads = 256;

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

// A row is cut into pieces of 16 bytes, at whatever address they have; the last one begins early enough to end with the row, so
// that up to PER - 1 cells are computed twice, with the same bits.  (By element, as rows narrower than a piece still are: 264 us on
// 32768 x 2048 bf16 forward and backward, in pieces 188.)
template <class T>
struct Piece {
  static constexpr int PER = 16 / sizeof(T);
  alignas(16) T e[PER];
  __device__ __forceinline__ void load(const T* p) { *reinterpret_cast<u32x4_t*>(e) = load_any<u32x4_t>(p); }
  __device__ __forceinline__ void store(T* p) const { store_any(p, *reinterpret_cast<const u32x4_t*>(e)); }
};

struct PieceAt {
  long long row;
  int col;
};
// 32-bit arithmetic behind one 64-bit division per work-group: `in_row` pieces behind the start of row0.
__device__ __forceinline__ PieceAt piece_at(long long row0, uint32_t in_row, uint32_t per_row, int f, int per) {
  const uint32_t down = in_row / per_row;
  return {row0 + down, imin((int)(in_row - down * per_row) * per, f - per)};
}

template <class T, int U>
__global__ __launch_bounds__(kSwigluThreads) void moe_swiglu_kernel(const T* __restrict__ y, T* __restrict__ out, long long pieces, int f) {
  constexpr int PER = Piece<T>::PER;
  const uint32_t per_row = (uint32_t)(f + PER - 1) / PER;
  const long long first = (long long)blockIdx.x * (kSwigluThreads * U), row0 = first / per_row;
  const uint32_t in_row = (uint32_t)(first - row0 * per_row) + threadIdx.x;
  Piece<T> g[U], u[U];
  PieceAt at[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (first + threadIdx.x + i * kSwigluThreads >= pieces) break;
    at[i] = piece_at(row0, in_row + i * kSwigluThreads, per_row, f, PER);
    g[i].load(y + at[i].row * 2 * f + at[i].col);
    u[i].load(y + at[i].row * 2 * f + f + at[i].col);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (first + threadIdx.x + i * kSwigluThreads >= pieces) break;
#pragma unroll
    for (int e = 0; e < PER; ++e) g[i].e[e] = from_f32<T>(swiglu_of<T>(to_f32<T>(g[i].e[e]), to_f32<T>(u[i].e[e])));
    g[i].store(out + at[i].row * f + at[i].col);
  }
}

template <class T, int U>
__global__ __launch_bounds__(kSwigluThreads) void moe_swiglu_grad_kernel(const T* __restrict__ y, const T* __restrict__ dout,
                                                                         T* __restrict__ dy, long long pieces, int f) {
  constexpr int PER = Piece<T>::PER;
  const uint32_t per_row = (uint32_t)(f + PER - 1) / PER;
  const long long first = (long long)blockIdx.x * (kSwigluThreads * U), row0 = first / per_row;
  const uint32_t in_row = (uint32_t)(first - row0 * per_row) + threadIdx.x;
  Piece<T> g[U], u[U], d[U];
  PieceAt at[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (first + threadIdx.x + i * kSwigluThreads >= pieces) break;
    at[i] = piece_at(row0, in_row + i * kSwigluThreads, per_row, f, PER);
    g[i].load(y + at[i].row * 2 * f + at[i].col);
    u[i].load(y + at[i].row * 2 * f + f + at[i].col);
    d[i].load(dout + at[i].row * f + at[i].col);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (first + threadIdx.x + i * kSwigluThreads >= pieces) break;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      float dg, du;
      swiglu_grad_of<T>(to_f32<T>(g[i].e[e]), to_f32<T>(u[i].e[e]), to_f32<T>(d[i].e[e]), &dg, &du);
      g[i].e[e] = from_f32<T>(dg);
      u[i].e[e] = from_f32<T>(du);
    }
    g[i].store(dy + at[i].row * 2 * f + at[i].col);
    u[i].store(dy + at[i].row * 2 * f + f + at[i].col);
  }
}

// Rows narrower than a piece, a cell per thread.
template <class T>
__global__ __launch_bounds__(kSwigluThreads) void moe_swiglu_narrow_kernel(const T* __restrict__ y, T* __restrict__ out, long long cells, int f) {
  for (long long i = (long long)blockIdx.x * kSwigluThreads + threadIdx.x; i < cells; i += (long long)gridDim.x * kSwigluThreads) {
    const long long row = i / f, at = row * 2 * f + (i - row * f);
    out[i] = from_f32<T>(swiglu_of<T>(to_f32<T>(y[at]), to_f32<T>(y[at + f])));
  }
}
template <class T>
__global__ __launch_bounds__(kSwigluThreads) void moe_swiglu_narrow_grad_kernel(const T* __restrict__ y, const T* __restrict__ dout,
                                                                                T* __restrict__ dy, long long cells, int f) {
  for (long long i = (long long)blockIdx.x * kSwigluThreads + threadIdx.x; i < cells; i += (long long)gridDim.x * kSwigluThreads) {
    const long long row = i / f, at = row * 2 * f + (i - row * f);
    float dg, du;
    swiglu_grad_of<T>(to_f32<T>(y[at]), to_f32<T>(y[at + f]), to_f32<T>(dout[i]), &dg, &du);
    dy[at] = from_f32<T>(dg);
    dy[at + f] = from_f32<T>(du);
  }
}

// Pieces per thread: one while that many work-groups do not fill the device, then several loads in flight.
constexpr long long kFewPieces = 256ll * kSwigluThreads * 8;

dim3 blocks_for(long long work, int per_block) { return dim3((unsigned)((work + per_block - 1) / per_block)); }
template <class T>
long long pieces_of(long long rows, int f) { return rows * ((f + Piece<T>::PER - 1) / Piece<T>::PER); }

template <class T>
int swiglu_t(hipStream_t s, const void* y_, void* out_, long long rows, int f) {
  const T* y = (const T*)y_;
  T* out = (T*)out_;
  const long long pieces = pieces_of<T>(rows, f);
  if (f < Piece<T>::PER) hipLaunchKernelGGL((moe_swiglu_narrow_kernel<T>), dim3(1024), dim3(kSwigluThreads), 0, s, y, out, rows * f, f);
  else if (pieces <= kFewPieces) hipLaunchKernelGGL((moe_swiglu_kernel<T, 1>), blocks_for(pieces, kSwigluThreads), dim3(kSwigluThreads), 0, s, y, out, pieces, f);
  else hipLaunchKernelGGL((moe_swiglu_kernel<T, 4>), blocks_for(pieces, kSwigluThreads * 4), dim3(kSwigluThreads), 0, s, y, out, pieces, f);
  return (int)hipGetLastError();
}
template <class T>
int swiglu_grad_t(hipStream_t s, const void* y_, const void* dout_, void* dy_, long long rows, int f) {
  const T *y = (const T*)y_, *dout = (const T*)dout_;
  T* dy = (T*)dy_;
  const long long pieces = pieces_of<T>(rows, f);
  if (f < Piece<T>::PER) hipLaunchKernelGGL((moe_swiglu_narrow_grad_kernel<T>), dim3(1024), dim3(kSwigluThreads), 0, s, y, dout, dy, rows * f, f);
  else if (pieces <= kFewPieces) hipLaunchKernelGGL((moe_swiglu_grad_kernel<T, 1>), blocks_for(pieces, kSwigluThreads), dim3(kSwigluThreads), 0, s, y, dout, dy, pieces, f);
  else hipLaunchKernelGGL((moe_swiglu_grad_kernel<T, 2>), blocks_for(pieces, kSwigluThreads * 2), dim3(kSwigluThreads), 0, s, y, dout, dy, pieces, f);
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
