// Expert scores to expert ids and weights, and the gradient of the logits.
//
//   s = softmax(l) or sigmoid(l) over a row's E experts;  c = s + bias;  an expert with a logit or a bias of -inf is shut
//   clusters of E / C neighbours score the largest c or the sum of the two largest; all but the best `top_clusters` are shut
//   ids = the top_k largest c that are not shut, ties to the lower index; w = scale s[ids], divided by the sum of s[ids] if renormalised
//
// Which expert is larger is decided in 64 bits: a row's scores lie as close as 1e-4 of each other, and two ways to round an
// exponential to 32 bits would choose other experts for a few tokens in every batch.  Where neither a bias nor a sum of
// scores comes in, the logits' own order is the scores'.
#include "rd_elem.h"
#include "rd_moe.h"

namespace rd {

namespace {

constexpr int kGateThreads = 256;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
template <class V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The largest value of the wave and its lowest index.
__device__ __forceinline__ void wave_best(double& v, int& at) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const double v2 = __shfl_xor(v, o, 64);
    const int at2 = __shfl_xor(at, o, 64);
    if (v2 > v || (v2 == v && at2 < at)) { v = v2; at = at2; }
  }
}

// A wave to a row, expert lane + 64 i in register i.
template <class T, int PER>
__global__ __launch_bounds__(kGateThreads) void moe_gate_kernel(const T* __restrict__ logits, const float* __restrict__ bias,
                                                                int32_t* __restrict__ ids, float* __restrict__ weights, GateSpec p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * (kGateThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.tokens) return;
  const T* src = logits + (size_t)row * p.experts;
  float l[PER];
  double c[PER];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    l[i] = e < p.experts ? to_f32<T>(src[e]) : -INFINITY;
    c[i] = l[i];
    top = fmaxf(top, l[i]);
  }
  top = wave_max(top);
  if (bias || (p.clusters > 1 && p.top2)) {
    double total = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = p.sigmoid ? 1.0 / (1.0 + exp(-(double)l[i])) : exp((double)l[i] - (double)top);
      total += c[i] == c[i] ? c[i] : 0.0;  // (NaN, also infinity less itself, would make every rank NaN)
    }
    if (!p.sigmoid) total = wave_sum(total);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 64 * i;
      if (!p.sigmoid && total > 0.0) c[i] /= total;
      if (bias && e < p.experts) c[i] += bias[e];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (c[i] != c[i]) c[i] = INFINITY;  // NaN comes first, as infinity: its row's weights tell
    if (l[i] == -INFINITY) c[i] = -INFINITY;
  }
  if (p.clusters > 1) {
    const int size = p.experts / p.clusters;
    double mine = -INFINITY;  // the score of cluster `lane`
    int ahead_of_mine = 0;
    for (int q = 0; q < p.clusters; ++q) {
      double sum = 0;
      int first = -1;
      for (int b = 0; b < (p.top2 && size > 1 ? 2 : 1); ++b) {
        double v = -INFINITY;
        int at = kGateMaxExperts;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int e = lane + 64 * i;
          if (e >= q * size && e < (q + 1) * size && e != first && (c[i] > v || at == kGateMaxExperts)) { v = c[i]; at = e; }
        }
        wave_best(v, at);
        sum += v;
        first = at;
      }
      if (lane == q) mine = sum == sum ? sum : INFINITY;  // (infinity and a shut expert)
    }
    for (int q = 0; q < p.clusters; ++q) {
      const double v = __shfl(mine, q, 64);
      const bool ahead = lane < p.clusters && (v > mine || (v == mine && q < lane));
      ahead_of_mine += ahead ? 1 : 0;
    }
    const unsigned long long open = __ballot(lane < p.clusters && ahead_of_mine < p.top_clusters);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 64 * i;
      if (e < p.experts && !((open >> (e / size)) & 1)) c[i] = -INFINITY;
    }
  }
  float my_logit = -INFINITY;  // of the choice in slot `lane`
  int my_id = -1;
  for (int s = 0; s < p.top_k; ++s) {
    double v = -INFINITY;
    int at = kGateMaxExperts;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (c[i] > v) { v = c[i]; at = lane + 64 * i; }
    wave_best(v, at);
    if (at == kGateMaxExperts) break;  // none left that is not shut
    float chosen = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == lane + 64 * i) { c[i] = -INFINITY; chosen = l[i]; }
    chosen = __shfl(chosen, at & 63, 64);
    if (lane == s) { my_id = at; my_logit = chosen; }
  }
  // the weights, in 32 bits
  float w = 0;
  if (p.renormalize) {
    // relative to the largest chosen one, so that scores too small for 32 bits divide all the same
    const float most = p.sigmoid ? fminf(wave_max(my_logit), 0.f) : wave_max(my_logit);
    if (my_id >= 0) w = !p.sigmoid ? expf(my_logit - most) : my_logit > 0.f ? 1.f / (1.f + expf(-my_logit)) : expf(my_logit - most) / (1.f + expf(my_logit));
    const float sum = wave_sum(w);
    w = my_id >= 0 ? p.scale * (w / sum) : 0.f;
  } else if (p.sigmoid) {
    w = my_id >= 0 ? p.scale / (1.f + expf(-my_logit)) : 0.f;
  } else {
    float sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += l[i] == -INFINITY ? 0.f : expf(l[i] - top);
    sum = wave_sum(sum);
    w = my_id >= 0 ? p.scale * (expf(my_logit - top) / sum) : 0.f;
  }
  if (lane < p.top_k) {
    ids[(size_t)row * p.top_k + lane] = my_id;
    weights[(size_t)row * p.top_k + lane] = w;
  }
}

// With q_i = w_i dw_i and Q their sum over a row's choices:
//   renormalised: dl_i = (q_i - w_i Q / scale) (1 - s_i for sigmoid), chosen ones only;
//   sigmoid: dl_i = q_i (1 - s_i);  softmax: dl_j = [j chosen] q_j - s_j Q for every expert.
template <class T, int PER>
__global__ __launch_bounds__(kGateThreads) void moe_gate_grad_kernel(const T* __restrict__ logits, const int32_t* __restrict__ ids,
                                                                     const float* __restrict__ weights, const float* __restrict__ dweights,
                                                                     T* __restrict__ dlogits, GateSpec p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * (kGateThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.tokens) return;
  const T* src = logits + (size_t)row * p.experts;
  const bool slot = lane < p.top_k;
  const int id = slot ? ids[(size_t)row * p.top_k + lane] : -1;
  const float w = id >= 0 ? weights[(size_t)row * p.top_k + lane] : 0.f;
  const float q = id >= 0 ? w * dweights[(size_t)row * p.top_k + lane] : 0.f;
  const float Q = wave_sum(q);
  float g = q;
  if (p.renormalize) g = q - w * (Q / p.scale);
  if (p.sigmoid && id >= 0) g /= 1.f + expf(to_f32<T>(src[id]));
  float d[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) d[i] = 0.f;
  if (!p.sigmoid && !p.renormalize) {
    float top = -INFINITY, sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      d[i] = lane + 64 * i < p.experts ? to_f32<T>(src[lane + 64 * i]) : -INFINITY;
      top = fmaxf(top, d[i]);
    }
    top = wave_max(top);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      d[i] = d[i] == -INFINITY ? 0.f : expf(d[i] - top);
      sum += d[i];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) d[i] = sum > 0.f ? -(d[i] / sum) * Q : sum;
  }
  for (int s = 0; s < p.top_k; ++s) {
    const int e = __shfl(id, s, 64);
    const float v = __shfl(g, s, 64);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e == lane + 64 * i) d[i] += v;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < p.experts) dlogits[(size_t)row * p.experts + lane + 64 * i] = from_f32<T>(d[i]);
}

template <class T, int PER>
int gate_t(hipStream_t s, const void* logits, const float* bias, int32_t* ids, float* weights, const GateSpec& p) {
  const int rows = kGateThreads / 64;
  hipLaunchKernelGGL((moe_gate_kernel<T, PER>), dim3((p.tokens + rows - 1) / rows), dim3(kGateThreads), 0, s, (const T*)logits, bias, ids, weights, p);
  return (int)hipGetLastError();
}
template <class T, int PER>
int gate_grad_t(hipStream_t s, const void* logits, const int32_t* ids, const float* w, const float* dw, void* dl, const GateSpec& p) {
  const int rows = kGateThreads / 64;
  hipLaunchKernelGGL((moe_gate_grad_kernel<T, PER>), dim3((p.tokens + rows - 1) / rows), dim3(kGateThreads), 0, s, (const T*)logits, ids, w, dw, (T*)dl, p);
  return (int)hipGetLastError();
}

template <class T, class... A>
int gate_per(hipStream_t s, const GateSpec& p, A... a) {
  return p.experts <= 64 ? gate_t<T, 1>(s, a..., p) : p.experts <= 128 ? gate_t<T, 2>(s, a..., p)
       : p.experts <= 256 ? gate_t<T, 4>(s, a..., p) : p.experts <= 512 ? gate_t<T, 8>(s, a..., p) : gate_t<T, 16>(s, a..., p);
}
template <class T, class... A>
int gate_grad_per(hipStream_t s, const GateSpec& p, A... a) {
  return p.experts <= 64 ? gate_grad_t<T, 1>(s, a..., p) : p.experts <= 128 ? gate_grad_t<T, 2>(s, a..., p)
       : p.experts <= 256 ? gate_grad_t<T, 4>(s, a..., p) : p.experts <= 512 ? gate_grad_t<T, 8>(s, a..., p) : gate_grad_t<T, 16>(s, a..., p);
}

}  // namespace

int launch_moe_gate(hipStream_t s, const void* logits, const float* bias, int32_t* ids, float* weights, const GateSpec& p) {
  return p.elem == 1 ? gate_per<float>(s, p, logits, bias, ids, weights)
       : p.elem == 2 ? gate_per<f16_t>(s, p, logits, bias, ids, weights)
                     : gate_per<bf16_bits>(s, p, logits, bias, ids, weights);
}

int launch_moe_gate_grad(hipStream_t s, const void* logits, const int32_t* ids, const float* weights, const float* dweights,
                         void* dlogits, const GateSpec& p) {
  return p.elem == 1 ? gate_grad_per<float>(s, p, logits, ids, weights, dweights, dlogits)
       : p.elem == 2 ? gate_grad_per<f16_t>(s, p, logits, ids, weights, dweights, dlogits)
                     : gate_grad_per<bf16_bits>(s, p, logits, ids, weights, dweights, dlogits);
}

}  // namespace rd
