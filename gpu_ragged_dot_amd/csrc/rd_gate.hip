// Expert scores to expert ids and weights, and the gradient of the logits.
//
//   s = softmax(l) or sigmoid(l) over a row's E experts;  c = s + bias;  an expert with a logit or a bias of -inf is shut
//   clusters of E / C neighbours score the largest c or the sum of the two largest; all but the best `top_clusters` are shut
//   ids = the top_k largest c that are not shut, ties to the lower index; w = scale s[ids], divided by the sum of s[ids] if renormalised
//
// Which expert is larger is decided in 64 bits: a row's scores lie as close as 1e-4 of each other, and two ways to round an
// exponential to 32 bits would choose other experts for a few tokens in every batch.  Where neither a bias nor a sum of
// scores comes in, the logits' own order is the scores'.
//
// What bounds it is arithmetic, not the one read of the logits: 64-bit exponentials for every expert and a search through the
// whole row per choice took 183 us for 32768 tokens of 256 experts (sigmoid, bias, 4 of 8 clusters, top 8), 33.5 MB.  So
//  * a row is held by 16 lanes, four rows to a wave, and its ranks are made in 32 bits, as fixed-point numbers of 23 bits with the
//    expert's index behind them: one unsigned maximum compares rank and index at once, and since no two keys are equal, the next
//    smaller one is the largest of key - previous (mod 2^32) - a subtraction and half a three-way maximum per expert, nothing to remove;
//  * whether that decided what 64 bits would decide shows in the keys.  Where two neighbours among the chosen and the first one left
//    out are closer than the error of 32-bit ranks (a row in a thousand on the sizes above), those, or the leading 16, are ranked in
//    64 bits, one to a lane, and clusters by those of their two best.  Rows that this leaves open the wave does again in 64 bits.  16-bit
//    logits that rank by themselves are exact in the key: there ties are ties.
// The sizes above take 21 us so (27 with logits from memory), 1250 vector instructions a wave; 4096 tokens, where a wave's latency is most
// of it, 9.  What 16 lanes do not hold (gate_per()) takes a wave to a row, all in 64 bits: 32768 x 264 in 8 clusters 202 us, 96 in 6
// clusters 127 (in 8: 15), 768 and top 12 without clusters 138, 256 and top 17 117.
// Ranks of scores are spread over the biases' range: one finite bias of -1e9, as a mask, leaves all others too close for 32 bits, and the
// sizes above take 70 us.  A bias of -inf shuts its expert and costs nothing.
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

// A wave to a row, expert lane + 64 i in register i, everything compared in 64 bits.
template <class T, int PER>
__device__ __forceinline__ void gate_row(const T* __restrict__ logits, const float* __restrict__ bias, int32_t* __restrict__ ids,
                                         float* __restrict__ weights, const GateSpec& p, int row) {
  const int lane = threadIdx.x & 63;
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

template <class T, int PER>
__global__ __launch_bounds__(kGateThreads) void moe_gate_kernel(const T* __restrict__ logits, const float* __restrict__ bias,
                                                                int32_t* __restrict__ ids, float* __restrict__ weights, GateSpec p) {
  const int row = blockIdx.x * (kGateThreads / 64) + (threadIdx.x >> 6);
  if (row < p.tokens) gate_row<T, PER>(logits, bias, ids, weights, p, row);
}

// ---- four rows to a wave ---------------------------------------------------------------------------------------------------
// Over the 16 lanes of a row, all of which get the result.
template <int CTRL>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false); }
template <int CTRL>
__device__ __forceinline__ float from_lane(float v) { return __builtin_bit_cast(float, from_lane<CTRL>(__builtin_bit_cast(uint32_t, v))); }
constexpr int kRotate8 = 0x128, kRotate4 = 0x124, kRotate2 = 0x122, kRotate1 = 0x121;  // within rows of 16 lanes
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin32(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = umax(v, from_lane<kRotate8>(v)); v = umax(v, from_lane<kRotate4>(v));
  v = umax(v, from_lane<kRotate2>(v)); return umax(v, from_lane<kRotate1>(v));
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, from_lane<kRotate8>(v)); v = fmaxf(v, from_lane<kRotate4>(v));
  v = fmaxf(v, from_lane<kRotate2>(v)); return fmaxf(v, from_lane<kRotate1>(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += from_lane<kRotate8>(v); v += from_lane<kRotate4>(v); v += from_lane<kRotate2>(v); return v + from_lane<kRotate1>(v);
}

template <int CTRL>
__device__ __forceinline__ double from_lane(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)from_lane<CTRL>((uint32_t)b) | (uint64_t)from_lane<CTRL>((uint32_t)(b >> 32)) << 32);
}
__device__ __forceinline__ double row_max(double v) {
  v = fmax(v, from_lane<kRotate8>(v)); v = fmax(v, from_lane<kRotate4>(v));
  v = fmax(v, from_lane<kRotate2>(v)); return fmax(v, from_lane<kRotate1>(v));
}
__device__ __forceinline__ double row_sum(double v) {
  v += from_lane<kRotate8>(v); v += from_lane<kRotate4>(v); v += from_lane<kRotate2>(v); return v + from_lane<kRotate1>(v);
}

constexpr int kKeyIndexBits = 9;                       // experts of the kernel below: 512
constexpr uint32_t kKeyIndexMask = (1u << kKeyIndexBits) - 1;
constexpr float kKeyRanks = 8388608.f;                 // 2^23: what is left for the rank, 0 for experts that are shut
constexpr int kRowLanes = 16, kRowMaxTopK = 16, kRowMaxExperts = 512;

// The two largest keys of a lane, then of 2, 4, 8 or 16 neighbours.
struct Two {
  uint32_t first, second;
};
template <int CTRL>
__device__ __forceinline__ Two merge_lane(Two t) {
  const uint32_t f = from_lane<CTRL>(t.first), s = from_lane<CTRL>(t.second);
  return {umax(t.first, f), umax(umin32(t.first, f), umax(t.second, s))};
}

template <int CTRL>
__device__ __forceinline__ void merge_lane(double& first, double& second) {
  const double f = from_lane<CTRL>(first), s = from_lane<CTRL>(second);
  second = fmax(fmin(first, f), fmax(second, s));
  first = fmax(first, f);
}

// The choice in 64 bits: the expert of slot `at`, -1 for none.  Arguments as in the kernel below, `top` a row's largest logit.
template <class T, int PER>
__device__ __forceinline__ int choose_wide(const T* __restrict__ src, const float* __restrict__ bias, const GateSpec& p, int cluster_lanes,
                                           bool scored, int at, int e0, int own, float top) {
  const int lane = threadIdx.x & 63;
  double c[PER], total = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float l = i < own ? to_f32<T>(src[e0 + i]) : -INFINITY;
    c[i] = l;
    if (scored && l != -INFINITY) {
      c[i] = p.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - (double)top);
      total += c[i] == c[i] ? c[i] : 0.0;  // (NaN, also infinity less itself, would make every rank NaN)
    }
  }
  if (scored) {
    const double sum = p.sigmoid ? 1.0 : row_sum(total), by = sum > 0.0 ? sum : 1.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (c[i] == -INFINITY) continue;  // (scores are no less than 0)
      if (!p.sigmoid) c[i] /= by;
      if (bias) c[i] += bias[e0 + i];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (c[i] != c[i]) c[i] = INFINITY;  // NaN comes first, as infinity: its row's weights tell
  if (p.clusters > 1) {
    double first = -INFINITY, second = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) { second = fmax(second, fmin(first, c[i])); first = fmax(first, c[i]); }
    if (cluster_lanes >= 2) merge_lane<kSwap1>(first, second);
    if (cluster_lanes >= 4) merge_lane<kSwap2>(first, second);
    if (cluster_lanes >= 8) merge_lane<kMirror8>(first, second);
    double score = p.top2 ? first + second : first;
    if (score != score) score = INFINITY;  // (infinity and a shut expert)
    const int mine = at / cluster_lanes;
    int ahead = 0;
    for (int q = 0; q < p.clusters; ++q) {
      const double other = __shfl(score, (lane & 48) + q * cluster_lanes, 64);
      ahead += other > score || (other == score && q < mine) ? 1 : 0;
    }
    if (ahead >= p.top_clusters)
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = -INFINITY;
  }
  int id = -1;
  for (int s = 0; s < p.top_k; ++s) {
    double best = c[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = fmax(best, c[i]);
    best = row_max(best);
    uint32_t e = ~0u;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (c[i] == best) e = (uint32_t)(e0 + i);
    e = ~row_max(~e);  // the least
    if (best == -INFINITY) e = ~0u;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e == (uint32_t)(e0 + i)) c[i] = -INFINITY;
    if (at == s) id = (int)e;
  }
  return id;
}

// PER: experts a lane has registers for; `chunk` (<= PER): experts it holds, chunk * lane and on.  VEC: in whole pieces of 16 bytes.
// (PER is such pieces then.)  cluster_lanes: lanes that hold a cluster (1, 2, 4, 8 or 16).
template <class T, int PER, bool VEC>
__global__ __launch_bounds__(kGateThreads) void moe_gate_rows_kernel(const T* __restrict__ logits, const float* __restrict__ bias,
                                                                     int32_t* __restrict__ ids, float* __restrict__ weights, GateSpec p,
                                                                     int chunk, int cluster_lanes) {
  const int lane = threadIdx.x & 63, at = lane & (kRowLanes - 1);
  const int first_row = (blockIdx.x * (kGateThreads / 64) + (threadIdx.x >> 6)) * (64 / kRowLanes);
  if (first_row >= p.tokens) return;
  const int row = imin(first_row + (lane >> 4), p.tokens - 1);  // (rows past the last one do it again, and store nothing)
  const T* src = logits + (size_t)row * p.experts;
  const int e0 = at * chunk, own = imin(chunk, p.experts - e0);  // this lane's experts (own <= 0: none)
  constexpr int EPP = 16 / sizeof(T);
  float l[PER];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < PER; i += EPP) {
      alignas(16) T v[EPP];
      if (i < own) *reinterpret_cast<u32x4_t*>(v) = *reinterpret_cast<const u32x4_t*>(src + e0 + i);
#pragma unroll
      for (int e = 0; e < EPP; ++e) l[i + e] = i < own ? to_f32<T>(v[e]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) l[i] = i < own ? to_f32<T>(src[e0 + i]) : -INFINITY;
  }
  const bool scored = bias || (cluster_lanes < kRowLanes && p.top2);  // ranks are scores, not logits
  const bool exact = sizeof(T) == 2 && !scored;
  float top = l[0];
  bool odd = false;  // left to 64 bits
#pragma unroll
  for (int i = 0; i < PER; ++i) { top = fmaxf(top, l[i]); odd |= l[i] != l[i]; }
  top = row_max(top);
  odd = !exact && (odd || top == INFINITY);

  // ---- keys ----
  uint32_t key[PER];
  float closest = 0.f;  // ranks closer than this are not told apart
  if (exact) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t b = __is_same(T, f16_t) ? (uint32_t)__builtin_bit_cast(uint16_t, (f16_t)l[i]) : __builtin_bit_cast(uint32_t, l[i]) >> 16;
      const uint32_t sorted = b == 0x8000u ? 0x8000u : (b & 0x8000u) ? b ^ 0xffffu : b | 0x8000u;  // -0 is 0
      key[i] = l[i] == -INFINITY ? 0u : l[i] != l[i] ? 0xffffu : sorted;
    }
  } else {
    float low, per_rank;  // rank 0 and the ranks per unit
    if (scored) {
      float c[PER], total = 0.f, least = INFINITY, most = -INFINITY;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        c[i] = p.sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-l[i])) : __expf(l[i] - top);
        total += l[i] == -INFINITY ? 0.f : c[i];
      }
      const float norm = p.sigmoid ? 1.f : __builtin_amdgcn_rcpf(row_sum(total));
      if (bias) {
        float bs[PER];
        if constexpr (VEC) {
#pragma unroll
          for (int i = 0; i < PER; i += 4) {
            f32x4_t v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (i < own) v = load_any<f32x4_t>(bias + e0 + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) bs[i + e] = v[e];
          }
        } else {
#pragma unroll
          for (int i = 0; i < PER; ++i) bs[i] = i < own ? bias[e0 + i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float b = bs[i];
          least = b == -INFINITY ? least : fminf(least, b);
          most = fmaxf(most, b);
          odd |= !(b < INFINITY);  // NaN, infinity
          c[i] = c[i] * norm + b;
          l[i] = b == -INFINITY ? b : l[i];
        }
        least = -row_max(-least);
        most = row_max(most);
        odd |= !(least <= most);  // every expert shut by its bias
      } else {
        least = most = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] *= norm;
      }
      // 32-bit scores are good to 4e-7 (sigmoid: an argument's rounding times the slope, a quotient) or 25e-7 (softmax: the sum
      // too), a sum with the bias to its rounding, the rank to one on each side
      low = least;
      per_rank = (kKeyRanks - 8.f) / (1.f + most - least);
      closest = 4.f + 2.f * ((p.sigmoid ? 4e-7f : 25e-7f) + 1.2e-7f * (1.f + fmaxf(fabsf(least), fabsf(most)))) * per_rank;
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = l[i] == -INFINITY ? 0u : 1u + (uint32_t)fminf(fmaxf((c[i] - low) * per_rank, 0.f), kKeyRanks - 3.f);
    } else {
      low = top - 16.f;  // what lies lower has rank 1: equals, should it come to that
      per_rank = kKeyRanks / 16.f;
      closest = 4.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = l[i] == -INFINITY ? 0u : 1u + (uint32_t)fminf(fmaxf((l[i] - low) * per_rank, 0.f), kKeyRanks - 3.f);
    }
  }
  const uint32_t near = (uint32_t)fminf(closest, 1e9f);  // (twice that fits, too)
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = key[i] ? key[i] << kKeyIndexBits | (kKeyIndexMask - (uint32_t)(e0 + i)) : 0u;

  auto expert_of = [](uint32_t k) { return k ? (int)(kKeyIndexMask - (k & kKeyIndexMask)) : -1; };
  // The rank of expert e in 64 bits, and the sum that softmax ranks take.
  auto wide_total = [&]() {
    if (!scored || p.sigmoid) return 1.0;
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float x = i < own ? to_f32<T>(src[e0 + i]) : -INFINITY;
      if (x > -INFINITY) total += exp((double)x - (double)top);  // (a row with NaN is odd)
    }
    return row_sum(total);
  };
  auto wide_rank = [&](int e, double total) -> double {
    if (e < 0) return -INFINITY;
    const double x = to_f32<T>(src[e]);
    const double v = !scored ? x : p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double)top) / total;
    return bias ? v + bias[e] : v;
  };

  // ---- clusters ----
  if (p.clusters > 1) {
    Two t = {0u, 0u};
#pragma unroll
    for (int i = 0; i < PER; ++i) { t.second = umax(t.second, umin32(t.first, key[i])); t.first = umax(t.first, key[i]); }
    if (cluster_lanes >= 2) t = merge_lane<kSwap1>(t);
    if (cluster_lanes >= 4) t = merge_lane<kSwap2>(t);
    if (cluster_lanes >= 8) t = merge_lane<kMirror8>(t);
    const uint32_t q1 = t.first >> kKeyIndexBits, q2 = t.second >> kKeyIndexBits;
    const uint32_t score = !p.top2 ? q1 : q2 ? q1 + q2 : 0u;  // (a sum with a shut expert is -inf)
    const int mine = at / cluster_lanes;
    int ahead = 0;
    for (int q = 0; q < p.clusters; ++q) {
      const uint32_t other = (uint32_t)__shfl((int)score, (lane & 48) + q * cluster_lanes, 64);
      ahead += other > score || (other == score && q < mine) ? 1 : 0;
    }
    if (!exact && p.top_clusters < p.clusters) {  // the worst of those kept against the best of the others
      const uint32_t worst = ~row_max(ahead < p.top_clusters && mine < p.clusters ? ~score : 0u);
      const uint32_t best = row_max(ahead >= p.top_clusters && mine < p.clusters ? score : 0u);
      const bool close = worst - best <= (p.top2 ? 2 * near : near);
      // Close ones in some row: by the ranks of each cluster's two best in 64 bits, if no third one comes into question.
      if (__ballot(close)) {
        uint32_t third = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) third = umax(third, key[i] - t.second);
        if (cluster_lanes >= 2) third = umax(third, from_lane<kSwap1>(third));
        if (cluster_lanes >= 4) third = umax(third, from_lane<kSwap2>(third));
        if (cluster_lanes >= 8) third = umax(third, from_lane<kMirror8>(third));
        third = t.second ? third + t.second : 0u;
        const bool questionable = third && (p.top2 ? q2 : q1) - (third >> kKeyIndexBits) <= near;
        odd |= close && row_max(questionable ? 1u : 0u) != 0u;
        const double total = wide_total();
        const double v1 = wide_rank(expert_of(t.first), total), v2 = wide_rank(expert_of(t.second), total);
        const double exact_score = p.top2 ? v1 + v2 : fmax(v1, v2);
        int exact_ahead = 0;
        for (int q = 0; q < p.clusters; ++q) {
          const double other = __shfl(exact_score, (lane & 48) + q * cluster_lanes, 64);
          exact_ahead += other > exact_score || (other == exact_score && q < mine) ? 1 : 0;
        }
        if (close) ahead = exact_ahead;
      }
    }
    if (ahead >= p.top_clusters)
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = 0u;
  }

  // ---- the top_k largest keys and the one behind them, slot s in lane s ----
  uint32_t previous = ~0u, chosen = 0u;  // (no key is as large: ranks end at 2^23 - 2)
  auto next_key = [&]() {  // the largest key - previous, which has wrapped around for every smaller key
    uint32_t below = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) below = umax(below, key[i] - previous);
    return previous ? row_max(below) + previous : 0u;
  };
  bool close = false;
  for (int s = 0; s <= p.top_k; ++s) {
    const uint32_t next = next_key();
    close |= s > 0 && next != 0u && (previous >> kKeyIndexBits) - (next >> kKeyIndexBits) <= near;
    if (at == s) chosen = next;
    previous = next;
  }
  close = close && !exact;
  // Close ones in some row: those chosen and the first left out by their ranks in 64 bits, one to a lane; where that one is close
  // to the last chosen, as many more as there are lanes, if the last of them is out of the question.
  if (__ballot(close)) {
    const uint32_t kth = (uint32_t)__shfl((int)chosen, (lane & 48) + p.top_k - 1, 64) >> kKeyIndexBits;
    auto out_of_question = [&]() { return previous == 0u || kth - (previous >> kKeyIndexBits) > near; };
    if (__ballot(close && !out_of_question()))
      for (int s = p.top_k + 1; s < kRowLanes; ++s) {
        previous = next_key();
        if (at == s) chosen = previous;
      }
    const bool settled = out_of_question();
    odd |= close && !settled;
    const int e = expert_of(chosen);
    const double v = wide_rank(e, wide_total());
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    int ahead = 0;
    for (int q = 0; q < kRowLanes; ++q) {
      const int from = (lane & 48) + q;
      const uint64_t ob = (uint64_t)(uint32_t)__shfl((int)(uint32_t)bits, from, 64) | (uint64_t)(uint32_t)__shfl((int)(uint32_t)(bits >> 32), from, 64) << 32;
      const double other = __builtin_bit_cast(double, ob);
      const int oe = __shfl(e, from, 64);
      ahead += other > v || (other == v && (oe < e || (oe == e && q < at))) ? 1 : 0;  // (those that are none, among themselves by lane)
    }
    const uint32_t sorted = (uint32_t)__builtin_amdgcn_ds_permute(((lane & 48) + ahead) << 2, (int)chosen);
    if (settled) chosen = sorted;
  }
  int id = at < p.top_k ? expert_of(chosen) : -1;
  if (__ballot(odd)) id = choose_wide<T, PER>(src, bias, p, cluster_lanes, scored, at, e0, own, top);

  // ---- weights ----
  const float logit = id >= 0 ? to_f32<T>(src[id]) : -INFINITY;
  float w = 0.f;
  if (p.renormalize) {
    // relative to the largest chosen one, so that scores too small for 32 bits divide all the same
    const float most = p.sigmoid ? fminf(row_max(logit), 0.f) : row_max(logit);
    if (id >= 0) w = !p.sigmoid ? expf(logit - most) : logit > 0.f ? 1.f / (1.f + expf(-logit)) : expf(logit - most) / (1.f + expf(logit));
    const float sum = row_sum(w);
    w = id >= 0 ? p.scale * (w / sum) : 0.f;
  } else if (p.sigmoid) {
    w = id >= 0 ? p.scale / (1.f + expf(-logit)) : 0.f;
  } else {
    float sum = 0.f;
    if (bias) {  // (an expert that its bias shuts still counts in the softmax)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < own) l[i] = to_f32<T>(src[e0 + i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += l[i] == -INFINITY ? 0.f : expf(l[i] - top);
    sum = row_sum(sum);
    w = id >= 0 ? p.scale * (expf(logit - top) / sum) : 0.f;
  }
  const bool live = first_row + (lane >> 4) < p.tokens;
  if (live && at < p.top_k) {
    ids[(size_t)row * p.top_k + at] = id;
    weights[(size_t)row * p.top_k + at] = w;
  }
}

// With q_i = w_i dw_i and Q their sum over a row's choices:
//   renormalised: dl_i = (q_i - w_i / scale Q) (1 - s_i for sigmoid), chosen ones only;
//   sigmoid: dl_i = q_i (1 - s_i);  softmax: dl_j = [j chosen] q_j - s_j Q for every expert.
template <class T, int PER>
__global__ __launch_bounds__(kGateThreads) void moe_gate_grad_kernel(const T* __restrict__ logits, const int32_t* __restrict__ ids,
                                                                     const float* __restrict__ weights, const float* __restrict__ dweights,
                                                                     T* __restrict__ dlogits, GateSpec p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * (kGateThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.tokens) return;
  const T* src = logits + (size_t)row * p.experts;
  const int given = lane < p.top_k ? ids[(size_t)row * p.top_k + lane] : -1, id = given < p.experts ? given : -1;
  const float w = id >= 0 ? weights[(size_t)row * p.top_k + lane] : 0.f;
  const float q = id >= 0 ? w * dweights[(size_t)row * p.top_k + lane] : 0.f;
  const float Q = wave_sum(q);
  float g = q;
  if (p.renormalize) g = q - w / p.scale * Q;  // (0 where one choice has it all)
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

// The same with 16 lanes to a row, four rows to a wave: a choice per lane, the row put together in LDS and stored in pieces of 16
// bytes.  10 us on 32768 x 256 float32, 33.5 MB.  (A wave to a row and every choice held against every expert: 16.)
template <class T>
__global__ __launch_bounds__(kGateThreads) void moe_gate_rows_grad_kernel(const T* __restrict__ logits, const int32_t* __restrict__ ids,
                                                                          const float* __restrict__ weights, const float* __restrict__ dweights,
                                                                          T* __restrict__ dlogits, GateSpec p) {
  constexpr int EPP = 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) float rows[kGateThreads / kRowLanes][kRowMaxExperts + 16];  // (a wave's four rows in banks of their own)
  const int at = threadIdx.x & (kRowLanes - 1), mine = threadIdx.x / kRowLanes;
  const int want = blockIdx.x * (kGateThreads / kRowLanes) + mine, row = imin(want, p.tokens - 1);
  float* d = rows[mine];
  const int given = at < p.top_k ? ids[(size_t)row * p.top_k + at] : -1, id = given < p.experts ? given : -1;
  const float w = id >= 0 ? weights[(size_t)row * p.top_k + at] : 0.f;
  const float q = id >= 0 ? w * dweights[(size_t)row * p.top_k + at] : 0.f;
  const float Q = row_sum(q);
  const T* src = logits + (size_t)row * p.experts;
  float g = q;
  if (p.renormalize) g = q - w / p.scale * Q;  // (0 where one choice has it all)
  if (p.sigmoid && id >= 0) g /= 1.f + expf(to_f32<T>(src[id]));
  if (!p.sigmoid && !p.renormalize) {
    float top = -INFINITY, sum = 0.f;
    for (int e = at; e < p.experts; e += kRowLanes) {
      d[e] = to_f32<T>(src[e]);
      top = fmaxf(top, d[e]);
    }
    top = row_max(top);
    for (int e = at; e < p.experts; e += kRowLanes) {
      d[e] = d[e] == -INFINITY ? 0.f : expf(d[e] - top);
      sum += d[e];
    }
    sum = row_sum(sum);
    for (int e = at; e < p.experts; e += kRowLanes) d[e] = sum > 0.f ? -(d[e] / sum) * Q : sum;
  } else {
    for (int e = at * 4; e < p.experts; e += kRowLanes * 4) *reinterpret_cast<f32x4_t*>(d + e) = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  if (id >= 0) d[id] += g;  // (a row's choices are distinct)
  __syncthreads();
  if (want >= p.tokens) return;
  T* dst = dlogits + (size_t)row * p.experts;
  for (int e = at * EPP; e < p.experts; e += kRowLanes * EPP) {
    alignas(16) T v[EPP];
#pragma unroll
    for (int i = 0; i < EPP; ++i) v[i] = from_f32<T>(d[e + i]);  // (past the row's end: still LDS, not stored)
    if (e + EPP <= p.experts) store_any(dst + e, *reinterpret_cast<u32x4_t*>(v));
    else
#pragma unroll
      for (int i = 0; i < EPP - 1; ++i)
        if (e + i < p.experts) dst[e + i] = v[i];
  }
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

template <class T, int PER>
int gate_rows_t(hipStream_t s, const void* logits, const float* bias, int32_t* ids, float* weights, const GateSpec& p, int chunk, int cluster_lanes) {
  const int rows = kGateThreads / kRowLanes;
  const dim3 grid((p.tokens + rows - 1) / rows);
  if constexpr (PER * sizeof(T) >= 16) {
    if (chunk * sizeof(T) % 16 == 0 && (size_t)p.experts * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0) {
      hipLaunchKernelGGL((moe_gate_rows_kernel<T, PER, true>), grid, dim3(kGateThreads), 0, s, (const T*)logits, bias, ids, weights, p, chunk, cluster_lanes);
      return (int)hipGetLastError();
    }
  }
  hipLaunchKernelGGL((moe_gate_rows_kernel<T, PER, false>), grid, dim3(kGateThreads), 0, s, (const T*)logits, bias, ids, weights, p, chunk, cluster_lanes);
  return (int)hipGetLastError();
}

// Sixteen lanes to a row where they hold it: up to 512 experts, 16 choices, and clusters that are one, two, four or eight lanes'.
template <class T>
int gate_per(hipStream_t s, GateSpec p, const void* logits, const float* bias, int32_t* ids, float* weights) {
  const int size = p.experts / p.clusters, chunk = (p.experts + kRowLanes - 1) / kRowLanes;
  if (size == 1 || p.clusters == 1) p.top2 = false;  // one expert's sum is its rank
  const int lanes = p.clusters == 1 ? kRowLanes : size % chunk == 0 ? size / chunk : 0;
  if (p.experts <= kRowMaxExperts && p.top_k <= kRowMaxTopK && (lanes == 1 || lanes == 2 || lanes == 4 || lanes == 8 || lanes == 16))
    return chunk <= 1 ? gate_rows_t<T, 1>(s, logits, bias, ids, weights, p, chunk, lanes)
         : chunk <= 4 ? gate_rows_t<T, 4>(s, logits, bias, ids, weights, p, chunk, lanes)
         : chunk <= 8 ? gate_rows_t<T, 8>(s, logits, bias, ids, weights, p, chunk, lanes)
         : chunk <= 16 ? gate_rows_t<T, 16>(s, logits, bias, ids, weights, p, chunk, lanes)
                       : gate_rows_t<T, 32>(s, logits, bias, ids, weights, p, chunk, lanes);
  return p.experts <= 64 ? gate_t<T, 1>(s, logits, bias, ids, weights, p) : p.experts <= 128 ? gate_t<T, 2>(s, logits, bias, ids, weights, p)
       : p.experts <= 256 ? gate_t<T, 4>(s, logits, bias, ids, weights, p) : p.experts <= 512 ? gate_t<T, 8>(s, logits, bias, ids, weights, p)
                                                                                          : gate_t<T, 16>(s, logits, bias, ids, weights, p);
}
template <class T>
int gate_grad_per(hipStream_t s, const GateSpec& p, const void* logits, const int32_t* ids, const float* w, const float* dw, void* dl) {
  if (p.experts <= kRowMaxExperts && p.top_k <= kRowMaxTopK) {
    const int rows = kGateThreads / kRowLanes;
    hipLaunchKernelGGL((moe_gate_rows_grad_kernel<T>), dim3((p.tokens + rows - 1) / rows), dim3(kGateThreads), 0, s, (const T*)logits, ids, w, dw, (T*)dl, p);
    return (int)hipGetLastError();
  }
  return p.experts <= 64 ? gate_grad_t<T, 1>(s, logits, ids, w, dw, dl, p) : p.experts <= 128 ? gate_grad_t<T, 2>(s, logits, ids, w, dw, dl, p)
       : p.experts <= 256 ? gate_grad_t<T, 4>(s, logits, ids, w, dw, dl, p) : p.experts <= 512 ? gate_grad_t<T, 8>(s, logits, ids, w, dw, dl, p)
                                                                                          : gate_grad_t<T, 16>(s, logits, ids, w, dw, dl, p);
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
