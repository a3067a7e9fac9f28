// GEMM core of the ragged product on 4-bit weights, for groups of many rows: y[t, c] = sum_kk x[t, kk] A[kk, c] with A =
// scale (q - zero) made from its codes (layout in rd_int4.h) on the way into LDS.
//
// A tile of BM x 256 held by a 2 x 2 grid of waves, in 64-wide slabs; x goes HBM -> registers -> LDS as in rd_gemm_rs.h, at any
// pitch and address, two slabs in LDS and two in registers.  A lane owns four pieces of a run of 128 indices (16 bytes, 32 codes,
// each), with two runs in registers, and turns half of each into 16-bit weights per slab: eight words to 128 bytes of LDS, in the
// chunk order that the fragment reads undo.  So a code is converted once per row tile and not once per wave.
//  * A word costs 17 vector instructions (float16 rows: 13).  An and-or makes the float16 numbers 1024 + q or 64 + q of a pair of codes,
//    for half of the pairs without a shift, and the fused multiply-add of mixed types takes them as they are: scale v - scale (1024 +
//    zero), whose terms have 22 bits at most, so that the difference is exact.  (A conversion of bytes each: 23.)
//  * What a wave does beside matrix-core instructions is dealt out over the gaps between them, which leave seven issue slots each, by
//    the slots that it takes (schedule() below): 400 slots a slab beside 64 instructions of eight, for BM 256.  What bounds the kernel
//    is the power that the matrix cores draw, first, and these slots.  bf16 (float16), 8 groups of 2048 x 4096 x 14336, us: 1905
//    (1955) with byte conversions, writes to LDS two lanes to a bank and an op to a gap whatever it takes; 1850 (1845, and 0.4 % for what
//    trim_b() clears) as it is.
//  * The weight is rounded to the rows' type, once: scale (q - zero) itself is exact in fp32 (scale has at most 11 bits, the
//    difference 9).  Kept exact, as in the streaming kernel, the sums of every block would have to be scaled apart - three vector
//    instructions per accumulator and block of 128, more than the matrix-core instructions leave.
#pragma once
#include <utility>
#include "rd_gemm_rs.h"
#include "rd_int4.h"

namespace rd {

template <int BM_, bool HALF_, int BLOCK_>
struct Int4TileCfg {
  typedef typename std::conditional<HALF_, f16_t, bf16_bits>::type Elem;
  static constexpr bool HALF = HALF_;
  static constexpr int BM = BM_, BN = 256, BK = 64, BLOCK = BLOCK_, NW = 4, NT = 256;
  static constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, SLOT_BYTES = A_BYTES + B_BYTES;
  static constexpr int EPI_PITCH = WN * 2 + 16, EPI_BYTES = NW * WM * EPI_PITCH;
  static constexpr int LDS_BYTES = 2 * SLOT_BYTES > EPI_BYTES ? 2 * SLOT_BYTES : EPI_BYTES;
  static constexpr int PER_RUN = kInt4Run / BLOCK;  // scales of a column per run
  static constexpr bool DLDS = true;  // (splitk_combine(): four waves with many accumulators take 16 vectors of two pieces at a time)
  static_assert(BM % 64 == 0 && LDS_BYTES <= 160 * 1024, "tile shape");
};

// What a tile reads of the weights.
struct Int4Columns {
  const char* codes;   // of the tile's first strip and first run
  const char* scales;  // of the group's first run, column 0
  const char* zeros;   // the same; where there are none, any memory as large
  int first, n;        // the tile's first column; columns of the matrix
  int runs, stride;    // the tile's runs; runs from one strip to the next
  bool has_zeros, scale_half;
};

namespace int4_detail {
template <int V>
struct Int { static constexpr int value = V; };

template <int BYTES> struct Bits;
template <> struct Bits<1> { typedef uint8_t type; };
template <> struct Bits<2> { typedef uint16_t type; };
template <> struct Bits<4> { typedef uint32_t type; };
template <> struct Bits<8> { typedef uint64_t type; };

// A pointer that all lanes share, kept in scalar registers whatever is added to it, and a load at a lane's offset from it.
__device__ __forceinline__ const char* scalar_base(const void* p, size_t offset) {
  uint64_t b = reinterpret_cast<uint64_t>(p) + offset;
  asm("" : "+s"(b));
  return reinterpret_cast<const char*>(b);
}
template <class V, int ALIGNED = 2>
__device__ __forceinline__ V load_at(const char* base, uint32_t offset) {
  typedef const __attribute__((address_space(1))) char* global_bytes;
  typedef V unaligned_t __attribute__((aligned(ALIGNED)));
  return *reinterpret_cast<const __attribute__((address_space(1))) unaligned_t*>((global_bytes)base + offset);
}

__device__ __forceinline__ float scale_to_f32(uint32_t bits, bool half) {
  const float b = bf16_to_f32((bf16_bits)bits), h = (float)__builtin_bit_cast(f16_t, (uint16_t)bits);
  return half ? h : b;
}

template <int N, class F, int... I>
__device__ __forceinline__ void static_for(F&& f, std::integer_sequence<int, I...>) { (f(Int<I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) { static_for<N>(f, std::make_integer_sequence<int, N>{}); }

// What a wave does beside the matrix-core instructions of a substep, an op to a gap behind another by the issue slots that it takes:
// an instruction of another kind takes one of the seven that a matrix-core instruction leaves, a write to LDS five.
enum Op { kReadA, kReadB, kConvert, kCommit, kFetch, kRun, kBarrier };
constexpr int kMaxOps = 32;
struct Schedule {
  int count = 0;
  Op op[kMaxOps] = {};
  int arg[kMaxOps] = {}, gap[kMaxOps] = {};
};
constexpr Schedule schedule(int tm, int tn, int pieces, bool run, bool barrier) {
  Schedule s;
  int cost[kMaxOps] = {}, total = 0;
  auto add = [&](Op op, int arg, int c) { s.op[s.count] = op; s.arg[s.count] = arg; cost[s.count++] = c; total += c; };
  const int reads = tm + tn;
  // the first column of A's fragments, B's, A's others: the order in which the next substep wants them
  auto read = [&](int r) { if (r == 0) add(kReadA, 0, 1); else if (r <= tn) add(kReadB, r - 1, 1); else add(kReadA, r - tn, 1); };
  int r = 0, moved = 0;
  const int ahead = barrier ? 3 : 0;  // steps of a conversion before the barrier: time for what was written last
  for (int c = 0; c < 8; ++c) {
    if (c == ahead && barrier) add(kBarrier, 0, 1);
    for (; c >= ahead && r < reads && r * (8 - ahead) <= (c - ahead) * reads; ++r) read(r);
    add(kConvert, c, c % 4 == 3 ? 9 : 4);
    for (; c >= ahead && moved < 2 * pieces && moved * (8 - ahead) < (c - ahead + 1) * 2 * pieces; ++moved)
      add(moved % 2 == 0 ? kCommit : kFetch, moved / 2, 5);
  }
  for (; r < reads; ++r) read(r);
  if (run) add(kRun, 0, 12);
  int before = 0;
  for (int o = 0; o < s.count; ++o) {
    s.gap[o] = (2 * before + cost[o]) * tm * tn / (2 * total);
    before += cost[o];
  }
  return s;
}
}  // namespace int4_detail

template <class C>
__device__ __forceinline__ void int4_tile_kloop(const typename C::Elem* __restrict__ Ap, int lda, int a_lim, const Int4Columns& b, int klen,
                                                unsigned char* smem, int wave, int lane, f32x16_t (&acc)[C::TM][C::TN]) {
  using int4_detail::Int;
  const int wm = wave >> 1, wn = wave & 1;
  typedef RsLoader<C::BM, C::BK, C::NW, true, typename C::Elem, false> LdA;
  LdA la;
  la.init(Ap, lda, a_lim, klen, wave, lane);
  DldsFragReader<C::BM, C::BK, C::TM, true> fra;
  DldsFragReader<C::BN, C::BK, C::TN, true> frb;
  fra.init(wm * C::WM, lane);
  frb.init(wn * C::WN, lane);
  const int nk = (klen + C::BK - 1) / C::BK;

  // ---- x: piece q of the loader's slab -> a[SET][q]; a[SET][q] -> LDS ----
  constexpr int PA = LdA::PER;
  u32x4_t a[2][PA];
  auto fetch_a = [&](auto set, int q) { a[decltype(set)::value][q] = la.fetch(q); };
  auto commit_a = [&](auto set, int slot, int q) { la.commit(smem + slot, q, a[decltype(set)::value][q]); };
  auto trim_a = [&](auto set, int step, int first, int count, auto&& also) {
    constexpr int SET = decltype(set)::value;
    if (step >= nk - 1) {
      asm volatile("");  // (a branch, not selects in every slab)
      also();
#pragma unroll
      for (int q = 0; q < PA; ++q)
        if (q >= first && q < first + count) a[SET][q] = la.trim(wave, lane, q, step, a[SET][q]);
    }
  };

  // ---- weights: piece i of a run is strip wave + 4 i of the tile; a lane has its piece (h, c).  Eight lanes that write to LDS together
  // have columns two apart, whose chunks are permuted differently: neighbours would be two to a bank ----
  typedef typename int4_detail::Bits<2 * C::PER_RUN>::type Scales;
  typedef typename int4_detail::Bits<C::PER_RUN>::type Zeros;
  u32x4_t codes[2][4];
  Scales scales[2][4];
  Zeros zeros[2][4];
  const int c = 2 * (lane & 7) + (lane >> 3 & 1), h = lane >> 4, last_strip = int4_strips(b.n) - 1 - b.first / kInt4Strip;
  const uint32_t piece = (uint32_t)(16 * h + c) * 16u;
  uint32_t column[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) column[i] = (uint32_t)imin(b.first + kInt4Strip * (wave + 4 * i) + c, b.n - 1);
  auto fetch_b = [&](auto set, int run, int i) {
    constexpr int SET = decltype(set)::value;
    const int r = imin(run, b.runs - 1);  // (behind the last run x is zero)
    const size_t strip = (size_t)imin(wave + 4 * i, last_strip) * b.stride + r;
    codes[SET][i] = int4_detail::load_at<u32x4_t>(int4_detail::scalar_base(b.codes, strip * 1024), piece);
    const size_t at = (size_t)r * b.n;
    scales[SET][i] = int4_detail::load_at<Scales>(int4_detail::scalar_base(b.scales, at * sizeof(Scales)), column[i] * (uint32_t)sizeof(Scales));
    zeros[SET][i] = int4_detail::load_at<Zeros, 1>(int4_detail::scalar_base(b.zeros, at * sizeof(Zeros)), column[i] * (uint32_t)sizeof(Zeros));
  };
  // Where a word's weights go: row `column of the tile`, chunk (j & 1) 4 + h, permuted as DldsFragReader reads it.
  const int b_row = kInt4Strip * wave + c, b_sw = (b_row >> 1) & 7;  // (strips four apart: the permutation repeats)
  int b_at[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) b_at[j] = C::A_BYTES + b_row * 128 + (((4 * j + h) ^ b_sw) << 4);
  // Step st of word w (of the slab's half HALF_RUN) of piece i: a pair of weights; with the last one all eight are written.
  float s = 0.f, from1024 = 0.f, from64 = 0.f;
  uint32_t word = 0;
  float lo = 0.f, hi = 0.f;
  u32x4_t out;
  uint32_t mask0 = 0x000f000fu, mask4 = 0x00f000f0u, one0 = 0x64006400u, one4 = 0x54005400u;  // 1024, 64
  asm("" : "+s"(mask0), "+s"(mask4));
  asm("" : "+v"(one0), "+v"(one4));
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  constexpr int kSteps = 4;
  auto convert = [&](auto set, auto half_run, int slot, int i, int w, int st) {
    constexpr int SET = decltype(set)::value, J0 = 2 * decltype(half_run)::value;
    const int j = J0 + w;
    if (st == 0) {
      if (w == 0 || C::BLOCK == 32) {
        const int e = j * 32 / C::BLOCK;
        s = int4_detail::scale_to_f32((uint32_t)(scales[SET][i] >> (16 * e)) & 0xffff, b.scale_half);
        const float z = b.has_zeros ? (float)((uint32_t)(zeros[SET][i] >> (8 * e)) & 0xff) : 8.f;
        from1024 = -s * (1024.f + z);
        from64 = -s * (64.f + z);
      }
      word = codes[SET][i][j];
    }
    if (st == 2) word >>= 8;
    const f16x2_t v = __builtin_bit_cast(f16x2_t, (st & 1) ? (word & mask4) | one4 : (word & mask0) | one0);
    const float from = (st & 1) ? from64 : from1024;
    if (C::HALF) {
      const f16x2_t both = {(_Float16)__builtin_fmaf((float)v[0], s, from), (_Float16)__builtin_fmaf((float)v[1], s, from)};
      out[st] = __builtin_bit_cast(uint32_t, both);
    } else {
      if (st > 0) out[st - 1] = pack_out_x2<C::HALF>(lo, hi);
      lo = __builtin_fmaf((float)v[0], s, from);
      hi = __builtin_fmaf((float)v[1], s, from);
      if (st == kSteps - 1) out[st] = pack_out_x2<C::HALF>(lo, hi);
    }
    if (st == kSteps - 1) *reinterpret_cast<u32x4_t*>(smem + slot + b_at[w] + i * 4 * kInt4Strip * 128) = out;
  };
  // float16 rows: what piece i has of slab `step` past the contraction becomes zero in LDS, behind the writes of convert().  It stands on
  // the scale of the last block, on which the padding's codes may be infinite in float16 where the operand's are not, and infinite
  // times x's zeros is NaN.  (bfloat16 holds every weight.)  To be called where trim_a() has its branch.
  auto trim_b = [&](int step, int slot, int i) {
    const int left = klen - step * C::BK;
    if (!C::HALF || left >= C::BK) return;
    unsigned char* at = smem + slot + i * 4 * kInt4Strip * 128;
    if (left <= 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w) *reinterpret_cast<u32x4_t*>(at + b_at[w]) = u32x4_t{0, 0, 0, 0};
    } else {
#pragma unroll 1
      for (int e = 0; e < 16; ++e)
        if ((e >> 3) * 32 + 8 * h + (e & 7) >= left) *reinterpret_cast<uint16_t*>(at + (e < 8 ? b_at[0] : b_at[1]) + 2 * (e & 7)) = 0;
    }
  };

  constexpr auto part = [](int u) constexpr { return u * PA / 4; };
  constexpr int HEAD = part(1), HEAD_MOST = (PA + 3) / 4;

  // ---- slab 0 in LDS, slab 1 in registers with its first quarter written, slab 2 requested; runs 0 and 1 ----
#pragma unroll
  for (int i = 0; i < 4; ++i) fetch_b(Int<0>{}, 0, i);
#pragma unroll
  for (int q = 0; q < PA; ++q) fetch_a(Int<0>{}, q);
  la.advance(wave, lane);
#pragma unroll
  for (int i = 0; i < 4; ++i) fetch_b(Int<1>{}, 1, i);
#pragma unroll
  for (int q = 0; q < PA; ++q) fetch_a(Int<1>{}, q);
  la.advance(wave, lane);
  trim_a(Int<0>{}, 0, 0, PA, [] {});
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int st = 0; st < kSteps; ++st) convert(Int<0>{}, Int<0>{}, 0, i, w, st);
  if (nk == 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) trim_b(0, 0, i);
#pragma unroll
  for (int q = 0; q < PA; ++q) commit_a(Int<0>{}, 0, q);
#pragma unroll
  for (int q = 0; q < PA; ++q) fetch_a(Int<0>{}, q);
  la.advance(wave, lane);
  trim_a(Int<1>{}, 1, 0, HEAD, [] {});
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int st = 0; st < kSteps; ++st) convert(Int<0>{}, Int<1>{}, C::SLOT_BYTES, 0, w, st);
  fetch_b(Int<0>{}, 2, 0);
#pragma unroll
  for (int q = 0; q < HEAD; ++q) commit_a(Int<1>{}, C::SLOT_BYTES, q);
#pragma unroll
  for (int q = 0; q < HEAD; ++q) fetch_a(Int<1>{}, q);
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): slab 0 is written
  __builtin_amdgcn_s_barrier();

  bf16x8_t fa[2][C::TM], fb[2][C::TN];
#pragma unroll
  for (int i = 0; i < C::TM; ++i) fa[0][i] = fra.read(smem, i, 0);
#pragma unroll
  for (int j = 0; j < C::TN; ++j) fb[0][j] = frb.read(smem + C::A_BYTES, j, 0);

  // Slab t, PHASE = t & 3.  Substeps 0 .. 2 write quarters 1 .. 3 of slab t + 1, substep 3, behind the slab's barrier, quarter 0 of
  // slab t + 2 into the slot that slab t has left.  A piece of x is followed by its load two slabs on, a piece of a run, once its
  // second half is written, by its load two runs on.
  auto slab = [&](int t, auto phase) {
    constexpr int PHASE = decltype(phase)::value, CUR = PHASE & 1, NEXT = 1 - CUR;
    int4_detail::static_for<4>([&](auto substep) {
      constexpr int U = decltype(substep)::value, MF = C::TM * C::TN;
      constexpr bool LAST = U == 3;
      constexpr int QUARTER = LAST ? 0 : U + 1, FIRST = part(QUARTER), COUNT = part(QUARTER + 1) - FIRST;
      // what is written: quarter QUARTER of slab t + 2 (LAST) or t + 1, half HALF_RUN of run SET
      constexpr int SIDE = LAST ? CUR : NEXT, SET = ((PHASE + (LAST ? 2 : 1)) >> 1) & 1, OFF = SIDE * C::SLOT_BYTES;
      constexpr int4_detail::Schedule plan = int4_detail::schedule(C::TM, C::TN, COUNT, SIDE == 1, LAST);
      const unsigned char* ra = smem + (LAST ? NEXT : CUR) * C::SLOT_BYTES;  // fragments of the next substep
      constexpr int US = LAST ? 0 : U + 1;
      if (LAST) la.advance(wave, lane);
      trim_a(Int<SIDE>{}, t + (LAST ? 2 : 1), FIRST, COUNT, [&] { trim_b(t + 1, NEXT * C::SLOT_BYTES, U); });  // (the quarter written last)
      int4_detail::static_for<MF>([&](auto gap) {
        constexpr int M = decltype(gap)::value, I = M / C::TN, J = M % C::TN;
        int4_detail::static_for<int4_detail::kMaxOps>([&](auto index) {
          constexpr int O = decltype(index)::value;
          if constexpr (O < plan.count && plan.gap[O] == M) {
            constexpr int ARG = plan.arg[O];
            constexpr int4_detail::Op OP = plan.op[O];
            if constexpr (OP == int4_detail::kReadA) fa[(U + 1) & 1][ARG] = fra.read(ra, ARG, US);
            if constexpr (OP == int4_detail::kReadB) fb[(U + 1) & 1][ARG] = frb.read(ra + C::A_BYTES, ARG, US);
            if constexpr (OP == int4_detail::kConvert) convert(Int<SET>{}, Int<SIDE>{}, OFF, QUARTER, ARG / kSteps, ARG % kSteps);
            if constexpr (OP == int4_detail::kCommit) commit_a(Int<SIDE>{}, OFF, FIRST + ARG);
            if constexpr (OP == int4_detail::kFetch) fetch_a(Int<SIDE>{}, FIRST + ARG);
            if constexpr (OP == int4_detail::kRun) fetch_b(Int<SET>{}, ((t + (LAST ? 2 : 1)) >> 1) + 2, QUARTER);
            if constexpr (OP == int4_detail::kBarrier) {  // own reads of slab t returned, own part of slab t + 1 written; behind it slab t + 1 is complete
              __builtin_amdgcn_sched_barrier(0);
              __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
              __builtin_amdgcn_s_barrier();
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        });
        acc[I][J] = mfma_32x32x16<C::HALF>(fb[U & 1][J], fa[U & 1][I], acc[I][J]);
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };
  // (an nk that is no multiple of four multiplies up to three slabs of zeros: a way out of the middle of the loop had the compiler
  // hold two sets of accumulators, 600 registers spilled)
  for (int t = 0; t < nk; t += 4) {
    slab(t, Int<0>{});
    slab(t + 1, Int<1>{});
    slab(t + 2, Int<2>{});
    slab(t + 3, Int<3>{});
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_s_barrier();  // the slots are no longer read by any wave
}

// rows x min(256, n - first column) of y at Op (row pitch n); klen >= 8.
template <class C>
__device__ __forceinline__ void int4_tile(const void* Ap, int lda, int rows, const Int4Columns& b, int klen, void* Op, unsigned char* smem,
                                          const SplitK& sk) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x16_t acc[C::TM][C::TN];
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  int4_tile_kloop<C>(static_cast<const typename C::Elem*>(Ap), lda, rows, b, klen, smem, wave, lane, acc);
  if (!splitk_combine<C>(acc, sk, threadIdx.x, smem)) return;
  rs_store16<C>(acc, wave >> 1, wave & 1, wave, lane, rows, imin(C::BN, b.n - b.first), static_cast<typename C::Elem*>(Op), b.n, smem);
}

}  // namespace rd
