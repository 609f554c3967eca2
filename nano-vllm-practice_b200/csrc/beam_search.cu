// Beam search's selection: the num_select best continuations of every request over its
// beams and the vocabulary, one pass over the logits.
//
// The reference decodes one continuation per request (femtovllm/engine/sampler.py:15-114) and has
// no beams.  For beam w of a request with score c_w and logits x_w:
//
//   score(w, i) = c_w + x_w[i] - lse_w,   lse_w = log sum_j exp(x_w[j])
//
// and the selection takes the largest scores, on ties the lowest w * vocab + i.  Within a
// beam the order of the scores is the order of its logits, which needs no arithmetic: only
// the beams' best num_select logits can be chosen, and only the comparison of candidates of
// different beams depends on lse.  Two launches:
//
//   partials  CTA (part of a row): its warps stream the part once, fold sum 2^(x log2e - m)
//             with a lazily moved integer m, and keep one number per segment of 32 logits, the
//             largest.  Of 64 or 128 groups of segments the num_select-th largest maximum is a
//             bound that at least num_select logits reach, and hardly any more do: only the
//             segments that reach it are read again, from L2, and their few logits at or above
//             it are ranked against each other.
//   finish    CTA per request (programmatic dependent): lse of each beam, then a merge of the
//             beams' and parts' sorted lists by their scores in fp64, again by a bound.
//
// A sum of exponentials is off by a share that does not depend on the logits: a tile's 16 or 32 of a lane are added as a
// tree (five roundings, 5 * 2^-24), tiles in two floats by Knuth's TwoSum and lanes, warps and parts in fp64, all exact
// beside that since sums relative to different m differ by powers of two.  Add ex2.approx (2^-22), the rounding of
// x log2e - m (2^-24 of itself, at most 10.8 on a warp's average: 4.5e-7) and log2e's own (1.3e-8 times what the logits
// lie below the largest on average, at most 22 nats), and an lse is off by less than 1.3e-6, a difference of two by less
// than 2.6e-6.  Scores of different beams closer than kNearTie are therefore in doubt, where one of them is chosen, and
// the lse of those beams is computed again in fp64 (2 of 4800 requests of 8 beams x 151936, 16 chosen), so the order
// does not depend on rounding.  (Added up one by one, 128 equal terms alone can be off by 1.9e-6.)
//
// Measured: 32 requests x 8 beams x 151936 bf16, 16 chosen (62 MB) 25 us out of L2, 28.7 us out of HBM.  Of the 25: the
// loads alone 12.5, the exponentials 3.6 (16 a clock and SM), bound and ranking 4, finish 5 (two overlap with the next
// part's loads).  1 x 4 x 151936: 9 us, two launches' latency.  A beam in doubt takes 40 us more in its request's CTA:
// 32 x 8 with one such pair 115 us, 1 x 4 90 us.  One whose row is a copy of a row already summed is found by comparing
// them, 17 us: requests of 8 beams that are all copies 187 us (420 with a sum each).
// The first version kept sorted lists in every thread and merged them serially: 110 and 19 us.
//
// A finished beam has one continuation, eos at its own score, and its logits are not read.
// A score that is not a number (a NaN or +inf logit, a row of -inf) counts as -inf.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "common.cuh"
#include "kernels.h"

namespace fvb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kNearTie = 3e-6;

struct BeamArgs {
  const void* logits;
  int64_t row_stride, vocab;
  const float* scores;
  const uint8_t* finished;
  int64_t eos;
  int num_beams, num_select, parts;
  int64_t part_vecs;  // 16-byte vectors per part
  uint64_t* keys;     // [row][part][num_select], best first; 0 = none
  double2* sums;      // [row][part] (m, s): sum of 2^(x log2e) = s 2^m
  int64_t *tokens, *parents;
  float* out_scores;
};

// Logits as unsigned integers of the same order, with the index below: larger keys are
// larger logits and, among equal ones, lower indices.  Every logit's key is above 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 and +0 are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// The same for fp64 scores.
__device__ __forceinline__ uint64_t ordered64(double x) {
  const int64_t b = __double_as_longlong(x == 0.0 ? 0.0 : x);
  return b < 0 ? ~uint64_t(b) : uint64_t(b) | (uint64_t(1) << 63);
}
__device__ __forceinline__ double unordered64(uint64_t u) {
  return __longlong_as_double(int64_t(u >> 63 ? u & ~(uint64_t(1) << 63) : ~u));
}
__device__ __forceinline__ float key_logit(uint64_t k) { return unordered(uint32_t(k >> 32)); }
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~uint32_t(k); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 2^x on the SFU without the volatile qualifier, so the compiler may schedule it freely.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x of an integer x <= 0, exact; 0 below the normal numbers, and of a NaN.
__device__ __forceinline__ float pow2(float x) { return __int_as_float((int(fmaxf(x, -127.f)) + 127) << 23); }
__device__ __forceinline__ double pow2(double x) { return __hiloint2double((int(fmax(x, -1023.0)) + 1023) << 20, 0); }

// hi + lo += x, where only lo's own sum is rounded.
__device__ __forceinline__ void add_exactly(float& hi, float& lo, float x) {
  const float sum = __fadd_rn(hi, x), back = __fsub_rn(sum, hi);
  lo = __fadd_rn(lo, __fadd_rn(__fsub_rn(hi, __fsub_rn(sum, back)), __fsub_rn(x, back)));
  hi = sum;
}

// Rows may start at any element: vectors are counted from the 16-byte boundary at or before
// the row, so vector j holds logits j * VE - shift .. and only the first and last may reach outside.
template <typename T>
struct Row {
  static constexpr int VE = 16 / sizeof(T);
  const T* p;
  int64_t vocab;
  int shift;
  __device__ __forceinline__ Row(const BeamArgs& a, int64_t row) {
    p = static_cast<const T*>(a.logits) + row * a.row_stride;
    vocab = a.vocab;
    shift = int((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  }
  __device__ __forceinline__ int64_t vecs() const { return (vocab + shift + VE - 1) / VE; }
  __device__ __forceinline__ int64_t index(int64_t vec) const { return vec * VE - shift; }
  // Vector vec with -inf past the row's ends.
  __device__ __forceinline__ uint4 load_ragged(int64_t vec) const {
    const int64_t i = index(vec);
    __align__(16) T x[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = i + e >= 0 && i + e < vocab ? p[i + e] : Elem<T>::from_f(-INFINITY);
    return *reinterpret_cast<const uint4*>(x);
  }
};

// Elementwise maximum of 32-bit words (one float, or two 16-bit logits); of a number and a NaN the number.
template <typename T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}
template <typename T>
__device__ __forceinline__ float word_max(uint32_t a) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(a);
  float f[8];
  unpack16<T>(make_uint4(a, 0, 0, 0), f);
  return fmaxf(f[0], f[1]);
}

constexpr int kCtasPerSm = 4;          // CTAs the parts are sized for
constexpr int kLists = 2;              // sorted lists a thread of the finish kernel merges
constexpr int kRanked = 512;           // candidates it ranks at once
constexpr int kFinishThreads = 512;
constexpr int kFinishWarps = kFinishThreads / 32;
constexpr int kSegment = 32;           // logits
constexpr int kMaxSegments = 4096;     // of a part: their maxima fill 16 KB of shared memory
constexpr int kVecs = 4;               // vectors per lane and tile
constexpr int kFewSegments = 128;      // of a part whose segments are ranked one by one
constexpr int kListSegs = 1024, kListLogits = 1024;  // segments and logits at or above the bound that are ranked

// The k-th largest (from 0) of `groups` <= 128 values into *bound, where there are so many; whole CTAs of WARPS warps.
template <int WARPS>
__device__ __forceinline__ void kth_largest(const uint32_t* values, int groups, int k, uint32_t* bound) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = lane + 32 * j < groups ? values[lane + 32 * j] : 0;
#pragma unroll 2
  for (int g = warp; g < groups; g += WARPS) {
    const uint32_t own = values[g];
    int before = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < 2 || groups > 64)
        before += __popc(__ballot_sync(0xffffffffu, v[j] > own || (v[j] == own && lane + 32 * j < g)));
    }
    if (before == k && lane == 0) *bound = own;
  }
}

// The n best (value, lower index first) of what the warp's lanes hold, one at a time: lane
// state (best, at) is each lane's best and its index; take(n-th best's index) is called in
// the lane that held it and must refresh its state.  Values of 0 are void.
template <typename Take, typename Emit>
__device__ __forceinline__ void extract(int n, uint32_t& best, uint32_t& at, Take take, Emit emit) {
  for (int k = 0; k < n; ++k) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    if (top == 0) {
      emit(k, 0u, 0u);
      continue;
    }
    const uint32_t index = __reduce_min_sync(0xffffffffu, best == top ? at : 0xffffffffu);
    emit(k, top, index);
    if (best == top && at == index) take(index);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) beam_partials_kernel(const BeamArgs a) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int kSegVecs = kSegment / VE;  // 4 (16-bit) or 8 (fp32) lanes share a segment
  constexpr int kTile = 32 * kVecs;        // vectors of a warp's tile
  extern __shared__ uint32_t sh[];         // segment maxima as ordered(); then the chosen segments' logits
  __shared__ double2 sh_sums[kWarps];
  __shared__ uint32_t sh_runs[kThreads / 2];  // largest segment maximum of each group of two or four lanes
  __shared__ uint64_t cand[kListLogits];
  __shared__ uint16_t list[kListSegs];
  __shared__ uint32_t bound;
  __shared__ int n_list, n_cand;
  launch_dependents();
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.finished != nullptr && __ldg(a.finished + row) != 0) return;
  const Row<T> r(a, row);
  const int64_t part_begin = part * a.part_vecs;
  const int n_vecs = int(max(min(r.vecs() - part_begin, a.part_vecs), int64_t(0)));
  const int n_segs = (n_vecs + kSegVecs - 1) / kSegVecs;

  if (threadIdx.x == 0) n_list = n_cand = bound = 0;
  float m = -INFINITY;
  uint32_t run = 0;  // of segments of this thread alone; 0: none
  float hi = 0.f, lo = 0.f;  // this lane's sum, relative to 2^m
  // Vectors [w0, w1) of the part lie wholly inside the row.
  const int w0 = part_begin == 0 && r.shift != 0 ? 1 : 0;
  const int w1 = int(min((a.vocab + r.shift) / VE - part_begin, int64_t(n_vecs)));
  const T* lane_p = r.p + r.index(part_begin + lane);
  uint4 ahead[kVecs];  // the warp's next tile, in flight while this one is folded
  auto fetch = [&](int v0) {
    if (v0 >= w0 && v0 + kTile <= w1) {
      const T* p = lane_p + int64_t(v0) * VE;
#pragma unroll
      for (int u = 0; u < kVecs; ++u) ahead[u] = ldg_nc_v4(p + u * 32 * VE);
    } else {
#pragma unroll 1
      for (int u = 0; u < kVecs; ++u) {
        // (past the part: void, no logit of the row)
        const int v = v0 + u * 32 + lane;
        const uint4 x = r.load_ragged(v < n_vecs ? part_begin + v : r.vecs() + 1);
        ahead[0] = u == 0 ? x : ahead[0];
        ahead[1] = u == 1 ? x : ahead[1];
        ahead[2] = u == 2 ? x : ahead[2];
        ahead[3] = u == 3 ? x : ahead[3];
      }
    }
  };
  if (warp * kTile < n_vecs) fetch(warp * kTile);
  for (int v0 = warp * kTile; v0 < n_vecs; v0 += kWarps * kTile) {
    uint4 x[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) x[u] = ahead[u];
    if (v0 + kWarps * kTile < n_vecs) fetch(v0 + kWarps * kTile);
    // ---- segment maxima: in the lane, then over the segment's lanes, which end up with one u each ----
    uint32_t w[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) w[u] = max_word<T>(max_word<T>(x[u].x, x[u].y), max_word<T>(x[u].z, x[u].w));
    {
      const bool odd = lane & 1;
      const uint32_t a0 = __shfl_xor_sync(0xffffffffu, odd ? w[0] : w[1], 1);
      const uint32_t a1 = __shfl_xor_sync(0xffffffffu, odd ? w[2] : w[3], 1);
      w[0] = max_word<T>(odd ? w[1] : w[0], a0);  // u = lane & 1
      w[1] = max_word<T>(odd ? w[3] : w[2], a1);  // u = 2 + (lane & 1)
      const bool two = lane & 2;
      const uint32_t b0 = __shfl_xor_sync(0xffffffffu, two ? w[0] : w[1], 2);
      w[0] = max_word<T>(two ? w[1] : w[0], b0);  // u = lane & 3
      if constexpr (kSegVecs == 8) w[0] = max_word<T>(w[0], __shfl_xor_sync(0xffffffffu, w[0], 4));
    }
    const float g = word_max<T>(w[0]);
    const int seg = (v0 + (lane & 3) * 32) / kSegVecs + lane / kSegVecs;
    if (seg < n_segs && (kSegVecs == 4 || (lane & 4) == 0)) {
      const uint32_t og = ordered(g);
      sh[seg] = og;
      run = max(run, og);
    }
    // ---- sum of exponentials; the warp's m moves only when a tile passes it by more than 2^8 ----
    if (__any_sync(0xffffffffu, g * kLog2e > m + 8.f)) {
      const float top = ceilf(unordered(__reduce_max_sync(0xffffffffu, ordered(g))) * kLog2e);
      const float f = pow2(m - top);  // 0 while m is -inf
      hi *= f;
      lo *= f;
      m = top;
    }
    // m is -inf while every logit was: nothing to add, except that a NaN has to show in the sum
    const float ms = m == -INFINITY ? 0.f : -m;
    float2 v[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      float f[VE];
      unpack16<T>(x[u], f);
      float2 e[VE / 2];
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const float2 t =
            __ffma2_rn(make_float2(f[2 * i], f[2 * i + 1]), make_float2(kLog2e, kLog2e), make_float2(ms, ms));
        e[i] = make_float2(ex2(t.x), ex2(t.y));
      }
      v[u] = __fadd2_rn(e[0], e[1]);
      if constexpr (VE == 8) v[u] = __fadd2_rn(v[u], __fadd2_rn(e[2], e[3]));
    }
    const float2 tile = __fadd2_rn(__fadd2_rn(v[0], v[1]), __fadd2_rn(v[2], v[3]));
    add_exactly(hi, lo, __fadd_rn(tile.x, tile.y));
  }
  // ---- the part's sum ----
  double sum = double(hi) + double(lo);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);  // m is the warp's
  if (lane == 0) sh_sums[warp] = make_double2(double(m), sum);
  const int64_t out = row * a.parts + part;
  const int K = a.num_select;
  // Groups of four lanes give 64 maxima (fp32: 32, every other lane's segments are its neighbour's), pairs twice as
  // many; the fewer there are above K, the more logits reach the bound (about G ln(G / (G - K)) of them).
  const int shift = K <= (kSegVecs == 4 ? 32 : 16) ? 2 : 1, groups = kThreads >> shift;
  run = max(run, __shfl_xor_sync(0xffffffffu, run, 1));
  if (shift == 2) run = max(run, __shfl_xor_sync(0xffffffffu, run, 2));
  if ((lane & ((1 << shift) - 1)) == 0) sh_runs[threadIdx.x >> shift] = run;
  __syncthreads();
  if (warp == kWarps - 1) {
    const double2 v = lane < kWarps ? sh_sums[lane] : make_double2(-INFINITY, 0.0);
    const double mm = double(warp_max(float(v.x)));
    double ss = v.x == -INFINITY ? v.y : v.y * pow2(v.x - mm);
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) a.sums[out] = make_double2(mm, ss);
  }
  // ---- bound: the K-th largest group (0, every logit, where fewer than K groups have one).  A part of few segments
  // leaves most groups without one, and its segments are groups themselves (the last 107 vectors of a row of 50001
  // 16-bit logits, K 10: all 856 logits reached the bound, and ranking them took 22 us). ----
  const bool few = n_segs <= kFewSegments;
  kth_largest<kWarps>(few ? sh : sh_runs, few ? n_segs : groups, K - 1, &bound);
  __syncthreads();
  const uint32_t least = bound;
  // ---- segments that reach it, and their logits that do ----
  for (int i = threadIdx.x; i < n_segs; i += kThreads) {
    if (sh[i] < least) continue;
    const int n = atomicAdd(&n_list, 1);
    if (n < kListSegs) list[n] = uint16_t(i);
  }
  __syncthreads();
  const int segs = n_list;
  if (segs <= kListSegs) {
    constexpr int kReads = 4;  // segments a warp reads at once
    for (int n0 = warp; n0 < segs; n0 += kWarps * kReads) {
      uint32_t v[kReads], id[kReads];
#pragma unroll
      for (int u = 0; u < kReads; ++u) {
        const int n = n0 + u * kWarps;
        v[u] = id[u] = 0;
        if (n < segs) {
          const int64_t i = r.index(part_begin + int64_t(list[n]) * kSegVecs) + lane;
          id[u] = uint32_t(i);
          if (i >= 0 && i < a.vocab) v[u] = ordered(Elem<T>::to_f(r.p[i]));
        }
      }
#pragma unroll
      for (int u = 0; u < kReads; ++u) {
        if (v[u] == 0 || v[u] < least) continue;
        const int at = atomicAdd(&n_cand, 1);
        if (at < kListLogits) cand[at] = uint64_t(v[u]) << 32 | ~id[u];
      }
    }
  }
  __syncthreads();
  const int n = n_cand;
  if (segs <= kListSegs && n <= kListLogits) {
    // ---- rank them: keys are different, and fewer than K logits in the part leave 0 behind them ----
    for (int i = threadIdx.x; i < max(n, K); i += kThreads) {
      const uint64_t mine = i < n ? cand[i] : 0;
      int before = i < n ? 0 : i;
      if (i < n) {
#pragma unroll 8
        for (int j = 0; j < n; ++j) before += cand[j] > mine;
      }
      if (before < K) a.keys[out * K + before] = mine;
    }
    return;
  }
  // ---- too many logits tie with the bound (masked vocabularies), or a few threads hold nearly all of the
  // largest ones: one warp takes the K largest segments (on ties the lower ones) one by one, then the K best
  // of their logits.  No other segment can hold one of those: each of the chosen has a logit that is larger,
  // or equal and of a lower index.  (About 40 us where the ranking takes 2.) ----
  if (warp != 0) return;
  const int picks = min(K, n_segs);
  uint32_t best = 0, at = 0;
  auto rescan = [&]() {  // the lane's segments lane, lane + 32, ..: the largest, among equal ones the lowest
    best = 0;
    for (int i = lane; i < n_segs; i += 32) {
      const uint32_t v = sh[i];
      if (v > best) {
        best = v;
        at = i;
      }
    }
  };
  rescan();
  extract(
      picks, best, at,
      [&](uint32_t i) {
        sh[i] = 0;
        rescan();
      },
      [&](int k, uint32_t, uint32_t i) {
        if (lane == 0) list[k] = uint16_t(i);
      });
  __syncwarp();
  auto index_of = [&](int k) { return r.index(part_begin + int64_t(list[k]) * kSegVecs) + lane; };
  for (int k = 0; k < picks; ++k) {
    const int64_t i = index_of(k);
    sh[k * 32 + lane] = i >= 0 && i < a.vocab ? ordered(Elem<T>::to_f(r.p[i])) : 0u;
  }
  int mine = 0;
  auto rescan_logits = [&]() {  // entry [k][lane] is the lane's own
    best = 0;
    for (int k = 0; k < picks; ++k) {
      const uint32_t v = sh[k * 32 + lane];
      if (v > best || (v == best && v != 0 && uint32_t(index_of(k)) < at)) {
        best = v;
        at = uint32_t(index_of(k));
        mine = k;
      }
    }
  };
  rescan_logits();
  extract(
      K, best, at,
      [&](uint32_t) {
        sh[mine * 32 + lane] = 0;
        rescan_logits();
      },
      [&](int k, uint32_t v, uint32_t i) {
        if (lane == 0) a.keys[out * K + k] = v == 0 ? 0 : uint64_t(v) << 32 | uint32_t(~i);
      });
}

// State of one beam in the finish kernel.
enum { kLive = 0, kDone = 1, kDead = 2 };  // has logits; one continuation; every score is -inf
struct Beam {
  double base;   // score of its best continuation: score + best - lse, exact whatever the logits' size
  double guess;  // lse - best, from the parts' sums
  double above;  // the same from fp64, of a beam that is summed
  float best;   // its largest logit
  int kind;
  bool exact;   // base is from fp64 or the caller's score itself
  bool redo;    // base has to be computed again in fp64
  bool summed;  // it has been
};
__device__ __forceinline__ bool finite(double x) { return x >= -DBL_MAX && x <= DBL_MAX; }

// The next candidate of a sorted list: `score` as ordered64() (0: none left), its token.
struct Head {
  uint64_t score;
  uint32_t token;
};

template <typename T>
__global__ void __launch_bounds__(kFinishThreads, 1) beam_finish_kernel(const BeamArgs a) {
  __shared__ Beam beams[64];
  __shared__ double red[kFinishWarps];
  __shared__ uint32_t best_of[kFinishThreads / 4];
  __shared__ uint64_t cand_score[kRanked], cand_id[kRanked];
  __shared__ uint32_t bound;
  __shared__ uint16_t sorted[kRanked];
  __shared__ double last_score;
  __shared__ int last_beam;
  __shared__ uint64_t top_score[kFinishWarps];
  __shared__ uint32_t top_beam[kFinishWarps], top_token[kFinishWarps];
  __shared__ int again, n_cand;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int W = a.num_beams, K = a.num_select;
  const int64_t row0 = int64_t(blockIdx.x) * W;
  const int per_row = a.parts * K;
  if (threadIdx.x == 0) again = n_cand = 0;
  // The call's inputs (the kernel in front only reads them): each beam's score and kind.
  for (int w = threadIdx.x; w < W; w += kFinishThreads) {
    const double score = a.scores[row0 + w];
    const bool done = a.finished != nullptr && a.finished[row0 + w] != 0;
    const int kind = !finite(score) ? kDead : done ? kDone : kLive;
    beams[w] = Beam{score, 0.0, 0.0, 0.f, kind, kind != kLive, false, false};
  }
  __syncthreads();
  const unsigned long long* lists = reinterpret_cast<const unsigned long long*>(a.keys) + row0 * per_row;
  grid_dependency_wait();
  const int n_keys = W * per_row;
  // Key of the thread's turn: 512 of them at a time, eight neighbours' (a group's, below) from eight different
  // places of eight different lists, since the best ones stand together at the heads of the lists.
  const int my_key = (threadIdx.x & 7) * 64 + ((threadIdx.x >> 3) + 5 * (threadIdx.x & 7)) % 64;
  const uint64_t first_key = my_key < n_keys ? __ldcg(lists + my_key) : 0;  // in flight with the sums
  __syncthreads();

  // ---- each beam's lse ----
  for (int w = warp; w < W; w += kFinishWarps) {
    if (beams[w].kind != kLive) continue;
    const double2* sums = a.sums + (row0 + w) * a.parts;
    const unsigned long long* heads = lists + int64_t(w) * per_row;
    uint64_t first = 0;  // of the parts' best keys, the best
    float m = -INFINITY;
    double2 v = make_double2(-INFINITY, 0.0);
    for (int p = lane; p < a.parts; p += 32) {
      v = __ldcg(sums + p);
      m = fmaxf(m, float(v.x));
      first = max(first, uint64_t(__ldcg(heads + int64_t(p) * K)));
    }
    m = warp_max(m);
    const float best = unordered(__reduce_max_sync(0xffffffffu, uint32_t(first >> 32)));
    double s = 0.0;
    for (int p = lane; p < a.parts; p += 32) {
      if (a.parts > 32) v = __ldcg(sums + p);
      s += v.x == -INFINITY ? v.y : v.y * pow2(v.x - double(m));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      // s 2^m = sum 2^(x c), c = kLog2e in fp32; taken relative to the largest logit, so that c's own
      // rounding acts on differences of logits only.
      const double above = 0.69314718055994530942 * (log2(s) + (double(m) - double(best) * double(kLog2e)));
      beams[w].base -= above;
      beams[w].guess = above;
      beams[w].best = best;
      // +inf or only -inf: no distribution.  Otherwise a NaN, or logits so large that x log2e left the
      // range of fp32: fp64 tells.
      if (best == INFINITY || best == -INFINITY) {
        beams[w].kind = kDead;
        beams[w].exact = true;
      } else if (!finite(beams[w].base)) {
        beams[w].redo = true;
        again = 1;
      }
    }
  }
  __syncthreads();

  // base of the beams that ask for it in fp64, and a new start
  constexpr int kAhead = 8;  // loads in flight: 40 us a beam of 151936 logits, by fp64's rate (one at a time: 84)
  auto exact_bases = [&]() {
    for (int w = 0; w < W; ++w) {
      if (!beams[w].redo) continue;
      const T* p = static_cast<const T*>(a.logits) + (row0 + w) * a.row_stride;
      // a beam that has been summed and may hold the same row: comparing takes less than half of the sum's time
      int twin = 0;
      auto alike = [&](const Beam& b) { return b.summed && b.guess == beams[w].guess && b.best == beams[w].best; };
      while (twin < W && !alike(beams[twin])) ++twin;
      bool same = twin < W;
      if (same) {
        using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
        const Bits* x = reinterpret_cast<const Bits*>(p);
        const Bits* y =
            reinterpret_cast<const Bits*>(static_cast<const T*>(a.logits) + (row0 + twin) * a.row_stride);
        Bits differ = 0;
#pragma unroll 32
        for (int64_t i = threadIdx.x; i < a.vocab; i += kFinishThreads) differ |= x[i] ^ y[i];
        same = __syncthreads_and(differ == 0);
      }
      double above = 0.0;
      if (same) {
        above = beams[twin].above;
      } else {
        const double top = double(beams[w].best);
        double s = 0.0;
#pragma unroll 1
        for (int64_t i0 = threadIdx.x; i0 < a.vocab; i0 += kAhead * kFinishThreads) {
          float x[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int64_t i = i0 + u * kFinishThreads;
            x[u] = i < a.vocab ? Elem<T>::to_f(p[i]) : -INFINITY;
          }
#pragma unroll
          for (int u = 0; u < kAhead; u += 4) {
            const double e0 = exp(double(x[u]) - top), e1 = exp(double(x[u + 1]) - top);
            const double e2 = exp(double(x[u + 2]) - top), e3 = exp(double(x[u + 3]) - top);
            s += (e0 + e1) + (e2 + e3);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
          double t = 0.0;
          for (int k = 0; k < kFinishWarps; ++k) t += red[k];
          above = log(t);
        }
      }
      if (threadIdx.x == 0) {
        beams[w].above = above;
        beams[w].base = double(a.scores[row0 + w]) - above;
        if (!finite(beams[w].base)) beams[w].kind = kDead;
        beams[w].exact = beams[w].summed = true;
        beams[w].redo = false;
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) again = n_cand = 0;
    __syncthreads();
  };
  if (again) exact_bases();

  // Scores of two beams that lie too close for their fp32 sums: both beams' in fp64.  (Equal ones too: rows that differ
  // in their smallest logits only have one and the same sum in fp32.)  Called for every selected candidate and the next
  // one, and for the last selected one and every candidate that is not: where any two, one of them selected, are in
  // doubt, neighbours between them are, or the last one and the second of them.
  auto compare = [&](double s, int w, double s2, int w2) {
    if (w == w2 || (beams[w].exact && beams[w2].exact) || !(fabs(s - s2) < kNearTie)) return;
    beams[w].redo = !beams[w].exact;
    beams[w2].redo = !beams[w2].exact;
    again = 1;
  };
  // Entry i of beam w's list of part p, whose key is `key`.  A live beam has a list per part; a beam without
  // logits has one, its first: eos and then every other token (done), or every token (dead), at -inf.
  auto candidate = [&](int w, int p, int i, uint64_t key) {
    Head h{0, 0};
    const Beam& b = beams[w];
    if (b.kind == kLive) {
      if (key == 0) return h;
      const float x = key_logit(key);
      h.token = key_index(key);
      h.score = ordered64(x == -INFINITY ? double(-INFINITY) : b.base + (double(x) - double(b.best)));
    } else if (p == 0 && i < a.vocab) {
      h.score = ordered64(b.kind == kDone && i == 0 ? b.base : double(-INFINITY));
      h.token = b.kind == kDead ? i : i == 0 ? uint32_t(a.eos) : i - 1 + (i - 1 >= a.eos ? 1 : 0);
    }
    return h;
  };
  auto nth = [&](int i, uint64_t key) {
    const int w = i / per_row, p = (i - w * per_row) / K;
    return candidate(w, p, i - w * per_row - p * K, key);
  };
  // ---- most requests: the candidates that reach a bound which at least K + 1 do, and those that may be as good as
  // they are, ranked against each other.  The bound is the (K + 1)-th largest of 64 or 128 groups' best scores, rounded
  // to fp32.  False where that cannot be done. ----
  auto select_ranked = [&]() {
    const int shift = K < 32 ? 3 : 2, groups = kFinishThreads >> shift;
    auto rounded = [](uint64_t score) { return score == 0 ? 0u : ordered(float(unordered64(score))); };
    const Head mine = my_key < n_keys ? nth(my_key, first_key) : Head{0, 0};
    uint32_t run = rounded(mine.score);
#pragma unroll 1
    for (int i = my_key + kFinishThreads; i < n_keys; i += kFinishThreads)
      run = max(run, rounded(nth(i, __ldcg(lists + i)).score));
    for (int o = 1; o < 1 << shift; o <<= 1) run = max(run, __shfl_xor_sync(0xffffffffu, run, o));
    if ((lane & ((1 << shift) - 1)) == 0) best_of[threadIdx.x >> shift] = run;
    __syncthreads();
    kth_largest<kFinishWarps>(best_of, groups, K, &bound);
    __syncthreads();
    if (bound <= ordered(-INFINITY)) return false;
    // Every score that rounds to the bound lies above the number before it; the K-th best is one of these or better.
    const uint64_t least = ordered64(double(unordered(bound - 1)) - kNearTie);
    auto keep = [&](int i, const Head& h) {
      if (h.score < least) return;
      const int at = atomicAdd(&n_cand, 1);
      if (at >= kRanked) return;
      cand_score[at] = h.score;
      cand_id[at] = uint64_t(i / per_row) << 32 | h.token;
    };
    keep(my_key, mine);
#pragma unroll 1
    for (int i = my_key + kFinishThreads; i < n_keys; i += kFinishThreads) keep(i, nth(i, __ldcg(lists + i)));
    __syncthreads();
    const int c = n_cand;
    if (c > kRanked) return false;
    if (threadIdx.x < c) {  // kRanked <= kFinishThreads
      const uint64_t score = cand_score[threadIdx.x], id = cand_id[threadIdx.x];
      int before = 0, equal = 0;
#pragma unroll 8
      for (int j = 0; j < c; ++j) {
        before += cand_score[j] > score;
        equal += cand_score[j] == score;
      }
      if (equal > 1) {
        for (int j = 0; j < c; ++j) before += cand_score[j] == score && cand_id[j] < id;
      }
      sorted[before] = threadIdx.x;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < c; k += kFinishThreads) {
      const uint64_t id = cand_id[sorted[k]];
      const double score = unordered64(cand_score[sorted[k]]);
      if (k < K) {
        const int64_t o = int64_t(blockIdx.x) * K + k;
        a.tokens[o] = uint32_t(id);
        a.parents[o] = id >> 32;
        a.out_scores[o] = float(score);
      }
      const int other = sorted[k < K ? min(k + 1, K - 1) : K - 1];
      compare(score, int(id >> 32), unordered64(cand_score[other]), int(cand_id[other] >> 32));
    }
    return true;
  };

  // ---- else (fewer than K + 1 finite candidates, or a crowd of equal ones), one by one: a merge of the W * parts
  // sorted lists, up to kLists a thread ----
  auto entry = [&](int l, int i) {
    const int w = l / a.parts;
    return i < K ? candidate(w, l - w * a.parts, i, __ldcg(lists + int64_t(l) * K + i)) : Head{0, 0};
  };
  // (score, beam, token) order: the higher score, then the lower beam, then the lower token
  auto better = [](uint64_t s, uint32_t w, uint32_t t, uint64_t s2, uint32_t w2, uint32_t t2) {
    return s != s2 ? s > s2 : w != w2 ? w < w2 : t < t2;
  };
  // The warp's best of its lanes' (score, beam, token), in every lane.
  auto warp_best = [&](uint64_t& s, uint32_t& w, uint32_t& t) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(s >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(s >> 32) == hi ? uint32_t(s) : 0u);
    const uint64_t top = uint64_t(hi) << 32 | lo;
    const uint32_t who = __ballot_sync(0xffffffffu, s == top);
    uint32_t w1 = w, t1 = t;
    if (__popc(who) == 1) {
      const int src = __ffs(who) - 1;
      w1 = __shfl_sync(0xffffffffu, w, src);
      t1 = __shfl_sync(0xffffffffu, t, src);
    } else {  // equal scores
      w1 = __reduce_min_sync(0xffffffffu, s == top ? w : 0xffffffffu);
      t1 = __reduce_min_sync(0xffffffffu, s == top && w == w1 ? t : 0xffffffffu);
    }
    s = top;
    w = w1;
    t = t1;
  };

  const int L = W * a.parts;
  const int warps = L <= 32 * kLists ? 1 : kFinishWarps;
  auto select_merged = [&]() {
    if (warp < warps) {
      Head head[kLists], next[kLists];  // each list's first candidate that is left, and the one behind it
      int at[kLists];
#pragma unroll
      for (int j = 0; j < kLists; ++j) {
        const int l = threadIdx.x + j * 32 * warps;
        head[j] = next[j] = Head{0, 0};
        at[j] = 1;
        if (l < L) {
          head[j] = entry(l, 0);
          next[j] = entry(l, 1);
        }
      }
      for (int n = 0; n < K; ++n) {
        const uint32_t w0 = threadIdx.x / a.parts, w1 = (threadIdx.x + 32 * warps) / a.parts;
        const int mine = better(head[1].score, w1, head[1].token, head[0].score, w0, head[0].token) ? 1 : 0;
        uint64_t s = mine ? head[1].score : head[0].score;
        uint32_t t = mine ? head[1].token : head[0].token;
        uint32_t w = mine ? w1 : w0;
        const uint64_t own = s;
        const uint32_t own_w = w, own_t = t;
        warp_best(s, w, t);
        if (warps > 1) {
          if (lane == 0) {
            top_score[warp] = s;
            top_beam[warp] = w;
            top_token[warp] = t;
          }
          __syncthreads();
          s = lane < kFinishWarps ? top_score[lane] : 0;
          w = lane < kFinishWarps ? top_beam[lane] : 0;
          t = lane < kFinishWarps ? top_token[lane] : 0;
          warp_best(s, w, t);
          __syncthreads();
        }
        const double best = unordered64(s);
        if (threadIdx.x == 0) {
          if (n > 0) compare(last_score, last_beam, best, int(w));
          last_score = best;
          last_beam = int(w);
        }
        if (own == s && own_w == w && own_t == t) {  // one list alone holds a beam's token
          const int64_t o = int64_t(blockIdx.x) * K + n;
          a.tokens[o] = t;
          a.parents[o] = w;
          a.out_scores[o] = float(best);
#pragma unroll
          for (int j = 0; j < kLists; ++j) {
            if (j != mine) continue;
            head[j] = next[j];
            next[j] = entry(threadIdx.x + j * 32 * warps, ++at[j]);
          }
        }
      }
    }
    __syncthreads();
    // the last one and all others (the selected among them are its neighbours' business, and no harm)
    for (int i = threadIdx.x; i < n_keys; i += kFinishThreads) {
      if (i / per_row == last_beam) continue;
      const Head h = nth(i, __ldcg(lists + i));
      if (h.score != 0) compare(unordered64(h.score), i / per_row, last_score, last_beam);
    }
  };

  for (int pass = 0; pass <= W; ++pass) {  // (a second one hardly ever, and one more beam is exact after each)
    if (!select_ranked()) select_merged();
    __syncthreads();
    if (again == 0) return;
    exact_bases();
  }
}

template <typename T>
cudaError_t launch_t(const BeamArgs& a, int num_requests, cudaStream_t stream) {
  const int segs = std::max(int((a.part_vecs * 16 / sizeof(T) + kSegment - 1) / kSegment), 32 * a.num_select);
  beam_partials_kernel<T><<<unsigned(num_requests) * a.num_beams * a.parts, kThreads, segs * 4, stream>>>(a);
  cudaError_t ce = cudaGetLastError();
  if (ce != cudaSuccess) return ce;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_requests);
  cfg.blockDim = dim3(kFinishThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_finish_kernel<T>, a);
}

// Vectors of a part, in whole tiles of a warp and even over the parts: as many CTAs as the device holds at once, no
// part below one tile of each of its warps, at most kMaxSegments segments, and no more lists a request than the finish
// kernel's threads merge where that allows.  (One part more a row, a second wave of the same CTAs: 150 rows x 50001
// bf16 15.6 us instead of 12.9, 32 x 151936 12.5 instead of 10.6; 200 x 146216, whose 400 CTAs leave a third of the
// places empty, 19.3 instead of 20.3.)
int64_t beam_part_vecs(int num_requests, int num_beams, int64_t vocab, int esize) {
  const int64_t vecs = (vocab * esize + 15) / 16 + 1;  // a row may straddle one vector more
  const int64_t rows = int64_t(num_requests) * num_beams, warp_tile = 32 * kVecs, tile = warp_tile * kWarps;
  const int64_t wanted = std::min<int64_t>(std::max<int64_t>(1, int64_t(device_sm_count()) * kCtasPerSm / rows),
                                           kLists * kFinishThreads / num_beams);
  const int64_t most = std::min<int64_t>(((vecs + wanted - 1) / wanted + tile - 1) / tile * tile,
                                         int64_t(kMaxSegments) * kSegment * esize / 16);
  const int64_t parts = (vecs + most - 1) / most;
  return ((vecs + parts - 1) / parts + warp_tile - 1) / warp_tile * warp_tile;
}
int64_t beam_parts(int num_requests, int num_beams, int64_t vocab, int esize) {
  const int64_t vecs = (vocab * esize + 15) / 16 + 1, per = beam_part_vecs(num_requests, num_beams, vocab, esize);
  return (vecs + per - 1) / per;
}

}  // namespace

bool beam_supported(int num_requests, int num_beams, int64_t vocab, int esize) {
  const int64_t parts = beam_parts(num_requests, num_beams, vocab, esize);
  return parts * num_beams <= kLists * kFinishThreads && parts * num_beams * num_requests < (int64_t(1) << 31);
}

size_t beam_workspace_size(int num_requests, int num_beams, int64_t vocab, int num_select, int esize) {
  const size_t parts = size_t(num_requests) * num_beams * beam_parts(num_requests, num_beams, vocab, esize);
  return ((parts * num_select * 8 + 255) & ~size_t(255)) + parts * 16;
}

cudaError_t launch_beam_select(const void* logits, int64_t row_stride, int num_requests, int num_beams, int64_t vocab,
                               int dtype, const float* scores, const uint8_t* finished, int64_t eos, int num_select,
                               int64_t* tokens, int64_t* parents, float* out_scores, void* workspace,
                               cudaStream_t stream) {
  const int64_t rows = int64_t(num_requests) * num_beams;
  const int es = dtype == FVB_DTYPE_F32 ? 4 : 2;
  BeamArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = vocab;
  a.scores = scores;
  a.finished = finished;
  a.eos = eos;
  a.num_beams = num_beams;
  a.num_select = num_select;
  a.parts = int(beam_parts(num_requests, num_beams, vocab, es));
  a.part_vecs = beam_part_vecs(num_requests, num_beams, vocab, es);
  a.keys = static_cast<uint64_t*>(workspace);
  const size_t key_bytes = (size_t(rows) * a.parts * num_select * 8 + 255) & ~size_t(255);
  a.sums = reinterpret_cast<double2*>(static_cast<uint8_t*>(workspace) + key_bytes);
  a.tokens = tokens;
  a.parents = parents;
  a.out_scores = out_scores;
  if (dtype == FVB_DTYPE_BF16) return launch_t<__nv_bfloat16>(a, num_requests, stream);
  if (dtype == FVB_DTYPE_F16) return launch_t<__half>(a, num_requests, stream);
  return launch_t<float>(a, num_requests, stream);
}

}  // namespace fvb
