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
//   partials  CTA (part of a row): each of 8 warps streams a contiguous run of it, folds
//             sum 2^(x log2e - m) with a lazily moved m, and keeps the run's best logits as
//             a sorted list across its lanes.  A tile of 32 lanes x 4 vectors enters the
//             list only where it holds a logit above the list's last one and the last one
//             of the CTA's best list, so the list costs little once it is warm.
//   finish    CTA per request (programmatic dependent): merges each row's lists and sums,
//             then merges the rows by their scores in fp64.  The sums carry an error of
//             about 1e-7 from ex2.approx and fp32; where two chosen candidates of different
//             beams are closer than kNearTie, the lse of the request's beams is computed
//             again in fp64 (about one request in a thousand), so the order does not
//             depend on rounding.
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
constexpr int kVecs = 4;  // 16-byte vectors per lane and tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kNearTie = 2e-6;

struct BeamArgs {
  const void* logits;
  int64_t row_stride, vocab;
  const float* scores;
  const uint8_t* finished;
  int64_t eos;
  int num_beams, num_select, parts;
  int64_t part_vecs;  // 16-byte vectors per part
  uint64_t* keys;     // [row][part][num_select], best first; 0 = none
  float2* sums;       // [row][part] (m, s): sum of 2^(x log2e) = s 2^m
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
__device__ __forceinline__ uint64_t make_key(float x, uint32_t i) { return uint64_t(ordered(x)) << 32 | uint32_t(~i); }
__device__ __forceinline__ float key_logit(uint64_t k) { return unordered(uint32_t(k >> 32)); }
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~uint32_t(k); }

// The best `n` keys of a warp, best first: lane l holds entries l and (KL = 2) l + 32.
template <int KL>
struct TopList {
  uint64_t k[KL];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < KL; ++i) k[i] = 0;
  }
  __device__ __forceinline__ uint64_t at(int i) const {
    uint64_t v = __shfl_sync(0xffffffffu, k[0], i & 31);
    if constexpr (KL == 2) {
      const uint64_t w = __shfl_sync(0xffffffffu, k[1], i & 31);
      if (i >= 32) v = w;
    }
    return v;
  }
  // c is the same in every lane; what falls off the end is lost.
  __device__ __forceinline__ void insert(uint64_t c) {
    const int lane = threadIdx.x & 31;
    const int pos = __popc(__ballot_sync(0xffffffffu, k[0] > c));
    const uint64_t up = __shfl_up_sync(0xffffffffu, k[0], 1);
    if constexpr (KL == 2) {
      const int pos2 = 32 + __popc(__ballot_sync(0xffffffffu, k[1] > c));
      const uint64_t last = __shfl_sync(0xffffffffu, k[0], 31);
      const uint64_t up2 = __shfl_up_sync(0xffffffffu, k[1], 1);
      if (pos < 32) {
        k[1] = lane == 0 ? last : up2;
      } else if (lane + 32 >= pos2) {
        k[1] = lane + 32 == pos2 ? c : up2;
      }
    }
    if (lane >= pos) k[0] = lane == pos ? c : up;
  }
};

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

// The n-th largest (n from 1) of the 32 lanes' v, in every lane: one bitonic sort.
__device__ __forceinline__ float nth_largest(float v, int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool keep_max = ((lane & k) == 0) == ((lane & j) == 0);
      v = keep_max ? fmaxf(v, o) : fminf(v, o);
    }
  }
  return __shfl_sync(0xffffffffu, v, n - 1);
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
  __device__ __forceinline__ bool whole(int64_t vec) const {
    const int64_t i = index(vec);
    return i >= 0 && i + VE <= vocab;
  }
  __device__ __forceinline__ uint4 load(int64_t vec) const { return ldg_nc_v4(p + index(vec)); }
  __device__ __forceinline__ void load_ragged(int64_t vec, float* x) const {
    const int64_t i = index(vec);
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = i + e >= 0 && i + e < vocab ? Elem<T>::to_f(p[i + e]) : -INFINITY;
  }
};

template <typename T, int KL>
__global__ void __launch_bounds__(kThreads) beam_partials_kernel(const BeamArgs a) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ int cta_last;  // ordered() of the best last entry of the warps' lists, as a signed maximum
  __shared__ uint64_t sh_keys[kWarps][32 * KL];
  __shared__ float2 sh_sums[kWarps];
  launch_dependents();
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.finished != nullptr && __ldg(a.finished + row) != 0) return;
  const Row<T> r(a, row);
  if (threadIdx.x == 0) cta_last = INT_MIN;
  __syncthreads();
  const int64_t part_begin = part * a.part_vecs;
  const int64_t part_end = min(r.vecs(), part_begin + a.part_vecs);
  // Each warp's run: whole tiles of the part, in vocabulary order.
  constexpr int kTile = 32 * kVecs;
  const int64_t tiles = part_end > part_begin ? (part_end - part_begin + kTile - 1) / kTile : 0;
  const int64_t per_warp = (tiles + kWarps - 1) / kWarps;
  const int64_t begin = part_begin + warp * per_warp * kTile;
  const int64_t end = min(part_end, begin + per_warp * kTile);

  const int K = a.num_select;
  TopList<KL> top;
  top.clear();
  float m = -INFINITY, s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  float last = -INFINITY;  // the list's K-th logit, once it has one
  bool first = true;
  for (int64_t v0 = begin; v0 < end; v0 += kTile) {
    float x[kVecs][VE];
    if (v0 > 0 && v0 + kTile <= end && r.whole(v0 + kTile - 1)) {
      uint4 raw[kVecs];
#pragma unroll
      for (int u = 0; u < kVecs; ++u) raw[u] = r.load(v0 + u * 32 + lane);
#pragma unroll
      for (int u = 0; u < kVecs; ++u) unpack16<T>(raw[u], x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int64_t v = v0 + u * 32 + lane;
        if (v < end) {
          r.load_ragged(v, x[u]);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) x[u][e] = -INFINITY;
        }
      }
    }
    float vmax[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      vmax[u] = x[u][0];
#pragma unroll
      for (int e = 1; e < VE; ++e) vmax[u] = fmaxf(vmax[u], x[u][e]);
    }
    const float g = fmaxf(fmaxf(vmax[0], vmax[1]), fmaxf(vmax[2], vmax[3]));
    // ---- sum of exponentials: m moves only when a tile passes it by more than 2^8 ----
    const float gm = g * kLog2e;
    if (gm > m + 8.f) {
      const float f = ex2(m - gm);  // 0 while m is -inf
      s0 *= f;
      s1 *= f;
      s2 *= f;
      s3 *= f;
      m = gm;
    }
    // m is -inf while every logit was: nothing to add, except that a NaN has to show in the sum
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
#pragma unroll
      for (int e = 0; e < VE; e += 4) {
        s0 += ex2(fmaf(x[u][e], kLog2e, -ms));
        s1 += ex2(fmaf(x[u][e + 1], kLog2e, -ms));
        s2 += ex2(fmaf(x[u][e + 2], kLog2e, -ms));
        s3 += ex2(fmaf(x[u][e + 3], kLog2e, -ms));
      }
    }
    // ---- the list ----
    float least = last, cta = -INFINITY;
    if (first) {
      // At least K of the tile's logits are at or above this (all of them where K > 32 or the tile is ragged).
      least = K <= 32 ? nth_largest(g, K) : -INFINITY;
    } else {
      const int c = *reinterpret_cast<volatile int*>(&cta_last);
      if (c != INT_MIN) cta = unordered(uint32_t(c) ^ 0x80000000u);
    }
    // Later logits of a run lose ties against its list, so > the list's last one; other warps' lists may
    // lie behind this run, so >= theirs.  The first tile fills the list: >=, and -inf counts.
    auto hit = [&](float y) { return first ? y >= least : (y > least && y >= cta && y >= last); };
    if (__any_sync(0xffffffffu, hit(g))) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        if (!__any_sync(0xffffffffu, hit(vmax[u]))) continue;
        const int64_t i0 = r.index(v0 + u * 32 + lane);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int64_t i = i0 + e;
          // (the bounds matter in the first tile only, where -inf fills the list)
          const bool in = v0 + u * 32 + lane < end && i >= 0 && i < a.vocab;
          uint32_t mask = __ballot_sync(0xffffffffu, in && hit(x[u][e]));
          const uint64_t key = make_key(x[u][e], uint32_t(i));
          while (mask) {
            const int src = __ffs(mask) - 1;
            mask &= mask - 1;
            top.insert(__shfl_sync(0xffffffffu, key, src));
          }
          if (!first) last = key_logit(top.at(K - 1));
        }
      }
      const uint64_t kth = top.at(K - 1);
      if (kth != 0) {
        last = key_logit(kth);
        if (lane == 0) atomicMax(&cta_last, int(uint32_t(kth >> 32) ^ 0x80000000u));
      }
      // Fewer than K logits so far can only be a run that ends inside its first tile.
    }
    first = false;
  }
  // ---- merge the warps' lists and sums ----
  float s = (s0 + s1) + (s2 + s3);
  const float M = warp_max(m);
  s = M == -INFINITY ? s : s * ex2(m - M);  // (a lane without a logit: s = 0, m = -inf)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh_sums[warp] = make_float2(M, s);
#pragma unroll
  for (int j = 0; j < KL; ++j) sh_keys[warp][lane + 32 * j] = top.k[j];
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < kWarps; ++w) {
    uint64_t kth = top.at(K - 1);
    for (int i = 0; i < K; ++i) {
      const uint64_t c = sh_keys[w][i];
      if (c <= kth) break;  // sorted: the rest of the list is smaller
      top.insert(c);
      kth = top.at(K - 1);
    }
  }
  const int64_t at = row * a.parts + part;
#pragma unroll
  for (int j = 0; j < KL; ++j) {
    if (lane + 32 * j < K) a.keys[at * K + lane + 32 * j] = top.k[j];
  }
  if (lane == 0) {
    float mm = -INFINITY;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sh_sums[w].x);
    float ss = 0.f;
    for (int w = 0; w < kWarps; ++w)
      ss += mm == -INFINITY ? sh_sums[w].y : sh_sums[w].y * ex2(sh_sums[w].x - mm);
    a.sums[at] = make_float2(mm, ss);
  }
}

// State of one beam in the finish kernel.
enum { kLive = 0, kDone = 1, kDead = 2 };  // has logits; one continuation; every score is -inf
struct Beam {
  double base;  // score of its best continuation: score + best - lse, exact whatever the logits' size
  float best;   // its largest logit
  int kind;
};
__device__ __forceinline__ bool finite(double x) { return x >= -DBL_MAX && x <= DBL_MAX; }

template <typename T, int KL>
__global__ void __launch_bounds__(kThreads) beam_finish_kernel(const BeamArgs a) {
  extern __shared__ uint64_t row_keys[];  // [num_beams][num_select]
  __shared__ Beam beams[64];
  __shared__ double red[kWarps];
  __shared__ int again;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int W = a.num_beams, K = a.num_select;
  const int64_t row0 = int64_t(blockIdx.x) * W;
  if (threadIdx.x == 0) again = 0;
  __syncthreads();
  grid_dependency_wait();

  // ---- each row's best K and lse ----
  for (int w = warp; w < W; w += kWarps) {
    const int64_t row = row0 + w;
    Beam b;
    b.base = a.scores[row];
    b.best = 0.f;
    b.kind = finite(b.base) ? kDone : kDead;
    if (a.finished == nullptr || a.finished[row] == 0) {
      TopList<KL> top;
      top.clear();
      const int64_t n = int64_t(a.parts) * K;
      const unsigned long long* src = reinterpret_cast<const unsigned long long*>(a.keys) + row * n;
      uint64_t kth = 0;
      for (int64_t i0 = 0; i0 < n; i0 += 32) {
        const uint64_t key = i0 + lane < n ? __ldcg(src + i0 + lane) : 0;
        uint32_t mask = __ballot_sync(0xffffffffu, key > kth);
        while (mask) {
          const int from = __ffs(mask) - 1;
          mask &= mask - 1;
          top.insert(__shfl_sync(0xffffffffu, key, from));
        }
        kth = top.at(K - 1);
      }
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        if (lane + 32 * j < K) row_keys[w * K + lane + 32 * j] = top.k[j];
      }
      b.best = key_logit(top.at(0));
      const float2* sums = a.sums + row * a.parts;
      float m = -INFINITY;
      for (int p = lane; p < a.parts; p += 32) m = fmaxf(m, __ldcg(sums + p).x);
      m = warp_max(m);
      double s = 0.0;
      for (int p = lane; p < a.parts; p += 32) {
        const float2 v = __ldcg(sums + p);
        s += v.x == -INFINITY ? double(v.y) : double(v.y) * exp2(double(v.x) - double(m));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      // s 2^m = sum 2^(x c), c = kLog2e in fp32; taken relative to the largest logit, so that c's own
      // rounding acts on differences of logits only.
      const double above = 0.69314718055994530942 * (log2(s) + (double(m) - double(b.best) * double(kLog2e)));
      if (b.kind == kDone) {
        b.kind = kLive;
        b.base -= above;  // lse - best
        // +inf or only -inf: no distribution.  Otherwise a NaN, or logits so large that x log2e left the
        // range of fp32: fp64 tells.
        if (b.best == INFINITY || b.best == -INFINITY) b.kind = kDead;
        else if (!finite(b.base) && lane == 0) again = 1;
      }
    }
    if (lane == 0) beams[w] = b;
  }
  __syncthreads();

  // base of the live beams (all, or those without one) in fp64
  auto exact_bases = [&](bool all) {
    for (int w = 0; w < W; ++w) {
      if (beams[w].kind != kLive || (!all && finite(beams[w].base))) continue;
      const T* p = static_cast<const T*>(a.logits) + (row0 + w) * a.row_stride;
      const double top = double(beams[w].best);
      double s = 0.0;
      for (int64_t i = threadIdx.x; i < a.vocab; i += kThreads) s += exp(double(Elem<T>::to_f(p[i])) - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) red[warp] = s;
      __syncthreads();
      if (threadIdx.x == 0) {
        double t = 0.0;
        for (int k = 0; k < kWarps; ++k) t += red[k];
        beams[w].base = double(a.scores[row0 + w]) - log(t);
        if (!finite(beams[w].base)) beams[w].kind = kDead;
      }
      __syncthreads();
    }
  };
  if (again) exact_bases(false);

  // Candidate i of beam w: its score and token; false past the vocabulary.
  auto candidate = [&](int w, int i, double* score, int64_t* token) {
    const Beam& b = beams[w];
    *score = -INFINITY;
    *token = i;
    if (i >= K || i >= a.vocab) return false;
    if (b.kind == kLive) {
      const uint64_t key = row_keys[w * K + i];
      *token = key_index(key);
      const float x = key_logit(key);
      if (x != -INFINITY) *score = b.base + (double(x) - double(b.best));
    } else if (b.kind == kDone) {
      if (i == 0) *score = b.base;
      *token = i == 0 ? a.eos : i - 1 + (i - 1 >= a.eos ? 1 : 0);
    }
    return true;
  };

  // ---- the request's best K: a merge of W sorted lists, one or two a lane ----
  for (int pass = 0; pass < 2; ++pass) {
    __syncthreads();
    if (warp == 0) {
      int at[2] = {0, 0};
      double sc[2];
      int64_t tk[2];
      bool have[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) have[j] = lane + 32 * j < W && candidate(lane + 32 * j, 0, &sc[j], &tk[j]);
      double prev = 0.0;
      int prev_w = 0;
      bool near = false;
      for (int n = 0; n <= K; ++n) {
        // the lane's better head, then the warp's: higher score, then lower beam
        int w = -1;
        double best = 0.0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (have[j] && (w < 0 || sc[j] > best)) {
            w = lane + 32 * j;
            best = sc[j];
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const double ob = __shfl_xor_sync(0xffffffffu, best, o);
          const int ow = __shfl_xor_sync(0xffffffffu, w, o);
          if (ow >= 0 && (w < 0 || ob > best || (ob == best && ow < w))) {
            best = ob;
            w = ow;
          }
        }
        if (w < 0) break;  // fewer than K + 1 candidates
        // Close scores of two beams, one of them from logits.  (Beams that are each other's copies tie
        // exactly, in any precision.)
        if (n > 0 && w != prev_w && best != -INFINITY && prev - best < kNearTie &&
            (beams[w].kind == kLive || beams[prev_w].kind == kLive) &&
            !(best == prev && beams[w].kind == beams[prev_w].kind && beams[w].base == beams[prev_w].base &&
              beams[w].best == beams[prev_w].best))
          near = true;
        prev = best;
        prev_w = w;
        if (n == K) break;
        const int j = w >> 5;
        if (lane == (w & 31)) {
          const int64_t o = int64_t(blockIdx.x) * K + n;
          a.tokens[o] = tk[j];
          a.parents[o] = w;
          a.out_scores[o] = float(best);
          ++at[j];
          have[j] = candidate(w, at[j], &sc[j], &tk[j]);
        }
      }
      if (lane == 0) again = near && pass == 0;
    }
    __syncthreads();
    if (again == 0) return;
    exact_bases(true);
  }
}

template <typename T, int KL>
cudaError_t launch_t(const BeamArgs& a, int num_requests, cudaStream_t stream) {
  beam_partials_kernel<T, KL><<<unsigned(num_requests) * a.num_beams * a.parts, kThreads, 0, stream>>>(a);
  cudaError_t ce = cudaGetLastError();
  if (ce != cudaSuccess) return ce;
  const int smem = a.num_beams * a.num_select * 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_requests);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_finish_kernel<T, KL>, a);
}

// Parts a row is cut into: enough CTAs for the device, parts of at least one tile a warp.
int beam_parts(int rows, int64_t vocab, int esize) {
  const int64_t vecs = (vocab * esize + 15) / 16 + 1;
  const int64_t most = std::max<int64_t>(1, vecs / (32 * kVecs * 2));
  const int64_t wanted = (int64_t(device_sm_count()) * 4 + rows - 1) / rows;
  return int(std::max<int64_t>(1, std::min(most, wanted)));
}

}  // namespace

size_t beam_workspace_size(int num_requests, int num_beams, int64_t vocab, int num_select, int esize) {
  const size_t rows = size_t(num_requests) * num_beams;
  const size_t parts = rows * beam_parts(int(rows), vocab, esize);
  return ((parts * num_select * 8 + 255) & ~size_t(255)) + parts * 8;
}

cudaError_t launch_beam_select(const void* logits, int64_t row_stride, int num_requests, int num_beams, int64_t vocab,
                               int dtype, const float* scores, const uint8_t* finished, int64_t eos, int num_select,
                               int64_t* tokens, int64_t* parents, float* out_scores, void* workspace,
                               cudaStream_t stream) {
  const int rows = num_requests * num_beams;
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
  a.parts = beam_parts(rows, vocab, es);
  const int64_t vecs = (vocab * es + 15) / 16 + 1;  // a row may straddle one vector more
  a.part_vecs = (vecs + a.parts - 1) / a.parts;
  a.keys = static_cast<uint64_t*>(workspace);
  const size_t key_bytes = (size_t(rows) * a.parts * num_select * 8 + 255) & ~size_t(255);
  a.sums = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + key_bytes);
  a.tokens = tokens;
  a.parents = parents;
  a.out_scores = out_scores;
#define FVB_BEAM(T) \
  (num_select <= 32 ? launch_t<T, 1>(a, num_requests, stream) : launch_t<T, 2>(a, num_requests, stream))
  if (dtype == FVB_DTYPE_BF16) return FVB_BEAM(__nv_bfloat16);
  if (dtype == FVB_DTYPE_F16) return FVB_BEAM(__half);
  return FVB_BEAM(float);
#undef FVB_BEAM
}

}  // namespace fvb
