// Decode paged attention on the tensor cores with the keys as matrix rows, 16-bit types:
// the window decode and the sequences' own keys behind a shared prefix.
//
// One query token has a GQA group's few heads to offer, a 128-row tile of query rows stays
// nearly empty, and its softmax still pays for every row.  Here the products are transposed,
// so that the 128 rows are keys (S) and head dims (O) and the heads are the 16 columns:
//
//   S^T[128 keys x 16]  = K [128 x D]   Q^T           (A = K tile, K-major;  B = Q, K-major)
//   O^T[D x 16]        += V^T[D x 128]  P^T[128 x 16] (A = V tile, MN-major; B = P, K-major)
//
// The tensor cores take P in 16 bits, so each probability is fed as two of them, p = hi + lo with hi = p rounded and
// lo = p - hi rounded: off by 2^-16 of itself in bf16, 2^-22 in fp16, where one of them alone (2^-8, 2^-11) adds as
// much error as the output's own rounding (measured, 256 sequences of window 1024: 0.0023 off against 0.0017, and the
// same 173 us).  hi and lo are rows of P, so they take columns of O that the group's
// heads leave unused (8 + h; from nine heads on 16 + h, N = 32), and are added in fp32 when the unit ends.  fp16 has
// no bits left below 2^-24, which long rows of small weights behind a large one reach: its lo is kept times 2^11.
//
// A softmax thread then owns one key: it takes its scores of the group's heads from TMEM,
// the mask is one predicate, and the exponentials are keys x heads, as they should be.
// What is left is the stream of K and V, 64 KB per tile of 128 keys at D 128.
//
//   work      every (sequence, kv head) is a unit of tiles of 8 pages, all units one line of
//             T tiles, and CTA c of G (one per SM) takes tiles [T c / G, T (c + 1) / G)
//             whatever the sequences' lengths are: no tail, at most two cut units a CTA.
//             Each CTA scans the tile counts itself (one load per sequence), so there is
//             no plan kernel in front.
//   warp 0/2  K / V producers: 8 page ids of the next tile are read by 8 lanes one tile
//             ahead, and each lane issues its page's TMA boxes; the rings run on across
//             units, so neither a unit's start nor its end interrupts the stream.
//   warp 1    issues every MMA: S of tile j, then O of tile j - 1.
//   warp 3    the heads' q of the next unit into shared memory (128-byte swizzle).
//   warps 4-7 softmax, one thread per key: P = 2^(s - m) with one reference maximum m per
//             head that moves only when a score passes it by more than 2^8 (one barrier with
//             an OR per tile tells), sums per thread until the unit ends, P to shared
//             memory as the next MMA's B; at a unit's end O / l, thread = head dim.
//
// A unit that one CTA holds whole is written directly (window) or as one partial (own keys
// behind a prefix); a cut one leaves partials by CTA, which a small dependent kernel merges.
//
// Bound by HBM: a tile takes 1.64 us of each of the 148 SMs' time, 5.9 TB/s; the first tile waits about 6 us for
// launch, scan, page ids and the first bytes.  Measured: 256 sequences x 8 heads x 128, group 2, window 1024 (1.04 GB)
// 164-173 us = 6.0-6.3 TB/s of the 6.54 a copy reaches (split-KV kernel: 189); 32 x 8 x 128, group 8, window 4096
// (0.555 GB) 93-97 us = 5.7-5.9 TB/s (on 128-row tiles of query rows, where the softmax bounds it: 185).
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace fvb {
namespace {

constexpr int kKeys = kKeysTile;    // keys per tile
constexpr int kTilePages = kKeys / kPageSize;
constexpr int kThreads = 256;
constexpr int kCols = kKeysCols;     // heads of a unit: columns of both products
constexpr int kHalf = kKeys * 128;  // 128 keys x one 128-byte swizzle span
constexpr int kBHalf = kCols * 128; // 16 rows of Q x one span
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrowLog2 = 8.0f;
constexpr float kLeast = -1e37f;
template <typename T>
constexpr float kLoScale = std::is_same<T, __half>::value ? 2048.f : 1.f;

template <int D, int HV, int MODE>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kHalves * kHalf;
  static constexpr int kStages = D == 128 ? 3 : 6;  // of K and of V
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kStages * kTileBytes;
  static constexpr int kOffQ = 2 * kStages * kTileBytes;        // two units' q
  static constexpr int kLoCol = HV <= 8 ? 8 : kCols;            // column of head 0's lo
  static constexpr int kPCols = 2 * kLoCol;                     // rows of P: hi and lo
  static constexpr int kPHalf = kPCols * 128;
  static constexpr int kOffP = kOffQ + 2 * kHalves * kBHalf;    // two tiles' P
  static constexpr int kOffBar = kOffP + 2 * 2 * kPHalf;
  // k_full, k_empty, v_full, v_empty [kStages]; s_full, p_full, pv_done, q_full, q_empty, o_empty [2]
  static constexpr int kNumBars = 4 * kStages + 12;
  static constexpr int kOffRed = kOffBar + kNumBars * 8 + 16;   // float[4][kCols]
  // int[num_seqs + 1] tiles before each sequence; window: int[num_seqs] its length; rest: int[num_seqs] keys skipped,
  // uint8_t[num_seqs] keys that its last tile lacks
  static constexpr int kOffSeqs = kOffRed + 4 * kCols * 4;
  static constexpr int smem_bytes(int num_seqs) {
    return kOffSeqs + (2 * num_seqs + 1) * 4 + (MODE == kKeysRest ? num_seqs : 0) + 1024;
  }
  static constexpr uint32_t kTmemCols = HV <= 8 ? 64 : 128;  // S twice, O twice
  static_assert(smem_bytes(kKeysMaxSeqs) <= 227 * 1024, "shared memory budget");
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int site) {
  const bool ok = mbar_wait(bar, parity, err, site);
  return __all_sync(0xffffffffu, ok);
}

// Maximum over the warp in one instruction (sm_100).
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

struct KeysArgs {
  const void* q;
  void* out;
  int64_t num_blocks;
  int n_kv_heads, group, chunks, num_seqs;
  const int32_t* block_tables;
  int max_blocks_per_seq;
  const int32_t* kv_lens;
  int kv_cap;
  QOLayout lay;
  DecodeExtra ex;
  int4* cuts;   // window: [G] {sequence, unit, last CTA, -} of the unit each CTA begins and leaves unfinished
  int4* spans;  // rest: [num_seqs] {keys of its shared prefix, tiles, tiles before it, tiles of the batch}
  float *cut_o, *cut_l;  // [G][2][kCols][D], [G][2][kCols]: cut units, begun before / in this CTA
  float *full_o, *full_l;  // [seq][head][D], [seq][head]: whole units (rest)
  int* err;
};

// The units of a CTA's tiles, in order: unit `u` of sequence `b`, its tiles [t0, t1) of n.
struct Walk {
  const int32_t* cum;
  int num_seqs, units;
  int64_t g, end;
  int b, u, t0, t1, n;
  __device__ __forceinline__ Walk(const int32_t* cum_, int num_seqs_, int units_, int64_t total, int grid)
      : cum(cum_), num_seqs(num_seqs_), units(units_) {
    g = total * blockIdx.x / grid;
    end = total * (blockIdx.x + 1) / grid;
    if (g >= end) return;
    int lo = 0, hi = num_seqs - 1;  // last sequence that begins at or before g (an empty one is followed by others)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (int64_t(cum[mid]) * units <= g) lo = mid; else hi = mid - 1;
    }
    b = lo;
    n = cum[b + 1] - cum[b];
    const int64_t in = g - int64_t(cum[b]) * units;
    u = int(in / n);
    t0 = int(in - int64_t(u) * n);
    t1 = int(min(int64_t(n), t0 + (end - g)));
  }
  __device__ __forceinline__ bool more() const { return g < end; }
  __device__ __forceinline__ void next() {
    g += t1 - t0;
    if (g >= end) return;
    if (++u == units) {
      u = 0;
      do ++b; while (cum[b + 1] == cum[b]);
      n = cum[b + 1] - cum[b];
    }
    t0 = 0;
    t1 = int(min(int64_t(n), end - g));
  }
};

// Pages of sequence b's visible keys: page number c of the unit is table page c for c < span.head, else c + span.gap.
template <int MODE>
__device__ __forceinline__ KeySpan unit_span(const KeysArgs& a, int kv_len, int skip) {
  if constexpr (MODE == kKeysWindow) return window_span(kv_len, kv_len, a.ex.window, a.ex.sinks, kPageSize);
  const int pages = (kv_len + kPageSize - 1) / kPageSize, first = skip / kPageSize;
  return KeySpan{0, first, max(pages - first, 0), 0};
}

template <typename T, int D, int HV, int MODE>
__global__ void __launch_bounds__(kThreads, 1) decode_keys_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                  const __grid_constant__ CUtensorMap vmap,
                                                                  const __grid_constant__ KeysArgs a) {
  using C = Cfg<D, HV, MODE>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kS = C::kStages;
  launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* k_empty = k_full + kS;
  uint64_t* v_full = k_empty + kS;
  uint64_t* v_empty = v_full + kS;
  uint64_t* s_full = v_empty + kS;
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_full = pv_done + 2;
  uint64_t* q_empty = q_full + 2;
  uint64_t* o_empty = q_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 2);
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  int32_t* cum = reinterpret_cast<int32_t*>(smem + C::kOffSeqs);
  int32_t* lens = cum + a.num_seqs + 1;  // window
  int32_t* skips = lens;                 // rest
  uint8_t* tails = reinterpret_cast<uint8_t*>(skips + a.num_seqs);
  // Length of sequence b, and the keys of it that are not this kernel's.
  auto skip_of = [&](int b) { return MODE == kKeysRest ? skips[b] : 0; };
  auto len_of = [&](int b) {
    return MODE == kKeysRest ? skips[b] + (cum[b + 1] - cum[b]) * kKeys - tails[b] : lens[b];
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_heads = a.n_kv_heads * a.group;
  const int units = a.n_kv_heads * a.chunks;
  const int B = a.num_seqs;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kKeys);
      mbar_init(&pv_done[i], 1);
      mbar_init(&q_full[i], 32);
      mbar_init(&q_empty[i], 1);
      mbar_init(&o_empty[i], kKeys);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }

  // ---- tiles of every sequence, and their running sum ----
  {
    int32_t* warp_sum = reinterpret_cast<int32_t*>(red);
    // The groups' table in the K ring, which is still empty, where it fits (it may hold empty groups).  Without
    // groups there is no table to read: both pointers may be null.
    int32_t* groups = reinterpret_cast<int32_t*>(smem + C::kOffK);
    const int G = a.ex.num_groups;
    const bool staged = MODE == kKeysRest && G > 0 && (2 * G + 1) * 4 <= kS * C::kTileBytes;
    if (staged) {
      for (int g = threadIdx.x; g <= G; g += kThreads) {
        groups[g] = __ldg(a.ex.cu_groups + g);
        if (g < G) groups[G + 1 + g] = __ldg(a.ex.prefix_lens + g);
      }
      __syncthreads();
    }
    DecodeExtra gx = a.ex;
    if (staged) {
      gx.cu_groups = groups;
      gx.prefix_lens = groups + G + 1;
    }
    int carry = 0;
    if (threadIdx.x == 0) cum[0] = 0;
    for (int base = 0; base < B; base += kThreads) {
      const int b = base + threadIdx.x;
      int n = 0;
      if (b < B) {
        int skip = 0;
        if constexpr (MODE == kKeysRest) {
          int lo = 0, hi = G;  // first group whose end lies behind b
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (gx.cu_groups[mid + 1] > b) hi = mid; else lo = mid + 1;
          }
          if (gx.prefix_cap > 0 && lo < G) {
            const int2 rows = group_rows(gx, lo, B);
            if (b >= rows.x) skip = group_prefix(gx, lo, rows);
          }
        }
        int kv = __ldg(a.kv_lens + b);
        if (blockIdx.x == 0 && kv > a.kv_cap) record_error(a.err, FVB_ERR_INVALID_ARGUMENT, b);
        kv = min(max(kv, 0), a.kv_cap);
        n = (unit_span<MODE>(a, kv, skip).count + kTilePages - 1) / kTilePages;
        if constexpr (MODE == kKeysRest) {
          skips[b] = skip;
          tails[b] = uint8_t(n > 0 ? skip + n * kKeys - kv : 0);
        } else {
          lens[b] = kv;
        }
      }
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) warp_sum[warp] = upto;
      __syncthreads();
      int before = carry;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += warp_sum[w];
        carry += warp_sum[w];
      }
      if (b < B) cum[b + 1] = before + upto;
      __syncthreads();
    }
    // The table's bytes are next written by TMA: ordinary accesses to them come first (a barrier for all threads
    // follows before any copy is issued).
    if (staged) fence_proxy_async_smem();
  }
  if constexpr (MODE == kKeysRest) {
    if (blockIdx.x == 0) {
      for (int g = threadIdx.x; g < a.ex.num_groups; g += kThreads) {
        const int lo = __ldg(a.ex.cu_groups + g), hi = __ldg(a.ex.cu_groups + g + 1);
        if (lo < 0 || hi < lo || hi > B || __ldg(a.ex.prefix_lens + g) < 0)
          record_error(a.err, FVB_ERR_INVALID_ARGUMENT, g);
      }
      for (int b = threadIdx.x; b < B; b += kThreads)
        a.spans[b] = make_int4(skips[b], cum[b + 1] - cum[b], cum[b], cum[B]);
    }
  }
  if constexpr (MODE == kKeysWindow) {  // empty contexts: zeros
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
      if (cum[b + 1] != cum[b]) continue;
      for (int e = threadIdx.x; e < n_heads * D; e += kThreads)
        static_cast<T*>(a.out)[int64_t(b) * a.lay.o_ts + int64_t(e / D) * a.lay.o_hs + e % D] = Elem<T>::from_f(0.f);
    }
  }
  const int64_t total = int64_t(cum[B]) * units;
  const int grid = int(min(int64_t(gridDim.x), total));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto col_s = [&](int j) { return tmem + uint32_t(j & 1) * kCols; };
  auto col_o = [&](int i) { return tmem + 32u + uint32_t(i & 1) * C::kPCols; };

  if (MODE == kKeysWindow && threadIdx.x == 96) {  // a lane that waits for nothing yet
    int4 cut = make_int4(-1, 0, 0, 0);
    if (int(blockIdx.x) < grid) {
      Walk w(cum, B, units, total, grid);
      while (w.g + (w.t1 - w.t0) < w.end) w.next();  // the CTA's last unit
      if (w.t0 == 0 && w.t1 < w.n) {
        const int64_t end = (int64_t(cum[w.b]) * units + int64_t(w.u + 1) * w.n);
        cut = make_int4(w.b, w.u, keys_cta_of(end - 1, total, grid), 0);
      }
    }
    a.cuts[blockIdx.x] = cut;
  }
  if (int(blockIdx.x) < grid) {
    Walk walk(cum, B, units, total, grid);
    if (warp == 0 || warp == 2) {
      // ======================= producers: warp 0 = K, warp 2 = V =======================
      const CUtensorMap* map = warp == 0 ? &kmap : &vmap;
      uint64_t* full = warp == 0 ? k_full : v_full;
      uint64_t* empty = warp == 0 ? k_empty : v_empty;
      uint8_t* ring = smem + (warp == 0 ? C::kOffK : C::kOffV);
      if (lane == 0) prefetch_tensormap(map);
      // Page id of this lane's page (lanes 0 .. 7) of tile t, -1 past the unit; read one tile ahead and looked
      // at only when its turn comes.
      KeySpan span{};
      int span_of = -1;
      auto page_id = [&](const Walk& w, int t, bool& in) {
        if (w.b != span_of) {
          span_of = w.b;
          span = unit_span<MODE>(a, len_of(w.b), skip_of(w.b));
        }
        const int c = t * kTilePages + lane;
        in = lane < kTilePages && c < span.count;
        const int32_t* table = a.block_tables + int64_t(w.b) * a.max_blocks_per_seq;
        return in ? __ldg(table + (c < span.head ? c : c + span.gap)) : 0;
      };
      bool in = false;
      int id = page_id(walk, walk.t0, in);
      int j = 0;
      bool ok = true;
      for (; walk.more() && ok; walk.next()) {
        const int kvh = walk.u / a.chunks;
        for (int t = walk.t0; t < walk.t1; ++t, ++j) {
          const int st = j % kS;
          if (j >= kS) ok = warp_wait(&empty[st], (j / kS - 1) & 1, a.err, 0x400 + warp);
          if (!ok) break;
          if (in && (id < 0 || id >= a.num_blocks)) {
            record_error(a.err, FVB_ERR_BAD_PAGE, walk.b);
            id = 0;
          }
          const int now = (id * a.n_kv_heads + kvh) * kPageSize;
          const int pages = __popc(__ballot_sync(0xffffffffu, in));
          int rows[kTilePages];
#pragma unroll
          for (int i = 0; i < kTilePages; ++i) rows[i] = __shfl_sync(0xffffffffu, now, i);
          if (t + 1 < walk.t1) {
            id = page_id(walk, t + 1, in);
          } else {
            Walk ahead = walk;
            ahead.next();
            if (ahead.more()) id = page_id(ahead, ahead.t0, in);
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[st], uint32_t(pages) * kPageSize * D * 2);
            uint8_t* dst = ring + st * C::kTileBytes;
#pragma unroll
            for (int i = 0; i < kTilePages; ++i) {
              if (i < pages) {  // a tile's pages are its first ones
#pragma unroll
                for (int h = 0; h < C::kHalves; ++h)
                  tma_load_2d(dst + h * kHalf + i * kPageSize * 128, map, h * 64, rows[i], &full[st]);
              }
            }
          }
          __syncwarp();
        }
      }
    } else if (warp == 1) {
      // ============================ MMA issuer ============================
      if (lane == 0) {
        constexpr uint32_t idesc_s = umma_idesc_f16(kBF16, 128, kCols, false);
        constexpr uint32_t idesc_o = umma_idesc_f16(kBF16, 128, C::kPCols, false, true);
        const uint64_t dk = umma_sdesc_sw128(smem_u32(smem + C::kOffK), 16, 1024);
        // At D 64 both halves of the 128 rows read the same 64 dims; rows 64 .. 127 of O are not used.
        const uint64_t dv = umma_sdesc_sw128(smem_u32(smem + C::kOffV), D == 128 ? kHalf : 0, 1024);
        const uint64_t dq = umma_sdesc_sw128(smem_u32(smem + C::kOffQ), 16, 1024);
        const uint64_t dp = umma_sdesc_sw128(smem_u32(smem + C::kOffP), 16, 1024);
        bool ok = true;
        auto issue_pv = [&](int j, int item, bool first) {
          const int st = j % kS;
          ok = mbar_wait(&v_full[st], (j / kS) & 1, a.err, 0x410) &&
               mbar_wait(&p_full[j & 1], (j >> 1) & 1, a.err, 0x411);
          if (ok && first && item >= 2) ok = mbar_wait(&o_empty[item & 1], ((item >> 1) - 1) & 1, a.err, 0x412);
          if (!ok) return;
          tc_fence_after();
          const uint64_t vd = dv + uint64_t((st * C::kTileBytes) >> 4);
          const uint64_t pd = dp + uint64_t(((j & 1) * 2 * C::kPHalf) >> 4);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_f16_ss(col_o(item), vd + uint64_t((kk * 16 * 128) >> 4),
                        pd + uint64_t(((kk >> 2) * C::kPHalf + (kk & 3) * 32) >> 4), idesc_o, first && kk == 0 ? 0u : 1u);
          umma_commit(&v_empty[st]);
          umma_commit(&pv_done[j & 1]);
        };
        int j = 0, item = 0;
        int prev_item = 0;
        bool prev_first = false;
        for (; walk.more() && ok; walk.next(), ++item) {
          for (int t = walk.t0; t < walk.t1 && ok; ++t, ++j) {
            const int st = j % kS;
            ok = mbar_wait(&k_full[st], (j / kS) & 1, a.err, 0x413);
            if (ok && t == walk.t0) ok = mbar_wait(&q_full[item & 1], (item >> 1) & 1, a.err, 0x414);
            if (!ok) break;
            tc_fence_after();
            // S buffer j & 1 is free: P of tile j - 2, made from it, was waited for before O of that tile
            const uint64_t kd = dk + uint64_t((st * C::kTileBytes) >> 4);
            const uint64_t qd = dq + uint64_t(((item & 1) * C::kHalves * kBHalf) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16_ss(col_s(j), kd + uint64_t(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4),
                          qd + uint64_t(((kk >> 2) * kBHalf + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
            umma_commit(&s_full[j & 1]);
            umma_commit(&k_empty[st]);
            if (t == walk.t1 - 1) umma_commit(&q_empty[item & 1]);
            if (j > 0) issue_pv(j - 1, prev_item, prev_first);
            prev_item = item;
            prev_first = t == walk.t0;
          }
        }
        if (ok && j > 0) issue_pv(j - 1, prev_item, prev_first);
      }
      __syncwarp();
    } else if (warp == 3) {
      // ============================ q of each unit ============================
      bool ok = true;
      for (int item = 0; walk.more() && ok; walk.next(), ++item) {
        const int kvh = walk.u / a.chunks, chunk = walk.u % a.chunks;
        const int head0 = kvh * a.group + chunk * kCols, nvh = min(kCols, a.group - chunk * kCols);
        if (item >= 2) ok = warp_wait(&q_empty[item & 1], ((item >> 1) - 1) & 1, a.err, 0x420);
        if (!ok) break;
        const uint32_t dst = smem_u32(smem + C::kOffQ + (item & 1) * C::kHalves * kBHalf);
        const T* src = static_cast<const T*>(a.q) + int64_t(walk.b) * a.lay.q_ts + int64_t(head0) * a.lay.q_hs;
        for (int e = lane; e < nvh * (D / 8); e += 32) {  // 16-byte vectors
          const int r = e / (D / 8), c = e % (D / 8);
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(src + int64_t(r) * a.lay.q_hs) + c);
          sts_v4(dst + (c >> 3) * kBHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4), x);
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full[item & 1]);
      }
    } else {
      // ============================ softmax, one thread per key ============================
      const int key_t = threadIdx.x - 128;
      const uint32_t t_row = uint32_t((warp & 3) * 32) << 16;
      const float scale = kLog2e * rsqrtf(float(D));
      // this key's place in a row of P: [half][column / 8][column % 8] rows of 128 bytes, 16-byte chunks swizzled
      const uint32_t p_base = smem_u32(smem + C::kOffP) + (key_t >> 6) * C::kPHalf + (key_t & 7) * 2;
      const int p_chunk = (key_t & 63) >> 3;
      // A wait that gives up (ok = false) ends no loop here: the four warps share barriers, so a warp that has
      // failed goes on without waiting or touching TMEM, and the others fail or finish in their own time.
      bool ok = true;
      int j = 0;
      // The unit whose last P V is under way: its result is taken when the next unit's first P is out, so that
      // product never holds up the softmax.
      struct Done {
        int item, tile, head0, nvh, b;
        int64_t at;      // partial's row, or -1: the unit goes to `out`
        float *o, *l;
      } done{};
      done.item = -1;
      float m[HV], l[HV], m_done[HV], l_done[HV];
      auto load_o = [&](int item, uint32_t(&o)[C::kPCols]) {
        if constexpr (C::kPCols == 16) tmem_ld_16cols(col_o(item) + t_row, o);
        else tmem_ld_32cols(col_o(item) + t_row, o);
      };
      auto finish = [&]() {
        // Sums over the 128 keys: lanes trade halves of the heads until each holds one, then warps meet in `red`.
        float s[HV];
#pragma unroll
        for (int h = 0; h < HV; ++h) s[h] = l_done[h];
        int mine = 0;
#pragma unroll
        for (int n = HV / 2, o = 16; n >= 1; n /= 2, o /= 2) {
          const bool upper = lane & o;
#pragma unroll
          for (int h = 0; h < n; ++h) {
            const float give = upper ? s[h] : s[h + n], keep = upper ? s[h + n] : s[h];
            s[h] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
          mine += upper ? n : 0;
        }
#pragma unroll
        for (int o = 16 / HV; o > 0; o >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
        if (lane % (32 / HV) == 0) red[(warp & 3) * kCols + mine] = s[0];
        named_barrier(1, kKeys);
        ok = ok && warp_wait(&pv_done[done.tile & 1], (done.tile >> 1) & 1, a.err, 0x434);
        uint32_t o[C::kPCols] = {};
        if (ok) {
          tc_fence_after();
          load_o(done.item, o);
          tc_fence_before();
        }
        mbar_arrive(&o_empty[done.item & 1]);
        // thread = head dim
#pragma unroll
        for (int h = 0; h < HV; ++h) {
          const float L = (red[h] + red[kCols + h]) + (red[2 * kCols + h] + red[3 * kCols + h]);
          // (an infinite V: lo = 0 of it is NaN, hi alone tells)
          const float hi = __uint_as_float(o[h]);
          const float sum = fmaf(__uint_as_float(o[C::kLoCol + h]), 1.f / kLoScale<T>, hi);
          const float v = (fabsf(hi) < INFINITY ? sum : hi) / L;
          if (h >= done.nvh || key_t >= D) continue;
          if (MODE == kKeysWindow && done.at < 0) {
            static_cast<T*>(a.out)[int64_t(done.b) * a.lay.o_ts + int64_t(done.head0 + h) * a.lay.o_hs + key_t] =
                Elem<T>::from_f(v);
          } else {
            done.o[(done.at + h) * D + key_t] = L == 0.f ? 0.f : v;  // (every score was -inf)
            if (key_t == 0) done.l[done.at + h] = m_done[h] + __log2f(L);
          }
        }
        named_barrier(1, kKeys);  // red is read before its next use
        done.item = -1;
      };
      for (int item = 0; walk.more(); walk.next(), ++item) {
        const int b = walk.b;
        const int kvh = walk.u / a.chunks, chunk = walk.u % a.chunks;
        const int head0 = kvh * a.group + chunk * kCols, nvh = min(kCols, a.group - chunk * kCols);
        const int kv_len = len_of(b);
        const KeySpan span = unit_span<MODE>(a, kv_len, skip_of(b));
#pragma unroll
        for (int h = 0; h < HV; ++h) {
          m[h] = -INFINITY;
          l[h] = 0.f;
        }
        for (int t = walk.t0; t < walk.t1; ++t, ++j) {
          const int c0 = t * kTilePages, c = c0 + (key_t >> 4);
          const int key = (c < span.head ? c : c + span.gap) * kPageSize + (key_t & 15);
          bool valid = c < span.count && key < kv_len;
          if (MODE == kKeysWindow) valid = valid && (key >= span.lo || key < a.ex.sinks);
          // tiles that may hold an invisible key: the last, and those around the gap
          const bool ragged = c0 + kTilePages >= span.count ||
                              (MODE == kKeysWindow && c0 <= span.head && c0 + kTilePages >= span.head);
          ok = ok && warp_wait(&s_full[j & 1], (j >> 1) & 1, a.err, 0x430);
          uint32_t sr[16];
          if (ok) {
            tc_fence_after();
            tmem_ld_16cols(col_s(j) + t_row, sr);
          }
          float x[HV];
          bool grow = false;
#pragma unroll
          for (int h = 0; h < HV; ++h) {
            x[h] = valid && ok ? __uint_as_float(sr[h]) * scale : -INFINITY;
            if (h < nvh) grow = grow || x[h] > m[h] + kGrowLog2;
          }
          if (t == walk.t0 || named_barrier_or(1, kKeys, grow)) {
            // New reference maxima: those of the tile where they exceed the old by more than 2^8 (at the
            // unit's first tile always; a tile holds a visible key).
#pragma unroll
            for (int h = 0; h < HV; ++h) {
              const float mx = warp_max(x[h]);
              if (lane == 0) red[(warp & 3) * kCols + h] = mx;
            }
            named_barrier(1, kKeys);
            float f[HV];
#pragma unroll
            for (int h = 0; h < HV; ++h) {
              const float mx = fmaxf(fmaxf(red[h], red[kCols + h]), fmaxf(red[2 * kCols + h], red[3 * kCols + h]));
              f[h] = 1.f;
              if (t == walk.t0) {
                // finite though every score were -inf (infinite keys): P is 0 then, and the next tile's maximum larger
                m[h] = fmaxf(mx, kLeast);
              } else if (mx > m[h] + kGrowLog2) {
                f[h] = fast_exp2(m[h] - mx);
                m[h] = mx;
              }
              l[h] *= f[h];
            }
            if (t > walk.t0) ok = ok && warp_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, a.err, 0x431);
            if (t > walk.t0 && ok) {
              tc_fence_after();
              uint32_t o[C::kPCols];
              load_o(item, o);
#pragma unroll
              for (int h = 0; h < HV; ++h) {
                o[h] = __float_as_uint(__uint_as_float(o[h]) * f[h]);
                o[C::kLoCol + h] = __float_as_uint(__uint_as_float(o[C::kLoCol + h]) * f[h]);
              }
              if constexpr (C::kPCols == 16) tmem_st_16cols(col_o(item) + t_row, o);
              else tmem_st_32cols(col_o(item) + t_row, o);
              tmem_wait_st();
            }
            named_barrier(1, kKeys);  // red is read before its next use
          }
          // P of tile j - 2 has been read
          if (j >= 2) ok = ok && warp_wait(&pv_done[j & 1], ((j >> 1) - 1) & 1, a.err, 0x432);
          const uint32_t p_row = p_base + (j & 1) * 2 * C::kPHalf;
#pragma unroll
          for (int h = 0; h < HV; ++h) {
            const float p = fast_exp2(x[h] - m[h]);
            l[h] += p;
            const T hi = Elem<T>::from_f(p);
            const T lo = Elem<T>::from_f((p - Elem<T>::to_f(hi)) * kLoScale<T>);
            const uint32_t at = p_row + h * 128 + ((p_chunk ^ (h & 7)) << 4);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(*reinterpret_cast<const uint16_t*>(&hi)) : "memory");
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + C::kLoCol * 128),
                         "h"(*reinterpret_cast<const uint16_t*>(&lo))
                         : "memory");
          }
          if (ragged) {
            // V of invisible keys may be stale shared memory or an unused slot, and 0 * NaN is not 0.
            const int st = j % kS;
            ok = ok && warp_wait(&v_full[st], (j / kS) & 1, a.err, 0x433);
            if (ok && !valid) {
#pragma unroll
              for (int h = 0; h < C::kHalves; ++h) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  sts_v4(smem_u32(smem + C::kOffV + st * C::kTileBytes + h * kHalf + key_t * 128 + i * 16),
                         make_uint4(0, 0, 0, 0));
              }
            }
          }
          fence_proxy_async_smem();
          tc_fence_before();
          mbar_arrive(&p_full[j & 1]);
          if (done.item >= 0) finish();
        }
        const bool whole = walk.t0 == 0 && walk.t1 == walk.n;
        done.item = item;
        done.tile = j - 1;
        done.head0 = head0;
        done.nvh = nvh;
        done.b = b;
        if (whole) {
          done.at = MODE == kKeysWindow ? -1 : int64_t(b) * n_heads + head0;
          done.o = a.full_o;
          done.l = a.full_l;
        } else {
          done.at = (int64_t(blockIdx.x) * 2 + (walk.t0 > 0 ? 0 : 1)) * kCols;
          done.o = a.cut_o;
          done.l = a.cut_l;
        }
#pragma unroll
        for (int h = 0; h < HV; ++h) {
          m_done[h] = m[h];
          l_done[h] = l[h];
        }
      }
      if (done.item >= 0) finish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
  if (blockIdx.x == gridDim.x - 1) {
    // As a programmatic dependent of the prefix kernel (which writes nothing read here) this grid may run
    // beside it; its last CTA holds the grid open until that kernel has completed, so what waits for this
    // grid (the merge) sees its partials too.
    grid_dependency_wait();
  }
}

// Cut units of the window form: CTA (c, h) merges head h of the unit that CTA c of the decode kernel begins
// and leaves unfinished, from the partials of the CTAs that hold it.
constexpr int kCutThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kCutThreads) keys_cut_kernel(const KeysArgs a) {
  constexpr int kWays = kCutThreads / D;
  __shared__ float sh_o[kWays][D], sh_m[kWays], sh_l[kWays];
  grid_dependency_wait();
  const int c = blockIdx.x, h = blockIdx.y;
  const int4 cut = __ldcg(a.cuts + c);  // {sequence, unit, last CTA, -}; -1: this CTA begins no cut unit
  if (cut.x < 0) return;
  const int kvh = cut.y / a.chunks, chunk = cut.y % a.chunks, last = cut.z;
  if (h >= min(kCols, a.group - chunk * kCols)) return;
  const int way = threadIdx.x / D, d = threadIdx.x % D;
  float m = -INFINITY, l = 0.f, acc = 0.f;
#pragma unroll 4
  for (int k = c + way; k <= last; k += kWays) {
    const int64_t at = (int64_t(k) * 2 + (k == c ? 1 : 0)) * kCols + h;
    const float ls = __ldcg(a.cut_l + at), o = __ldcg(a.cut_o + at * D + d);
    const float mn = fmaxf(m, ls), ref = mn == -INFINITY ? 0.f : mn;
    const float f = fast_exp2(m - ref), w = fast_exp2(ls - ref);
    l = fmaf(l, f, w);
    acc = fmaf(acc, f, w * o);
    m = mn;
  }
  sh_o[way][d] = acc;
  if (d == 0) {
    sh_m[way] = m;
    sh_l[way] = l;
  }
  __syncthreads();
  if (way != 0) return;
  float mx = m;
#pragma unroll
  for (int k = 1; k < kWays; ++k) mx = fmaxf(mx, sh_m[k]);
  l = 0.f;
  acc = 0.f;
#pragma unroll
  for (int k = 0; k < kWays; ++k) {
    const float w = fast_exp2(sh_m[k] - (mx == -INFINITY ? 0.f : mx));
    l = fmaf(sh_l[k], w, l);
    acc = fmaf(sh_o[k][d], w, acc);
  }
  const int head = kvh * a.group + chunk * kCols + h;
  static_cast<T*>(a.out)[int64_t(cut.x) * a.lay.o_ts + int64_t(head) * a.lay.o_hs + d] = Elem<T>::from_f(acc / l);
}

template <typename T, int D, int HV, int MODE>
cudaError_t launch_t(const KeysArgs& a, const void* k_pool, const void* v_pool, int grid, bool dependent,
                     cudaStream_t stream) {
  using C = Cfg<D, HV, MODE>;
  const CUtensorMapDataType tdt =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap kmap, vmap;
  const uint64_t rows = uint64_t(a.num_blocks) * a.n_kv_heads * kPageSize;
  cudaError_t ce = make_tma_2d(&kmap, k_pool, tdt, D, rows, D * 2, 64, kPageSize, true);
  if (ce == cudaSuccess) ce = make_tma_2d(&vmap, v_pool, tdt, D, rows, D * 2, 64, kPageSize, true);
  if (ce == cudaSuccess) ce = set_smem_once<decode_keys_kernel<T, D, HV, MODE>>(C::smem_bytes(kKeysMaxSeqs));
  if (ce != cudaSuccess) return ce;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::smem_bytes(a.num_seqs);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  ce = cudaLaunchKernelEx(&cfg, decode_keys_kernel<T, D, HV, MODE>, kmap, vmap, a);
  if (ce != cudaSuccess || MODE != kKeysWindow) return ce;
  cfg.gridDim = dim3(grid, std::min(kCols, a.group));
  cfg.blockDim = dim3(kCutThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, keys_cut_kernel<T, D>, a);
}

template <typename T, int D, int MODE>
cudaError_t dispatch(const KeysArgs& a, const void* k_pool, const void* v_pool, int grid, bool dependent,
                     cudaStream_t stream) {
  if (a.group <= 2) return launch_t<T, D, 2, MODE>(a, k_pool, v_pool, grid, dependent, stream);
  if (a.group <= 4) return launch_t<T, D, 4, MODE>(a, k_pool, v_pool, grid, dependent, stream);
  if (a.group <= 8) return launch_t<T, D, 8, MODE>(a, k_pool, v_pool, grid, dependent, stream);
  return launch_t<T, D, 16, MODE>(a, k_pool, v_pool, grid, dependent, stream);
}

}  // namespace

bool window_decode_on_keys(int num_seqs, int n_heads, int n_kv_heads, int max_kv_len, int window, int sinks, int dtype,
                           int num_sms) {
  if (dtype == FVB_DTYPE_F32 || num_seqs > kKeysMaxSeqs) return false;  // (the sequence table fills shared memory)
  // A call of this kernel costs 8 us before its first tile and 3 us a unit that has only one tile, and its tiles then
  // stream at HBM's rate whatever the group is.  The split-KV kernel starts in 4 us, but what a page costs it grows
  // with the group's heads, and from five on it is bound by its lanes.  Over 320 calls of random shapes the pages an SM
  // gets at most are what tells them apart; with these limits the choice is 2 % off the better kernel on average.
  // (201 sequences x 8 heads, window 5: 29.7 us here, 8.1 there; 256 x 8, group 2, window 1024: 165.5 and 189;
  // 190 x 2, group 16, window 1512: 67.5 and 157.)
  const int group = n_heads / n_kv_heads;
  const int64_t limit = group <= 4 ? 128 : group <= 8 ? 32 : 16;
  const int64_t pages = window_max_units(max_kv_len, window, sinks, kPageSize);
  return int64_t(num_seqs) * n_kv_heads * pages > limit * num_sms;
}

KeysPlan plan_keys(int num_seqs, int n_heads, int head_dim, int mode, int grid) {
  KeysPlan p{};
  p.grid = grid;
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  const size_t cut = size_t(p.grid) * 2 * kCols, full = mode == kKeysRest ? size_t(num_seqs) * n_heads : 0;
  // cuts [grid] or spans [num_seqs] at 0
  p.off_cut_o = up((mode == kKeysRest ? size_t(num_seqs) : size_t(p.grid)) * 16);
  p.off_cut_l = p.off_cut_o + up(cut * head_dim * 4);
  p.off_full_o = p.off_cut_l + up(cut * 4);
  p.off_full_l = p.off_full_o + up(full * head_dim * 4);
  p.ws_bytes = p.off_full_l + up(full * 4);
  return p;
}

cudaError_t launch_keys_decode(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                               int n_heads, int n_kv_heads, int head_dim, int num_seqs, const int32_t* block_tables,
                               int max_blocks_per_seq, const int32_t* kv_lens, int kv_cap, const DecodeExtra& ex,
                               int mode, int dtype, const KeysPlan& plan, const QOLayout& lay, void* workspace,
                               bool dependent, int* err, cudaStream_t stream) {
  if (num_seqs == 0) return cudaSuccess;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  KeysArgs a{};
  a.q = q;
  a.out = out;
  a.num_blocks = num_blocks;
  a.n_kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads;
  a.chunks = (a.group + kCols - 1) / kCols;
  a.num_seqs = num_seqs;
  a.block_tables = block_tables;
  a.max_blocks_per_seq = max_blocks_per_seq;
  a.kv_lens = kv_lens;
  a.kv_cap = kv_cap;
  a.lay = lay;
  a.ex = ex;
  a.cuts = reinterpret_cast<int4*>(ws);
  a.spans = reinterpret_cast<int4*>(ws);
  a.cut_o = reinterpret_cast<float*>(ws + plan.off_cut_o);
  a.cut_l = reinterpret_cast<float*>(ws + plan.off_cut_l);
  a.full_o = reinterpret_cast<float*>(ws + plan.off_full_o);
  a.full_l = reinterpret_cast<float*>(ws + plan.off_full_l);
  a.err = err;
#define FVB_KEYS(T, D)                                                                             \
  (mode == kKeysWindow ? dispatch<T, D, kKeysWindow>(a, k_pool, v_pool, plan.grid, dependent, stream) \
                       : dispatch<T, D, kKeysRest>(a, k_pool, v_pool, plan.grid, dependent, stream))
  if (dtype == FVB_DTYPE_BF16) return head_dim == 128 ? FVB_KEYS(__nv_bfloat16, 128) : FVB_KEYS(__nv_bfloat16, 64);
  return head_dim == 128 ? FVB_KEYS(__half, 128) : FVB_KEYS(__half, 64);
#undef FVB_KEYS
}

}  // namespace fvb
