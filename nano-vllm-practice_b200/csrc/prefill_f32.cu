// Chunked-prefill paged attention with a sliding window and sinks for fp32 operands.
//
// fp32 results have to hold fp32's accuracy, which the tensor cores' inputs do not, so the
// products run on the FMA pipe (128 a clock and SM: 72 TFLOP/s), tiled for it:
//
//   tile   64 (small calls 32) consecutive rows of one sequence and kv head (row = token x GQA
//          head, so a key that is fetched serves the whole group) against 64 keys at a time,
//          four rows a thread.
//   S      each thread 4 rows x 4 keys, 8 16-byte shared loads for 64 FMAs (32 paired ones);
//          the rows of a half-warp are its own, so the row maximum is four shuffles.
//   P V    the same 4 rows x D/16 dims, P through the warp's own 8 rows of shared memory:
//          O, m and l never leave their registers.
//   loads  K of the next tile is copied (cp.async) while this tile's softmax and PV run, V
//          while its S does; page ids are read a tile ahead.  Two CTAs per SM (three at D 64)
//          fill the barriers' gaps.
//   rows   a tile of at most 16 rows (a single token's group, the end of a chunk) takes the
//          same code with 1 or 2 rows a thread.
//   keys   only the pages that the tile's rows can see: the sinks' and the window's; keys of
//          them that no row sees are stored as zeros and masked.
//   split  with fewer tiles than the SMs hold, a cluster of 2 to 8 CTAs shares a tile's keys
//          and joins (m, l, O) through distributed shared memory.
//
// Bound by the shared-memory loads (74 % of their pipe; paired FMAs take 32 % of theirs): 7 chunks of 761 to 1019
// tokens, 32/8 heads x 128, window 1059 (37 GFLOP) 1.21 ms = 31 TFLOP/s; one warp a query row, as the causal fp32
// kernel has it, 38 ms.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "kernels.h"

namespace fvb {
namespace {

namespace cg = cooperative_groups;

// Threads of a tile of ROWS rows: four rows each.  (Two rows each in tiles of 32, 256 threads: 42.5 us where these
// take 34.6, from the shared-memory loads, and 12.3 where these take 14.2 in calls of one tile an SM and one of keys;
// eight each in tiles of 64, 128 threads: the largest call 5 % faster, the others up to 15 % slower.)
template <int ROWS>
constexpr int kThreadsOf = ROWS * 4;
constexpr int kKeys = 64;   // keys of a tile, four pages
constexpr int kPagesPerTile = kKeys / kPageSize;
constexpr int kFewRows = 16;
constexpr int kMaxSplits = 8;  // portable cluster size
constexpr float kLog2e = 1.4426950408889634f;

struct F32Args {
  const float *q, *k_pool, *v_pool;
  float* out;
  int64_t num_blocks, q_len_flatten;
  int n_kv_heads, group, num_seqs, max_blocks_per_seq, window, sinks;
  const int32_t *cu_seqlens, *block_tables, *kv_lens, *positions;
  QOLayout lay;
  int* err;
};

// ROWS: query rows of a tile, 64 or 32.
template <int D, int ROWS>
struct Smem {
  static constexpr int kQ = 0;                          // [ROWS][D], 16-byte chunk c of row r at c ^ (r & 1)
  static constexpr int kK = kQ + ROWS * D;              // [64][D], at c ^ (r & 7); at the end the split's O
  static constexpr int kV = kK + kKeys * D;             // [64][D]
  static constexpr int kP = kV + kKeys * D;             // [ROWS][64], at c ^ 4 (r & 1)
  static constexpr int kStats = kP + ROWS * kKeys;      // (m, l) of the split's rows
  static constexpr int kMeta = kStats + 2 * ROWS;       // sequence, first row, rows, earliest and latest position
  static constexpr int kFloats = kMeta + 16;
  static constexpr int kBytes = kFloats * 4;
};

__device__ __forceinline__ void copy16(float* dst, const float* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_copies_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// The tile of one CTA, R rows a thread: ROWS / 16, or 1 for at most kFewRows rows.
template <int D, int ROWS, int R>
__device__ __forceinline__ void attend_tile(const F32Args& a, float* sm, int seq, int kvh, int64_t tok0, int row0,
                                            int n_rows, int kv_len, const KeySpan span, int split, int splits) {
  constexpr int kChunks = D / 4;    // 16-byte chunks of a row
  constexpr int kVC = D / 64;       // chunks of V (and O) a thread holds
  constexpr int kThreads = kThreadsOf<ROWS>;
  using S = Smem<D, ROWS>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, col = lane & 15;
  const int my_row = warp * 2 * R + half;  // its rows: my_row + 2 i
  const int32_t* table = a.block_tables + int64_t(seq) * a.max_blocks_per_seq;

  int pos[R];  // -1: no row, sees nothing
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = my_row + 2 * i;
    pos[i] = row < n_rows ? __ldg(a.positions + tok0 + (row0 + row) / a.group) : -1;
  }
  const float scale = kLog2e * rsqrtf(float(D));
  for (int x = threadIdx.x; x < kThreads / 16 * R * kChunks; x += kThreads) {
    const int row = x / kChunks, c = x % kChunks;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < n_rows) {
      const int64_t tok = tok0 + (row0 + row) / a.group;
      const int head = kvh * a.group + (row0 + row) % a.group;
      v = __ldg(reinterpret_cast<const float4*>(a.q + tok * a.lay.q_ts + int64_t(head) * a.lay.q_hs) + c);
    }
    v = make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
    *reinterpret_cast<float4*>(sm + S::kQ + row * D + ((c ^ (row & 1)) << 2)) = v;
  }

  const int n_tiles = (span.count + kPagesPerTile - 1) / kPagesPerTile;
  const int t_begin = int(int64_t(n_tiles) * split / splits), t_end = int(int64_t(n_tiles) * (split + 1) / splits);
  auto page_of = [&](int c) { return c < span.head ? c : c + span.gap; };
  // Copies: thread t takes chunk t % kChunks of the keys t / kChunks + i * kRowStep.
  constexpr int kRowStep = kThreads / kChunks;
  const int ld_c = threadIdx.x % kChunks, ld_r = threadIdx.x / kChunks;
  const int64_t head_off = int64_t(kvh) * kPageSize * D, page_step = int64_t(a.n_kv_heads) * kPageSize * D;
  int next_id[kPagesPerTile];  // page ids one tile ahead
  auto read_ids = [&](int t) {
#pragma unroll
    for (int p = 0; p < kPagesPerTile; ++p) {
      const int c = t * kPagesPerTile + p;
      next_id[p] = t < t_end && c < span.count ? max(__ldg(table + page_of(c)), -1) : -2;  // -2: no page
    }
  };
  auto check_ids = [&](int* id) {
#pragma unroll
    for (int p = 0; p < kPagesPerTile; ++p) {
      id[p] = next_id[p];
      if (id[p] != -2 && (id[p] < 0 || id[p] >= a.num_blocks)) {
        record_error(a.err, FVB_ERR_BAD_PAGE, seq);
        id[p] = 0;
      }
    }
  };
  // A key that no row of the tile sees becomes zeros (its slot may never have been written).
  auto copy_tile = [&](const float* pool, float* dst, const int* id, int t, bool swizzle) {
#pragma unroll
    for (int i = 0; i < kKeys / kRowStep; ++i) {
      const int r = ld_r + i * kRowStep;
      const int p = (i * kRowStep) / kPageSize;  // (kRowStep divides a page)
      const int key = page_of(t * kPagesPerTile + p) * kPageSize + r % kPageSize;
      const bool live = id[p] >= 0 && key < kv_len && (key >= span.lo || key < a.sinks);
      const float* src = pool + (live ? int64_t(id[p]) * page_step + head_off + (r % kPageSize) * D + ld_c * 4 : 0);
      copy16(dst + r * D + ((swizzle ? ld_c ^ (r & 7) : ld_c) << 2), src, live);
    }
  };

  float m[R], l[R];
  float2 o[R][2 * kVC];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < 2 * kVC; ++d) o[i][d] = make_float2(0.f, 0.f);
  }
  int id[kPagesPerTile];
  read_ids(t_begin);
  check_ids(id);
  if (t_begin < t_end) copy_tile(a.k_pool, sm + S::kK, id, t_begin, true);
  commit_copies();
  if (t_begin < t_end) copy_tile(a.v_pool, sm + S::kV, id, t_begin, false);
  commit_copies();
  read_ids(t_begin + 1);

  const float* qp = sm + S::kQ + my_row * D;
  const float* kp = sm + S::kK + col * D;
  float* pp = sm + S::kP + my_row * kKeys;
  for (int t = t_begin; t < t_end; ++t) {
    wait_copies_but_one();
    __syncthreads();  // K (and, the first time, Q) is there
    // ---- S: keys col + 16 j ----
    float2 s2[R][4];  // even and odd dims
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int c = 0; c < kChunks; ++c) {
      float4 kv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        kv[j] = *reinterpret_cast<const float4*>(kp + j * 16 * D + ((c ^ (col & 7)) << 2));
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 qv = *reinterpret_cast<const float4*>(qp + 2 * i * D + ((c ^ (my_row & 1)) << 2));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s2[i][j] = __ffma2_rn(make_float2(qv.x, qv.y), make_float2(kv[j].x, kv[j].y), s2[i][j]);
          s2[i][j] = __ffma2_rn(make_float2(qv.z, qv.w), make_float2(kv[j].z, kv[j].w), s2[i][j]);
        }
      }
    }
    float s[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = s2[i][j].x + s2[i][j].y;
    __syncthreads();  // K is read
    check_ids(id);
    if (t + 1 < t_end) copy_tile(a.k_pool, sm + S::kK, id, t + 1, true);
    commit_copies();
    read_ids(t + 2);
    // ---- mask and softmax ----
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = t * kPagesPerTile + j;
      const int key = c < span.count ? page_of(c) * kPageSize + col : INT_MAX;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const bool seen = key <= pos[i] && key < kv_len && (pos[i] - key < a.window || key < a.sinks);
        if (!seen) s[i][j] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float top = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float next = fmaxf(m[i], top), ref = next == -INFINITY ? 0.f : next;
      const float f = fast_exp2(m[i] - ref);  // 0 while m is -inf
      m[i] = next;
      l[i] *= f;
#pragma unroll
      for (int d = 0; d < 2 * kVC; ++d) o[i][d] = __fmul2_rn(o[i][d], make_float2(f, f));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = fast_exp2(s[i][j] - ref);
        l[i] += p;
        // chunk (col + 16 j) / 4 of row my_row + 2 i
        pp[2 * i * kKeys + ((((col >> 2) + 4 * j) ^ ((my_row & 1) << 2)) << 2) + (col & 3)] = p;
      }
    }
    wait_copies_but_one();
    __syncthreads();  // V is there (and P, of the warp alone)
    // ---- O += P V: dims 4 col + 64 x ----
#pragma unroll 2
    for (int c = 0; c < kKeys / 4; ++c) {
      float4 pv[R];
#pragma unroll
      for (int i = 0; i < R; ++i)
        pv[i] = *reinterpret_cast<const float4*>(pp + 2 * i * kKeys + ((c ^ ((my_row & 1) << 2)) << 2));
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const float* vr = sm + S::kV + (c * 4 + kk) * D + col * 4;
#pragma unroll
        for (int x = 0; x < kVC; ++x) {
          const float4 vv = *reinterpret_cast<const float4*>(vr + x * 64);
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float p = kk == 0 ? pv[i].x : kk == 1 ? pv[i].y : kk == 2 ? pv[i].z : pv[i].w;
            o[i][2 * x] = __ffma2_rn(make_float2(p, p), make_float2(vv.x, vv.y), o[i][2 * x]);
            o[i][2 * x + 1] = __ffma2_rn(make_float2(p, p), make_float2(vv.z, vv.w), o[i][2 * x + 1]);
          }
        }
      }
    }
    __syncthreads();  // V is read
    if (t + 1 < t_end) copy_tile(a.v_pool, sm + S::kV, id, t + 1, false);
    commit_copies();
  }

  // ---- results: straight to out, or to the split's place in shared memory ----
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    const int row = my_row + 2 * i;
    if (splits > 1) {
#pragma unroll
      for (int x = 0; x < kVC; ++x)
        *reinterpret_cast<float4*>(sm + S::kK + row * D + 4 * col + 64 * x) =
            make_float4(o[i][2 * x].x, o[i][2 * x].y, o[i][2 * x + 1].x, o[i][2 * x + 1].y);
      if (col == 0) *reinterpret_cast<float2*>(sm + S::kStats + 2 * row) = make_float2(m[i], l[i]);
    } else if (row < n_rows) {
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];  // (a NaN stays one)
      const int64_t tok = tok0 + (row0 + row) / a.group;
      const int head = kvh * a.group + (row0 + row) % a.group;
      float* dst = a.out + tok * a.lay.o_ts + int64_t(head) * a.lay.o_hs;
#pragma unroll
      for (int x = 0; x < kVC; ++x)
        *reinterpret_cast<float4*>(dst + 4 * col + 64 * x) = make_float4(
            o[i][2 * x].x * inv, o[i][2 * x].y * inv, o[i][2 * x + 1].x * inv, o[i][2 * x + 1].y * inv);
    }
  }
}

template <int D, int ROWS>
__global__ void __launch_bounds__(kThreadsOf<ROWS>, D == 128 ? 2 : 3) window_prefill_f32_kernel(const F32Args a) {
  extern __shared__ __align__(16) float sm[];
  constexpr int kThreads = kThreadsOf<ROWS>;
  using S = Smem<D, ROWS>;
  int* meta = reinterpret_cast<int*>(sm + S::kMeta);
  const cg::cluster_group cluster = cg::this_cluster();
  const int splits = int(cluster.num_blocks()), split = int(cluster.block_rank());
  const int64_t unit = blockIdx.x / splits;
  const int kvh = int(unit % a.n_kv_heads);
  const int64_t tile = unit / a.n_kv_heads;
  // ---- the tile's sequence: the tiles of every sequence before it, 32 sequences at a time ----
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int seq = -1, first = 0, rows = 0;
    int64_t before = 0;
    for (int s0 = 0; s0 < a.num_seqs && seq < 0; s0 += 32) {
      const int s = s0 + lane;
      int64_t lo = 0, hi = 0;
      if (s < a.num_seqs) {  // inside [0, q_len_flatten) whatever cu_seqlens holds
        lo = min(max(int64_t(__ldg(a.cu_seqlens + s)), int64_t(0)), a.q_len_flatten);
        hi = min(max(int64_t(__ldg(a.cu_seqlens + s + 1)), lo), a.q_len_flatten);
      }
      const int64_t n = (hi - lo) * a.group;
      const int64_t mine = (n + ROWS - 1) / ROWS;
      int64_t sum = mine;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, sum, x);
        if (lane >= x) sum += y;
      }
      const int64_t begin = before + sum - mine;
      const bool here = tile >= begin && tile < begin + mine;
      const unsigned found = __ballot_sync(0xffffffffu, here);
      if (found != 0) {
        const int src = __ffs(found) - 1;
        const int64_t row = (tile - begin) * ROWS;
        seq = s0 + src;
        // (its place inside the sequence: a row takes 256 bytes or more, so fewer than 2^31 of them fit a device)
        first = __shfl_sync(0xffffffffu, int(row), src);
        rows = __shfl_sync(0xffffffffu, int(min(n - row, int64_t(ROWS))), src);
        if (lane == src) {
          meta[0] = seq;
          meta[1] = int(lo);
        }
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    __syncwarp();
    if (seq < 0) {
      if (lane == 0) meta[0] = -1;
    } else {
      int low = INT_MAX, high = -1;  // earliest and latest position
      const int64_t tok0 = meta[1];
      for (int t = first / a.group + lane; t <= (first + rows - 1) / a.group; t += 32) {
        const int p = __ldg(a.positions + tok0 + t);
        low = min(low, p);
        high = max(high, p);
      }
      low = __reduce_min_sync(0xffffffffu, low);
      high = __reduce_max_sync(0xffffffffu, high);
      if (lane == 0) {
        meta[2] = first;
        meta[3] = rows;
        meta[4] = low;
        meta[5] = high;
      }
    }
  }
  __syncthreads();
  const int seq = meta[0];
  if (seq < 0) return;  // the whole cluster: it has one tile
  const int64_t tok0 = meta[1];
  const int row0 = meta[2], n_rows = meta[3], low = max(meta[4], 0), high = meta[5];
  int kv_len = __ldg(a.kv_lens + seq);
  const int64_t cap = int64_t(a.max_blocks_per_seq) * kPageSize;
  if (kv_len > cap) {
    if (threadIdx.x == 0) record_error(a.err, FVB_ERR_INVALID_ARGUMENT, seq);
    kv_len = int(cap);
  }
  kv_len = max(0, high < kv_len ? high + 1 : kv_len);  // keys that some row sees end here
  const KeySpan span = window_span(low + 1, kv_len, a.window, a.sinks, kPageSize);
  if (n_rows <= kFewRows)
    attend_tile<D, ROWS, kFewRows * 16 / kThreads>(a, sm, seq, kvh, tok0, row0, n_rows, kv_len, span, split, splits);
  else
    attend_tile<D, ROWS, ROWS * 16 / kThreads>(a, sm, seq, kvh, tok0, row0, n_rows, kv_len, span, split, splits);
  if (splits == 1) return;
  // ---- join: CTA r of the cluster takes rows r, r + splits, ... ----
  cluster.sync();
  constexpr int kChunks = D / 4;
  const int c = threadIdx.x % kChunks;
  for (int row = split + splits * int(threadIdx.x / kChunks); row < n_rows; row += splits * (kThreads / kChunks)) {
    float top = -INFINITY;
    float2 st[kMaxSplits];
#pragma unroll
    for (int k = 0; k < kMaxSplits; ++k) {
      st[k] = k < splits ? *reinterpret_cast<const float2*>(cluster.map_shared_rank(sm + S::kStats + 2 * row, k))
                         : make_float2(-INFINITY, 0.f);
      top = fmaxf(top, st[k].x);
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kMaxSplits; ++k) {
      if (k >= splits) continue;
      const float f = fast_exp2(st[k].x - ref);
      const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(sm + S::kK + row * D + 4 * c, k));
      sum = fmaf(f, st[k].y, sum);
      o = make_float4(fmaf(f, x.x, o.x), fmaf(f, x.y, o.y), fmaf(f, x.z, o.z), fmaf(f, x.w, o.w));
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t tok = tok0 + (row0 + row) / a.group;
    const int head = kvh * a.group + (row0 + row) % a.group;
    float* dst = a.out + tok * a.lay.o_ts + int64_t(head) * a.lay.o_hs;
    *reinterpret_cast<float4*>(dst + 4 * c) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

template <int D, int ROWS>
cudaError_t launch_t(const F32Args& a, int64_t tiles, int splits, cudaStream_t stream) {
  using S = Smem<D, ROWS>;
  const cudaError_t ce = set_smem_once<window_prefill_f32_kernel<D, ROWS>>(S::kBytes);
  if (ce != cudaSuccess) return ce;
  const int64_t ctas = tiles * a.n_kv_heads * splits;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kThreadsOf<ROWS>);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, window_prefill_f32_kernel<D, ROWS>, a);
}

}  // namespace

cudaError_t launch_window_prefill_f32(const void* q, void* out, const void* k_pool, const void* v_pool,
                                      int64_t num_blocks, int n_heads, int n_kv_heads, int head_dim, int num_seqs,
                                      int64_t q_len_flatten, int max_q_len, const int32_t* cu_seqlens,
                                      const int32_t* block_tables, int max_blocks_per_seq, const int32_t* kv_lens,
                                      const int32_t* positions, int window, int sinks, const QOLayout& lay, int* err,
                                      cudaStream_t stream) {
  if (q_len_flatten == 0 || num_seqs == 0) return cudaSuccess;
  F32Args a{};
  a.q = static_cast<const float*>(q);
  a.k_pool = static_cast<const float*>(k_pool);
  a.v_pool = static_cast<const float*>(v_pool);
  a.out = static_cast<float*>(out);
  a.num_blocks = num_blocks;
  a.q_len_flatten = q_len_flatten;
  a.n_kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads;
  a.num_seqs = num_seqs;
  a.max_blocks_per_seq = max_blocks_per_seq;
  a.window = window;
  a.sinks = sinks;
  a.cu_seqlens = cu_seqlens;
  a.block_tables = block_tables;
  a.kv_lens = kv_lens;
  a.positions = positions;
  a.lay = lay;
  a.err = err;
  // A sequence's last tile is ragged, so the batch has at most this many.  Tiles of 32 rows where the SMs hold those of
  // 64 at once: what one tile takes is then the call's time (about 2 / 3 of it).
  const int places = device_sm_count() * (head_dim == 128 ? 2 : 3);
  auto tiles_of = [&](int rows) { return q_len_flatten * a.group / rows + num_seqs; };
  const int rows = tiles_of(64) * n_kv_heads > device_sm_count() ? 64 : 32;
  const int64_t tiles = tiles_of(rows);
  // As many CTAs share a tile's keys as leave each two tiles of them and fill the SMs' places once.
  const int64_t kv_cap = std::min<int64_t>(int64_t(max_blocks_per_seq) * kPageSize, 0x7fffffff);
  const int tokens = std::min(max_q_len, (rows + a.group - 2) / a.group + 1);  // of a tile at most
  const int64_t keys = std::min<int64_t>(kv_cap, int64_t(window) + tokens - 1);
  const int key_pages = window_max_units(int(kv_cap), int(std::max<int64_t>(1, keys)), sinks, kPageSize);
  const int key_tiles = key_pages / kPagesPerTile;
  int splits = 1;
  while (splits < kMaxSplits && tiles * n_kv_heads * splits * 2 <= places && key_tiles >= splits * 4) splits *= 2;
  if (rows == 64)
    return head_dim == 128 ? launch_t<128, 64>(a, tiles, splits, stream) : launch_t<64, 64>(a, tiles, splits, stream);
  return head_dim == 128 ? launch_t<128, 32>(a, tiles, splits, stream) : launch_t<64, 32>(a, tiles, splits, stream);
}

}  // namespace fvb
