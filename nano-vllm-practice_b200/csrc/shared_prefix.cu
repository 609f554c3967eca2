// Decode paged attention for a batch whose sequences share long prefixes by groups.
//
// The reference's prefix cache lets requests share the pages of a common prompt, and its
// decode kernel reads those pages once per request and query head
// (csrc/paged_attention/paged_attention_gemv.cu:16-221).  softmax(q K^T) V splits over the
// keys: with (o_i, lse_i) of disjoint key ranges i, o = sum_i 2^(lse_i - m) o_i / sum_i
// 2^(lse_i - m), m = max lse_i.  Here the prefix of a group is one range (or a few) that
// all its sequences attend together, so its K and V leave HBM once per group and feed
// 128-row tensor-core tiles of (sequence, query head) rows; the keys behind it are attended
// per sequence, bound by HBM.  Calls that are too small for that share nothing (plan_shared_prefix says where).  Else,
// for 16-bit types and up to kKeysMaxSeqs sequences, three launches:
//
//   prefix   prefill_tc.cuh (kTcPrefix);
//   rest     decode_keys.cu: the sequences' own tiles dealt evenly to one CTA per SM, as the
//            prefix's CTAs leave them (programmatic dependent launch), or with one group to
//            the SMs that the prefix kernel does not take, beside which it then runs;
//   merge    one or four warps per (sequence, query head).
//
// Measured: 32 requests behind 4096 tokens, 32/8 heads x 128, own keys U[64, 1024]: 33 us (86 MB: 2.6 TB/s; every
// sequence reading all its keys 116); 128 sequences in four groups behind 2048 to 12288 tokens 109 us (0.41 GB: 3.8
// TB/s; 529).  Of the 109: prefixes 43, bound by the softmax of 128-row tiles and two operands of P, rest 58 at HBM's
// rate, merge 5.
//
// fp32 and larger batches, four launches:
//
//   plan     one CTA: cuts the sequences' own pages into about target_items ranges of equal
//            length, whatever their lengths are (a grid of max_splits x sequences would be
//            mostly empty CTAs here, since the longest context bounds what every sequence
//            may hold behind its prefix);
//   prefix   fp32: decode_split.cuh (kDecodePrefix), else as above;
//   rest     decode_split.cuh (kDecodeRest), one CTA per (range, kv head);
//   merge    as above.
#include <climits>

#include "decode_split.cuh"

namespace fvb {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMinRangePages = 4;

// Sum over the CTA of v (every thread gets it) and the exclusive prefix of the thread's v.
__device__ __forceinline__ int2 block_scan(int v, int* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) sh[warp] = upto;
  __syncthreads();
  int w = sh[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  const int total = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  __syncthreads();
  return make_int2(total, before + upto - v);
}

// items[i] = {sequence, first page, pages, 0} ({-1, ..} behind the last one) and
// spans[b] = {prefix partials, first item, items, 0} of sequence b.
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const int32_t* __restrict__ kv_lens, int kv_cap,
                                                                   int num_seqs, int keys_per_split, int target_items,
                                                                   int max_items, const DecodeExtra ex,
                                                                   int4* __restrict__ items, int4* __restrict__ spans,
                                                                   int* __restrict__ err) {
  __shared__ int sh[32];
  launch_dependents();
  // {pages of sequence b's own keys, keys of its shared prefix}
  auto own_pages = [&](int b) {
    int kv = __ldg(kv_lens + b);
    if (kv > kv_cap) record_error(err, FVB_ERR_INVALID_ARGUMENT, b);
    kv = min(max(kv, 0), kv_cap);
    int lo = 0, hi = ex.num_groups;  // first group whose end lies behind b
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(ex.cu_groups + mid + 1) > b) hi = mid; else lo = mid + 1;
    }
    int prefix = 0;
    if (keys_per_split > 0 && lo < ex.num_groups) {
      const int2 rows = group_rows(ex, lo, num_seqs);
      if (b >= rows.x) prefix = group_prefix(ex, lo, rows);
    }
    return make_int2(max((kv + kPageSize - 1) / kPageSize - prefix / kPageSize, 0), prefix);
  };
  for (int g = threadIdx.x; g < ex.num_groups; g += kPlanThreads) {
    const int lo = __ldg(ex.cu_groups + g), hi = __ldg(ex.cu_groups + g + 1);
    if (lo < 0 || hi < lo || hi > num_seqs || __ldg(ex.prefix_lens + g) < 0)
      record_error(err, FVB_ERR_INVALID_ARGUMENT, g);
  }
  int2 mine = make_int2(0, 0);
  int sum = 0;
  for (int b = threadIdx.x; b < num_seqs; b += kPlanThreads) {
    mine = own_pages(b);
    sum += mine.x;
  }
  const int total = block_scan(sum, sh).x;
  // Whole stages of two pages; sum over b of ceil(pages_b / per) <= target_items + num_seqs.
  int per = max(kMinRangePages, (total + target_items - 1) / target_items);
  per += per & 1;
  int done = 0;
  for (int base = 0; base < num_seqs; base += kPlanThreads) {
    const int b = base + threadIdx.x;
    if (b < num_seqs && num_seqs > kPlanThreads) mine = own_pages(b);
    const int n = b < num_seqs ? (mine.x + per - 1) / per : 0;
    const int2 at = block_scan(n, sh);
    const int first = done + at.y;
    if (b < num_seqs) {
      const int skip = mine.y / kPageSize;
      for (int i = 0; i < n && first + i < max_items; ++i)
        items[first + i] = make_int4(b, skip + i * per, min(per, mine.x - i * per), 0);
      spans[b] = make_int4(keys_per_split > 0 ? (mine.y + keys_per_split - 1) / keys_per_split : 0, first, n, 0);
    }
    done += at.x;
  }
  for (int i = done + threadIdx.x; i < max_items; i += kPlanThreads) items[i] = make_int4(-1, 0, 0, 0);
}

// out[h][b] from the partials of its prefix and of its own keys; WARPS warps per row, whose
// lanes hold D / 32 dims each and take every WARPS-th partial, kInFlight at a time.
constexpr int kMergeThreads = 128;
constexpr int kInFlight = 4;

// Where a row's partials are.  KEYS: decode_keys.cu's (whole units by row, cut ones by CTA); else the ranges'.
struct MergeArgs {
  const float *po, *pl;  // prefix: [row][prefix_slots]
  const float *ro, *rl;  // ranges: [range][head]
  const int4* spans;
  const float *full_o, *full_l, *cut_o, *cut_l;
  int num_seqs, n_heads, prefix_slots, keys_per_split, group, units, grid;
};

template <typename T, int D, int WARPS, bool KEYS>
__global__ void __launch_bounds__(kMergeThreads) shared_merge_kernel(const MergeArgs a, T* __restrict__ out,
                                                                     const QOLayout lay) {
  constexpr int kDims = D / 32;
  constexpr int kRows = kMergeThreads / 32 / WARPS;
  __shared__ float sh_acc[WARPS > 1 ? WARPS : 1][WARPS > 1 ? D : 1];
  __shared__ float sh_m[WARPS], sh_l[WARPS];
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * kRows + (WARPS > 1 ? 0 : warp);  // (sequence, head), head fastest
  if (row >= int64_t(a.num_seqs) * a.n_heads) return;
  const int b = int(row / a.n_heads), head = int(row % a.n_heads);
  const int4 span = __ldcg(a.spans + b);
  // prefix partials, then those of the sequence's own keys: own_n of them from own_0 on
  int np = span.x, own_0 = span.y, own_n = span.z;
  bool whole = false;
  int column = 0;
  if constexpr (KEYS) {
    np = a.keys_per_split > 0 ? (span.x + a.keys_per_split - 1) / a.keys_per_split : 0;
    const int in_group = head % a.group, chunks = (a.group + kKeysCols - 1) / kKeysCols;
    const int unit = head / a.group * chunks + in_group / kKeysCols;
    column = in_group % kKeysCols;
    own_n = 0;
    if (span.y > 0) {
      const int64_t total = int64_t(span.w) * a.units, begin = int64_t(span.z) * a.units + int64_t(unit) * span.y;
      const int grid = int(min(int64_t(a.grid), total));
      own_0 = keys_cta_of(begin, total, grid);
      own_n = keys_cta_of(begin + span.y - 1, total, grid) - own_0 + 1;
      whole = own_n == 1;
    }
  }
  const int n = np + own_n, w = WARPS > 1 ? warp : 0;
  float m = -INFINITY, l = 0.f, acc[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) acc[d] = 0.f;
  for (int i0 = w; i0 < n; i0 += WARPS * kInFlight) {
    float o[kInFlight][kDims], ls[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int i = i0 + u * WARPS;
      const bool prefix = i < np;
      const int k = own_0 + i - np;
      int64_t at = prefix ? row * a.prefix_slots + i : int64_t(k) * a.n_heads + head;
      const float *po = prefix ? a.po : a.ro, *pl = prefix ? a.pl : a.rl;
      if (KEYS && !prefix) {
        at = whole ? row : (int64_t(k) * 2 + (k == own_0 ? 1 : 0)) * kKeysCols + column;
        po = whole ? a.full_o : a.cut_o;
        pl = whole ? a.full_l : a.cut_l;
      }
      ls[u] = i < n ? __ldcg(pl + at) : -INFINITY;
#pragma unroll
      for (int d = 0; d < kDims; ++d) o[u][d] = 0.f;
      if (i < n) {
        const float* src = po + at * D + lane * kDims;
        if constexpr (kDims == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          o[u][0] = v.x, o[u][1] = v.y, o[u][2] = v.z, o[u][3] = v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          o[u][0] = v.x, o[u][1] = v.y;
        }
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      mn = fmaxf(mn, ls[u]);
      if (ls[u] != ls[u]) l = ls[u];  // a NaN among the scores: one in the row
    }
    if (mn == -INFINITY) continue;  // no key seen so far
    const float corr = fast_exp2(m - mn);
    l *= corr;
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] *= corr;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (ls[u] == -INFINITY) continue;  // its O is not a number
      const float wt = fast_exp2(ls[u] - mn);
      l += wt;
#pragma unroll
      for (int d = 0; d < kDims; ++d) acc[d] = fmaf(wt, o[u][d], acc[d]);
    }
    m = mn;
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int d = 0; d < kDims; ++d) sh_acc[warp][lane * kDims + d] = acc[d];
    if (lane == 0) {
      sh_m[warp] = m;
      sh_l[warp] = l;
    }
    __syncthreads();
    if (warp != 0) return;
    float mx = m;
#pragma unroll
    for (int k = 1; k < WARPS; ++k) mx = fmaxf(mx, sh_m[k]);
    const float ms = mx == -INFINITY ? 0.f : mx;
    const float own = fast_exp2(m - ms);
    l *= own;
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] *= own;
#pragma unroll
    for (int k = 1; k < WARPS; ++k) {
      const float wt = fast_exp2(sh_m[k] - ms);
      l = fmaf(sh_l[k], wt, l);
#pragma unroll
      for (int d = 0; d < kDims; ++d) acc[d] = fmaf(wt, sh_acc[k][lane * kDims + d], acc[d]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // an empty context gives zeros
  T* dst = out + int64_t(b) * lay.o_ts + int64_t(head) * lay.o_hs + lane * kDims;
  __align__(16) T v[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) v[d] = Elem<T>::from_f(acc[d] * inv);
  if constexpr (sizeof(v) == 16) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
  } else if constexpr (sizeof(v) == 8) {
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
  } else {
    *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(v);
  }
}

struct SharedArgs {
  const void *q, *k_pool, *v_pool;
  void* out;
  int64_t num_blocks;
  int n_heads, n_kv_heads, num_seqs;
  const int32_t* block_tables;
  int max_blocks_per_seq;
  const int32_t* kv_lens;
  int kv_cap;
  SharedPrefixPlan plan;
  QOLayout lay;
  float *po, *pl, *ro, *rl;
  void* ws;
  DecodeExtra ex;
  int* err;
  cudaStream_t stream;
};

cudaLaunchConfig_t config(dim3 grid, int threads, int smem, cudaStream_t stream, cudaLaunchAttribute* dependent) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  if (dependent) {
    dependent->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = dependent;
    cfg.numAttrs = 1;
  }
  return cfg;
}

template <typename T, int D, int NREP, int MODE>
cudaError_t launch_split(const SharedArgs& a, dim3 grid, int pages_per_split, int splits, float* ws_o, float* ws_lse,
                         bool dependent) {
  using Tr = DecodeTraits<T, D, NREP>;
  const int group = a.n_heads / a.n_kv_heads, chunks = (group + NREP - 1) / NREP;
  CUtensorMap kmap;
  cudaError_t ce = make_k_map<T, D>(&kmap, a.k_pool, a.num_blocks, a.n_kv_heads);
  if (ce == cudaSuccess) ce = set_smem_once<decode_split_kernel<T, D, NREP, MODE>>(Tr::kSmemBytes);
  if (ce != cudaSuccess) return ce;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg =
      config(grid, kDecodeThreads, Tr::kSmemBytes, a.stream, dependent ? attr : nullptr);
  return cudaLaunchKernelEx(&cfg, decode_split_kernel<T, D, NREP, MODE>, kmap, static_cast<const T*>(a.q),
                            static_cast<T*>(a.out), static_cast<const uint8_t*>(a.v_pool), a.num_blocks, a.n_kv_heads,
                            a.num_seqs, a.block_tables, a.max_blocks_per_seq, a.kv_lens, a.kv_cap, pages_per_split,
                            splits, ws_o, ws_lse, a.lay, group, chunks, static_cast<const int32_t*>(nullptr),
                            static_cast<const int32_t*>(nullptr), a.ex, a.err);
}

template <typename T, int D, int NREP>
cudaError_t launch_rest(const SharedArgs& a) {
  const int chunks = (a.n_heads / a.n_kv_heads + NREP - 1) / NREP;
  // A dependent of the prefix kernel, which starts behind the plan; without one an ordinary launch.
  return launch_split<T, D, NREP, kDecodeRest>(a, dim3(a.plan.max_items, a.n_kv_heads * chunks), 0, 1, a.ro, a.rl,
                                               a.plan.keys_per_split > 0);
}

template <typename T, int D, int WARPS, bool KEYS>
cudaError_t launch_merge(const SharedArgs& a, const MergeArgs& m) {
  constexpr int kRows = kMergeThreads / 32 / WARPS;
  const int64_t ctas = (int64_t(a.num_seqs) * a.n_heads + kRows - 1) / kRows;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(dim3(unsigned(ctas)), kMergeThreads, 0, a.stream, attr);
  return cudaLaunchKernelEx(&cfg, shared_merge_kernel<T, D, WARPS, KEYS>, m, static_cast<T*>(a.out), a.lay);
}

template <typename T, int D>
cudaError_t run(const SharedArgs& a, const MergeArgs& m, int head_dim, int dtype) {
  const int group = a.n_heads / a.n_kv_heads;
  cudaError_t ce = cudaSuccess;
  if (!a.plan.keys) {
    shared_plan_kernel<<<1, kPlanThreads, 0, a.stream>>>(
        a.kv_lens, a.kv_cap, a.num_seqs, a.plan.keys_per_split, a.plan.target_items, a.plan.max_items, a.ex,
        const_cast<int4*>(a.ex.items), const_cast<int4*>(m.spans), a.err);
    ce = cudaGetLastError();
    if (ce != cudaSuccess) return ce;
  }
  if (a.plan.keys_per_split > 0) {
    if constexpr (sizeof(T) == 4) {
      // Rows are (sequence, head) pairs of a group, eight a CTA.
      const int64_t row_chunks = (int64_t(a.num_seqs) * group + 7) / 8;
      if (row_chunks * a.plan.prefix_splits > 0x7fffffff) return cudaErrorInvalidValue;
      ce = launch_split<T, D, 8, kDecodePrefix>(
          a, dim3(unsigned(row_chunks * a.plan.prefix_splits), a.n_kv_heads, a.ex.num_groups),
          a.plan.keys_per_split / kPageSize, a.plan.prefix_splits, a.po, a.pl, false);
    } else {
      ce = launch_prefix_tc(a.q, a.k_pool, a.v_pool, a.num_blocks, a.n_heads, a.n_kv_heads, head_dim, a.num_seqs,
                            a.block_tables, a.max_blocks_per_seq, a.kv_lens, dtype, a.plan, a.lay, a.po, a.pl, a.ex,
                            a.err, a.stream);
    }
    if (ce != cudaSuccess) return ce;
  }
  if (a.plan.keys) {
    ce = launch_keys_decode(a.q, a.out, a.k_pool, a.v_pool, a.num_blocks, a.n_heads, a.n_kv_heads, head_dim,
                            a.num_seqs, a.block_tables, a.max_blocks_per_seq, a.kv_lens, a.kv_cap, a.ex, kKeysRest,
                            dtype, a.plan.kp, a.lay, a.ws, a.plan.keys_per_split > 0, a.err, a.stream);
  } else {
    switch (decode_tile_heads(group)) {
      case 1:
        ce = launch_rest<T, D, 1>(a);
        break;
      case 2:
        ce = launch_rest<T, D, 2>(a);
        break;
      case 4:
        ce = launch_rest<T, D, 4>(a);
        break;
      default:
        ce = launch_rest<T, D, 8>(a);
    }
  }
  if (ce != cudaSuccess) return ce;
  // Partials a row merges on average: prefix splits and its share of the ranges (of the CTAs).
  const int64_t own = a.plan.keys ? int64_t(a.plan.kp.grid) / (int64_t(a.num_seqs) * m.units) + 1
                                  : a.plan.max_items / a.num_seqs;
  const bool many = a.plan.prefix_splits + own > 8;
  if (a.plan.keys) ce = many ? launch_merge<T, D, 4, true>(a, m) : launch_merge<T, D, 1, true>(a, m);
  else ce = many ? launch_merge<T, D, 4, false>(a, m) : launch_merge<T, D, 1, false>(a, m);
  return ce != cudaSuccess ? ce : cudaGetLastError();
}

}  // namespace

SharedPrefixPlan plan_shared_prefix(int num_seqs, int n_heads, int n_kv_heads, int head_dim, int max_kv_len,
                                    int num_groups, int max_prefix_len, int dtype, int num_sms) {
  SharedPrefixPlan p{};
  if (num_seqs <= 0 || n_kv_heads <= 0) return p;
  const int group = n_heads / n_kv_heads;
  const int prefix = std::max(0, std::min(max_prefix_len, max_kv_len)) / kPageSize * kPageSize;
  // Sharing takes three launches (fp32 four) that follow on one another, 10 to 14 us (17) however little there is to
  // read.  Where an SM has few pages to read, each sequence reading its own, out of L2 for all but one of a group, is
  // one launch of 4 to 10 us.  Which is faster goes by the pages an SM gets at most (halves of D 128 count each), and
  // by what a page costs the split-KV kernel: over 400 calls of random shapes the choice is 1 % off the better way on
  // average, and sharing always 40 %.  (70 sequences x 2 heads x 128 behind up to 182 keys, group 3: 18.0 us shared,
  // 9.9 each for itself; 8 x 8 x 128 behind 2000, group 2: 14.9 and 20.3; 32 x 8 x 128 behind 4096, group 4: 33.0 and
  // 116.)
  const int64_t pages = std::max<int64_t>(1, (int64_t(max_kv_len) + kPageSize - 1) / kPageSize) * (head_dim / 64);
  const int64_t direct_pages = dtype == FVB_DTYPE_F32 ? (group <= 8 ? 128 : 64)
                               : group <= 1           ? 256
                               : group <= 2           ? 96
                               : group <= 4           ? 64
                               : group <= 8           ? 28
                                                      : 22;
  if (int64_t(num_seqs) * n_kv_heads * pages <= direct_pages * num_sms) {
    p.direct = true;
    p.dp = plan_window_decode(num_seqs, n_heads, n_kv_heads, head_dim, max_kv_len, INT_MAX, 0, num_sms);
    p.ws_bytes = p.dp.ws_bytes;
    return p;
  }
  p.keys = dtype != FVB_DTYPE_F32 && num_seqs <= kKeysMaxSeqs;
  int taken = 0;  // SMs that the prefix kernel holds
  if (prefix > 0 && num_groups > 0) {
    // A group's rows are cut into tensor-core tiles (fp32: chunks of eight rows), its prefix into splits until
    // the CTAs fill the SMs that are the prefixes' share.  Groups of the average size that fit one query tile
    // take items of one tile, whose two softmax groups share it.
    const bool tc = dtype != FVB_DTYPE_F32;
    const int unit = tc ? 128 : kPageSize * 4;
    const int tile = tc ? 128 / tc_tile_heads(group) : 1;  // sequences of a query tile
    const int average = (num_seqs + num_groups - 1) / num_groups;
    p.single_tiles = tc && average <= tile;
    const int item = tile * (p.single_tiles ? 1 : 2);
    const int64_t per_group = tc ? (average + item - 1) / item : (int64_t(average) * group + 7) / 8;
    const int heads = tc ? n_kv_heads * ((group + tc_tile_heads(group) - 1) / tc_tile_heads(group)) : n_kv_heads;
    const int64_t ctas = std::max<int64_t>(1, per_group * num_groups * heads);
    const int units = (prefix + unit - 1) / unit;
    int64_t room = tc ? num_sms : num_sms * 6;
    if (p.keys && num_groups == 1) {
      // Both kernels hold an SM's shared memory alone, so they share the SMs out: a prefix tile (twice the work
      // in items of two) takes about 1.5 us of an SM from L2, a tile of the sequences' own keys 1.64 us from
      // HBM.  The contexts behind the prefix are taken for half of what max_kv_len leaves.  With one operand for P:
      // 8 beams 17.2 us one kernel after the other on all SMs, 12.7 beside each other; 32 requests behind 4096
      // tokens 39.6, 32.2; with two operands 14.9 and 33.0 beside each other (the same at 1.65 and 2.9 us a tile; with
      // a max_kv_len ten times too large 22.3 and 35.3).  With several groups the number of prefix CTAs is not known
      // here, and a CTA too many holds up a whole share of the rest (128 sequences in 4 groups, one operand: 100 us
      // after each other, 113 beside).
      const int own = std::max(0, max_kv_len - prefix) / 2;
      const double first = double(ctas) * units * (p.single_tiles ? 1.45 : 2.5);
      const double rest = double(num_seqs) * n_kv_heads * ((group + kKeysCols - 1) / kKeysCols) *
                          ((own + kKeysTile - 1) / kKeysTile) * 1.64;
      const int64_t share = int64_t(num_sms * first / (first + rest));
      room = std::max<int64_t>(num_sms / 8, std::min<int64_t>(num_sms * 7 / 8, share));
    }
    const int64_t wanted = std::min<int64_t>(std::max<int64_t>(1, room / ctas), units);
    const int per = int((units + wanted - 1) / wanted);
    p.keys_per_split = per * unit;
    p.prefix_splits = (prefix + p.keys_per_split - 1) / p.keys_per_split;
    if (num_groups == 1) taken = int(std::min<int64_t>(num_sms * 7 / 8, ctas * p.prefix_splits));
  }
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  const size_t rows = size_t(num_seqs) * n_heads * p.prefix_splits;
  if (p.keys) {
    p.kp = plan_keys(num_seqs, n_heads, head_dim, kKeysRest, num_sms - taken);
    p.off_po = up(p.kp.ws_bytes);
  } else {
    // About four waves of three resident split-KV CTAs per SM, as plan_decode.
    const int tile_heads = decode_tile_heads(group);
    const int units = n_kv_heads * ((group + tile_heads - 1) / tile_heads);
    p.target_items = std::max(1, (num_sms * 12 + units - 1) / units);
    p.max_items = p.target_items + num_seqs;
    const size_t rest = size_t(p.max_items) * n_heads;
    p.off_spans = up(size_t(p.max_items) * 16);
    p.off_ro = p.off_spans + up(size_t(num_seqs) * 16);
    p.off_rl = p.off_ro + up(rest * head_dim * 4);
    p.off_po = p.off_rl + up(rest * 4);
  }
  p.off_pl = p.off_po + up(rows * head_dim * 4);
  p.ws_bytes = p.off_pl + up(rows * 4);
  return p;
}

cudaError_t launch_shared_prefix(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                                 int n_heads, int n_kv_heads, int head_dim, int num_seqs, const int32_t* block_tables,
                                 int max_blocks_per_seq, const int32_t* kv_lens, int max_kv_len,
                                 const int32_t* cu_groups, int num_groups, const int32_t* prefix_lens,
                                 int max_prefix_len, int dtype, const SharedPrefixPlan& plan, const QOLayout& lay,
                                 void* workspace, int* err, cudaStream_t stream) {
  if (num_seqs == 0) return cudaSuccess;
  if (plan.direct) {
    DecodeExtra ex;
    ex.cu_groups = cu_groups;
    ex.prefix_lens = prefix_lens;
    ex.num_groups = num_groups;
    return launch_window_decode(q, out, k_pool, v_pool, num_blocks, n_heads, n_kv_heads, head_dim, num_seqs,
                                block_tables, max_blocks_per_seq, kv_lens, max_kv_len, INT_MAX, 0, dtype, plan.dp, lay,
                                workspace, err, stream, nullptr, nullptr, ex);
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SharedArgs a{};
  a.q = q;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.out = out;
  a.num_blocks = num_blocks;
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.num_seqs = num_seqs;
  a.block_tables = block_tables;
  a.max_blocks_per_seq = max_blocks_per_seq;
  a.kv_lens = kv_lens;
  a.kv_cap = int(std::min<int64_t>(max_kv_len, int64_t(max_blocks_per_seq) * kPageSize));
  a.plan = plan;
  a.lay = lay;
  a.po = reinterpret_cast<float*>(ws + plan.off_po);
  a.pl = reinterpret_cast<float*>(ws + plan.off_pl);
  a.ro = reinterpret_cast<float*>(ws + plan.off_ro);
  a.rl = reinterpret_cast<float*>(ws + plan.off_rl);
  a.ws = ws;
  a.ex.cu_groups = cu_groups;
  a.ex.prefix_lens = prefix_lens;
  a.ex.num_groups = num_groups;
  a.ex.prefix_cap = std::min(max_prefix_len, a.kv_cap);
  a.ex.slots = plan.prefix_splits;
  a.ex.items = reinterpret_cast<const int4*>(ws);
  a.err = err;
  a.stream = stream;
  MergeArgs m{};
  m.po = a.po;
  m.pl = a.pl;
  m.ro = a.ro;
  m.rl = a.rl;
  m.spans = reinterpret_cast<const int4*>(ws + plan.off_spans);  // (keys: at 0)
  m.num_seqs = num_seqs;
  m.n_heads = n_heads;
  m.prefix_slots = plan.prefix_splits;
  m.keys_per_split = plan.keys_per_split;
  m.group = n_heads / n_kv_heads;
  if (plan.keys) {
    m.full_o = reinterpret_cast<const float*>(ws + plan.kp.off_full_o);
    m.full_l = reinterpret_cast<const float*>(ws + plan.kp.off_full_l);
    m.cut_o = reinterpret_cast<const float*>(ws + plan.kp.off_cut_o);
    m.cut_l = reinterpret_cast<const float*>(ws + plan.kp.off_cut_l);
    m.units = n_kv_heads * ((m.group + kKeysCols - 1) / kKeysCols);
    m.grid = plan.kp.grid;
  }
  if (dtype == FVB_DTYPE_BF16)
    return head_dim == 128 ? run<__nv_bfloat16, 128>(a, m, head_dim, dtype)
                           : run<__nv_bfloat16, 64>(a, m, head_dim, dtype);
  if (dtype == FVB_DTYPE_F16)
    return head_dim == 128 ? run<__half, 128>(a, m, head_dim, dtype) : run<__half, 64>(a, m, head_dim, dtype);
  return head_dim == 128 ? run<float, 128>(a, m, head_dim, dtype) : run<float, 64>(a, m, head_dim, dtype);
}

}  // namespace fvb
