// Varlen chunked-prefill attention on the tensor cores: the work plan, the plain form of the
// kernel in prefill_tc.cuh (prefill and decode mode) and its dispatch.
#include "prefill_tc.cuh"

namespace fvb {
namespace {

constexpr int kSortMaxSeqs = 2048;

// Work plan of one launch (one CTA):
//  order[p]    = p-th sequence by descending kv_len (identity beyond kSortMaxSeqs
//                sequences), so the longest-context work is dispatched first;
//  cu_items[p] = exclusive scan of ceil(ceil(q_len / tile_tokens) / tiles_per_item)
//                (work items of that many query tiles) over that order; sequences of
//                one query token get none when skip_single is set (the split-KV decode
//                kernel serves them).
__global__ void __launch_bounds__(1024) prefill_plan_kernel(const int32_t* __restrict__ cu_seqlens,
                                                            const int32_t* __restrict__ kv_lens, int num_seqs,
                                                            int tile_tokens, int tiles_per_item,
                                                            int32_t* __restrict__ order,
                                                            int32_t* __restrict__ cu_items, int skip_single) {
  __shared__ int kv_sh[kSortMaxSeqs];
  __shared__ int warp_tot[32];
  __shared__ int carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const bool sort = num_seqs <= kSortMaxSeqs;
  if (sort) {
    for (int t = threadIdx.x; t < num_seqs; t += blockDim.x) kv_sh[t] = __ldg(kv_lens + t);
  }
  if (threadIdx.x == 0) {
    carry = 0;
    cu_items[0] = 0;
  }
  __syncthreads();
  for (int s = threadIdx.x; s < num_seqs; s += blockDim.x) {
    int rank = s;
    if (sort) {
      const int ks = kv_sh[s];
      rank = 0;
      for (int t = 0; t < num_seqs; ++t) {
        const int kt = kv_sh[t];
        rank += (kt > ks) || (kt == ks && t < s);
      }
    }
    order[rank] = s;
  }
  __syncthreads();
  for (int base = 0; base < num_seqs; base += blockDim.x) {
    const int p = base + threadIdx.x;
    int v = 0;
    if (p < num_seqs) {
      const int s = order[p];
      // decode mode (cu_seqlens == nullptr): one query token per sequence
      const int ql = cu_seqlens ? __ldg(cu_seqlens + s + 1) - __ldg(cu_seqlens + s) : 1;
      const int tiles = ql > 0 && !(skip_single && ql == 1) ? (ql + tile_tokens - 1) / tile_tokens : 0;
      v = (tiles + tiles_per_item - 1) / tiles_per_item;
    }
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_tot[warp] = x;
    __syncthreads();
    if (warp == 0) {
      int w = lane < nwarps ? warp_tot[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      warp_tot[lane] = w;
    }
    __syncthreads();
    const int incl = x + (warp > 0 ? warp_tot[warp - 1] : 0) + carry;
    if (p < num_seqs) cu_items[p + 1] = incl;
    __syncthreads();
    if (threadIdx.x == blockDim.x - 1) carry = incl;
    __syncthreads();
  }
}

template <typename T, int D, bool kIlv>
cudaError_t dispatch_tc(int nrep, const void* q, void* out, const void* k_pool, const void* v_pool,
                        int64_t num_blocks, int n_kv_heads, int num_seqs, int64_t q_len_flatten,
                        const int32_t* cu_seqlens, const int32_t* block_tables, int max_blocks_per_seq,
                        const int32_t* kv_lens, int kv_cap, const int32_t* positions, const PrefillPlan& plan,
                        const QOLayout& lay, int tiles_per_split, int max_splits, float* ws_o, float* ws_lse, void* ws,
                        int* err, cudaStream_t stream) {
#define FVB_TC_ARGS q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, q_len_flatten, cu_seqlens, block_tables, \
                    max_blocks_per_seq, kv_lens, kv_cap, positions, plan, lay, nrep, tiles_per_split, max_splits,  \
                    ws_o, ws_lse, ws, err, stream
  if constexpr (kIlv) {
    // decode mode serves groups of 5 and more: tiles of 8 or 16 heads
    return tc_tile_heads(nrep) == 8 ? launch_tc<T, D, 8, true>(FVB_TC_ARGS) : launch_tc<T, D, 16, true>(FVB_TC_ARGS);
  } else {
    switch (tc_tile_heads(nrep)) {
      case 1:
        return launch_tc<T, D, 1, false>(FVB_TC_ARGS);
      case 2:
        return launch_tc<T, D, 2, false>(FVB_TC_ARGS);
      case 4:
        return launch_tc<T, D, 4, false>(FVB_TC_ARGS);
      case 8:
        return launch_tc<T, D, 8, false>(FVB_TC_ARGS);
      default:
        return launch_tc<T, D, 16, false>(FVB_TC_ARGS);
    }
  }
#undef FVB_TC_ARGS
}

}  // namespace

cudaError_t launch_prefill_plan(const int32_t* cu_seqlens, const int32_t* kv_lens, int num_seqs, int tile_tokens,
                                int tiles_per_item, int32_t* order, int32_t* cu_items, cudaStream_t stream,
                                int skip_single) {
  prefill_plan_kernel<<<1, 1024, 0, stream>>>(cu_seqlens, kv_lens, num_seqs, tile_tokens, tiles_per_item, order,
                                              cu_items, skip_single);
  return cudaGetLastError();
}

PrefillPlan plan_prefill(int num_seqs, int n_heads, int n_kv_heads, int head_dim, int64_t q_len_flatten,
                         int max_q_len, int dtype) {
  (void)head_dim;
  (void)max_q_len;
  PrefillPlan p{};
  if (dtype == FVB_DTYPE_F32 || n_kv_heads <= 0 || n_heads % n_kv_heads) {
    p.tile_tokens = 0;
    p.max_tiles = 0;
    p.ws_bytes = 0;
    return p;
  }
  p.tile_tokens = kTileM / tc_tile_heads(n_heads / n_kv_heads);
  // Work items are query-tile pairs; each sequence wastes at most one partial pair.
  p.max_tiles = (q_len_flatten + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens) + num_seqs;
  // order[num_seqs] (padded to 64 entries) + cu_items[num_seqs + 1]
  p.ws_bytes = ((size_t((num_seqs + 63) & ~63) + num_seqs + 1) * 4 + 255) & ~size_t(255);
  // Sequences of one query token (decode rows of a mixed batch) fill 1 / tile_tokens of a
  // query tile here; with GQA groups of up to 4 they go to the split-KV decode kernel
  // instead, whose partials (at most kSingleRowMaxSplits splits per row) follow the plan
  // when they fit in 64 MB (and the sequences in the decode grid's third dimension).
  const int group = n_heads / n_kv_heads;
  const size_t rows = size_t(num_seqs) * n_heads * kSingleRowMaxSplits;
  const size_t single_bytes = ((rows * head_dim * 4 + 255) & ~size_t(255)) + rows * 4;
  p.single_rows_apart = group <= 4 && single_bytes <= (size_t(64) << 20) && num_seqs <= 65535;
  p.off_single = p.ws_bytes;
  if (p.single_rows_apart) p.ws_bytes += single_bytes;
  return p;
}

cudaError_t launch_prefill(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                           int n_heads, int n_kv_heads, int head_dim, int num_seqs, int64_t q_len_flatten,
                           const int32_t* cu_seqlens, int max_q_len, const int32_t* block_tables,
                           int max_blocks_per_seq, const int32_t* kv_lens, const int32_t* positions, int dtype,
                           const PrefillPlan& plan, const QOLayout& lay, void* workspace, int* err,
                           cudaStream_t stream) {
  (void)max_q_len;
  if (num_seqs == 0 || q_len_flatten == 0) return cudaSuccess;
  const int nrep = n_heads / n_kv_heads;
  const int kv_cap = int(std::min<int64_t>(int64_t(max_blocks_per_seq) * kPageSize, 0x7fffffff));
#define FVB_DISPATCH_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, q_len_flatten, cu_seqlens, \
                          block_tables, max_blocks_per_seq, kv_lens, kv_cap, positions, plan, lay, 0, 1, nullptr,  \
                          nullptr, workspace, err, stream
  cudaError_t ce;
  if (dtype == FVB_DTYPE_BF16) {
    ce = head_dim == 128 ? dispatch_tc<__nv_bfloat16, 128, false>(FVB_DISPATCH_ARGS)
                         : dispatch_tc<__nv_bfloat16, 64, false>(FVB_DISPATCH_ARGS);
  } else {
    ce = head_dim == 128 ? dispatch_tc<__half, 128, false>(FVB_DISPATCH_ARGS)
                         : dispatch_tc<__half, 64, false>(FVB_DISPATCH_ARGS);
  }
#undef FVB_DISPATCH_ARGS
  if (ce != cudaSuccess || !plan.single_rows_apart) return ce;
  // The split-KV decode kernel takes the single-token sequences (prefill_plan_kernel gave
  // them no tile), launched as a programmatic dependent of the tensor-core kernel so its
  // CTAs fill the SMs that kernel's last wave leaves idle.  Its plan is sized for the
  // block table's capacity, with splits lengthened until there are at most
  // kSingleRowMaxSplits.
  DecodePlan dp = plan_decode(num_seqs, n_heads, n_kv_heads, head_dim, kv_cap, device_sm_count());
  const int max_pages = std::max(1, (kv_cap + kPageSize - 1) / kPageSize);
  while (dp.max_splits > kSingleRowMaxSplits) {
    dp.pages_per_split *= 2;
    dp.max_splits = (max_pages + dp.pages_per_split - 1) / dp.pages_per_split;
  }
  return launch_decode(q, out, k_pool, v_pool, num_blocks, n_heads, n_kv_heads, head_dim, num_seqs, block_tables,
                       max_blocks_per_seq, kv_lens, kv_cap, dtype, dp, lay,
                       static_cast<uint8_t*>(workspace) + plan.off_single, err, stream, cu_seqlens, positions);
}

TcDecodePlan plan_tc_decode(int num_seqs, int n_heads, int n_kv_heads, int head_dim, int max_kv_len, int num_sms) {
  TcDecodePlan p{};
  p.base = plan_prefill(num_seqs, n_heads, n_kv_heads, head_dim, num_seqs, 1, FVB_DTYPE_BF16);
  p.tiles_per_split = 0;
  p.max_splits = 1;
  p.ws_bytes = p.base.ws_bytes;
  if (num_seqs <= 0 || n_kv_heads <= 0) return p;
  const int group = n_heads / n_kv_heads, tile = tc_tile_heads(group);
  const int64_t ctas = int64_t(num_seqs) * n_kv_heads * ((group + tile - 1) / tile);
  const int kv_tiles = std::max(1, (max_kv_len + kTileN - 1) / kTileN);
  // One resident CTA per SM (TMEM and shared memory): split the KV range until there
  // are about two waves, keeping at least 4 tiles (512 keys) per split.
  const int64_t target = int64_t(num_sms) * 2;
  if (ctas >= target || kv_tiles < 8) return p;
  int splits = int(std::min<int64_t>((target + ctas - 1) / ctas, kv_tiles / 4));
  if (splits <= 1) return p;
  const int tps = (kv_tiles + splits - 1) / splits;
  splits = (kv_tiles + tps - 1) / tps;
  if (splits <= 1) return p;
  p.tiles_per_split = tps;
  p.max_splits = splits;
  const size_t rows = size_t(num_seqs) * n_heads * splits;
  p.off_o = p.base.ws_bytes;
  p.off_lse = p.off_o + ((rows * head_dim * 4 + 255) & ~size_t(255));
  p.ws_bytes = p.off_lse + rows * 4;
  return p;
}

cudaError_t launch_tc_decode(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                             int n_heads, int n_kv_heads, int head_dim, int num_seqs, const int32_t* block_tables,
                             int max_blocks_per_seq, const int32_t* kv_lens, int max_kv_len, int dtype,
                             const TcDecodePlan& plan, const QOLayout& lay, void* workspace, int* err,
                             cudaStream_t stream) {
  if (num_seqs == 0) return cudaSuccess;
  const int nrep = n_heads / n_kv_heads;
  // The longest context any sequence may attend over: max_kv_len, the block-table row and,
  // with split-KV, the splits the plan launches (the combine sizes its shared memory and
  // reads its partial rows by the same bound).
  int64_t cap = std::min<int64_t>(max_kv_len, int64_t(max_blocks_per_seq) * kPageSize);
  if (plan.tiles_per_split > 0) cap = std::min<int64_t>(cap, int64_t(plan.max_splits) * plan.tiles_per_split * kTileN);
  const int kv_cap = int(cap);
  float* ws_o = nullptr;
  float* ws_lse = nullptr;
  if (plan.tiles_per_split > 0) {
    ws_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.off_o);
    ws_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.off_lse);
  }
  // decode mode: no cu_seqlens / positions (token s = sequence s at position kv_len - 1)
#define FVB_TCD_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, int64_t(num_seqs), nullptr, \
                     block_tables, max_blocks_per_seq, kv_lens, kv_cap, nullptr, plan.base, lay,                  \
                     plan.tiles_per_split, plan.max_splits, ws_o, ws_lse, workspace, err, stream
  cudaError_t ce;
  if (dtype == FVB_DTYPE_BF16) {
    ce = head_dim == 128 ? dispatch_tc<__nv_bfloat16, 128, true>(FVB_TCD_ARGS)
                         : dispatch_tc<__nv_bfloat16, 64, true>(FVB_TCD_ARGS);
  } else {
    ce = head_dim == 128 ? dispatch_tc<__half, 128, true>(FVB_TCD_ARGS) : dispatch_tc<__half, 64, true>(FVB_TCD_ARGS);
  }
#undef FVB_TCD_ARGS
  if (ce != cudaSuccess || plan.tiles_per_split == 0) return ce;
  return launch_decode_combine(ws_o, ws_lse, out, kv_lens, kv_cap, num_seqs, n_heads,
                               head_dim, plan.tiles_per_split * (kTileN / kPageSize), plan.max_splits, dtype, lay,
                               stream);
}

}  // namespace fvb
