// Paged attention with a sliding window and sinks on the tensor cores: chunked prefill and
// the decode of 16-bit GQA groups of 5 and more (window form of the kernel in prefill_tc.cuh).
#include "prefill_tc.cuh"

namespace fvb {
namespace {

template <typename T, int D, bool kIlv>
cudaError_t dispatch(int nrep, const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                     int n_kv_heads, int num_seqs, int64_t q_len_flatten, const int32_t* cu_seqlens,
                     const int32_t* block_tables, int max_blocks_per_seq, const int32_t* kv_lens, int kv_cap,
                     const int32_t* positions, const PrefillPlan& plan, const QOLayout& lay, int tiles_per_split,
                     int max_splits, float* ws_o, float* ws_lse, void* ws, int* err, cudaStream_t stream,
                     const DecodeExtra& ex) {
#define FVB_TW_ARGS q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, q_len_flatten, cu_seqlens, block_tables, \
                    max_blocks_per_seq, kv_lens, kv_cap, positions, plan, lay, nrep, tiles_per_split, max_splits,  \
                    ws_o, ws_lse, ws, err, stream, ex
  if constexpr (kIlv) {
    return tc_tile_heads(nrep) == 8 ? launch_tc<T, D, 8, true, kTcWindow>(FVB_TW_ARGS)
                                    : launch_tc<T, D, 16, true, kTcWindow>(FVB_TW_ARGS);
  } else {
    switch (tc_tile_heads(nrep)) {
      case 1:
        return launch_tc<T, D, 1, false, kTcWindow>(FVB_TW_ARGS);
      case 2:
        return launch_tc<T, D, 2, false, kTcWindow>(FVB_TW_ARGS);
      case 4:
        return launch_tc<T, D, 4, false, kTcWindow>(FVB_TW_ARGS);
      case 8:
        return launch_tc<T, D, 8, false, kTcWindow>(FVB_TW_ARGS);
      default:
        return launch_tc<T, D, 16, false, kTcWindow>(FVB_TW_ARGS);
    }
  }
#undef FVB_TW_ARGS
}

DecodeExtra window_extra(int window, int sinks) {
  DecodeExtra ex;
  ex.window = window;
  ex.sinks = sinks;
  ex.unit = kTileN;
  return ex;
}

}  // namespace

cudaError_t launch_window_prefill(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                                  int n_heads, int n_kv_heads, int head_dim, int num_seqs, int64_t q_len_flatten,
                                  const int32_t* cu_seqlens, const int32_t* block_tables, int max_blocks_per_seq,
                                  const int32_t* kv_lens, const int32_t* positions, int window, int sinks, int dtype,
                                  const PrefillPlan& plan, const QOLayout& lay, void* workspace, int* err,
                                  cudaStream_t stream) {
  if (num_seqs == 0 || q_len_flatten == 0) return cudaSuccess;
  const int nrep = n_heads / n_kv_heads;
  const int kv_cap = int(std::min<int64_t>(int64_t(max_blocks_per_seq) * kPageSize, 0x7fffffff));
  const DecodeExtra ex = window_extra(window, sinks);
#define FVB_WP_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, q_len_flatten, cu_seqlens, \
                    block_tables, max_blocks_per_seq, kv_lens, kv_cap, positions, plan, lay, 0, 1, nullptr, nullptr, \
                    workspace, err, stream, ex
  cudaError_t ce;
  if (dtype == FVB_DTYPE_BF16) {
    ce = head_dim == 128 ? dispatch<__nv_bfloat16, 128, false>(FVB_WP_ARGS)
                         : dispatch<__nv_bfloat16, 64, false>(FVB_WP_ARGS);
  } else {
    ce = head_dim == 128 ? dispatch<__half, 128, false>(FVB_WP_ARGS) : dispatch<__half, 64, false>(FVB_WP_ARGS);
  }
#undef FVB_WP_ARGS
  if (ce != cudaSuccess || !plan.single_rows_apart) return ce;
  // The single-token sequences, as in launch_prefill: the split-KV kernel's window form, as a
  // programmatic dependent, with at most the splits whose partials the workspace reserves.
  DecodePlan dp =
      plan_window_decode(num_seqs, n_heads, n_kv_heads, head_dim, kv_cap, window, sinks, device_sm_count());
  const int max_pages = window_max_units(kv_cap, window, sinks, kPageSize);
  while (dp.max_splits > kSingleRowMaxSplits) {
    dp.pages_per_split *= 2;
    dp.max_splits = (max_pages + dp.pages_per_split - 1) / dp.pages_per_split;
  }
  return launch_window_decode(q, out, k_pool, v_pool, num_blocks, n_heads, n_kv_heads, head_dim, num_seqs,
                              block_tables, max_blocks_per_seq, kv_lens, kv_cap, window, sinks, dtype, dp, lay,
                              static_cast<uint8_t*>(workspace) + plan.off_single, err, stream, cu_seqlens, positions);
}

TcDecodePlan plan_window_tc_decode(int num_seqs, int n_heads, int n_kv_heads, int head_dim, int max_kv_len, int window,
                                   int sinks, int num_sms) {
  const int64_t keys = int64_t(window_max_units(max_kv_len, window, sinks, kTileN)) * kTileN;
  return plan_tc_decode(num_seqs, n_heads, n_kv_heads, head_dim, int(std::min<int64_t>(keys, 0x7fffff80)), num_sms);
}

cudaError_t launch_window_tc_decode(const void* q, void* out, const void* k_pool, const void* v_pool,
                                    int64_t num_blocks, int n_heads, int n_kv_heads, int head_dim, int num_seqs,
                                    const int32_t* block_tables, int max_blocks_per_seq, const int32_t* kv_lens,
                                    int max_kv_len, int window, int sinks, int dtype, const TcDecodePlan& plan,
                                    const QOLayout& lay, void* workspace, int* err, cudaStream_t stream) {
  if (num_seqs == 0) return cudaSuccess;
  const int nrep = n_heads / n_kv_heads;
  const int kv_cap = int(std::min<int64_t>(max_kv_len, int64_t(max_blocks_per_seq) * kPageSize));
  float* ws_o = nullptr;
  float* ws_lse = nullptr;
  if (plan.tiles_per_split > 0) {
    ws_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.off_o);
    ws_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.off_lse);
  }
  const DecodeExtra ex = window_extra(window, sinks);
#define FVB_WD_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, int64_t(num_seqs), nullptr, \
                    block_tables, max_blocks_per_seq, kv_lens, kv_cap, nullptr, plan.base, lay,                  \
                    plan.tiles_per_split, plan.max_splits, ws_o, ws_lse, workspace, err, stream, ex
  cudaError_t ce;
  if (dtype == FVB_DTYPE_BF16) {
    ce = head_dim == 128 ? dispatch<__nv_bfloat16, 128, true>(FVB_WD_ARGS)
                         : dispatch<__nv_bfloat16, 64, true>(FVB_WD_ARGS);
  } else {
    ce = head_dim == 128 ? dispatch<__half, 128, true>(FVB_WD_ARGS) : dispatch<__half, 64, true>(FVB_WD_ARGS);
  }
#undef FVB_WD_ARGS
  if (ce != cudaSuccess || plan.tiles_per_split == 0) return ce;
  return launch_window_combine(ws_o, ws_lse, out, kv_lens, kv_cap, num_seqs, n_heads, head_dim, window, sinks, kTileN,
                               plan.tiles_per_split, plan.max_splits, dtype, lay, stream);
}

}  // namespace fvb
