// Chunked-prefill paged attention with a sliding window and sinks on the tensor cores (window
// form of the kernel in prefill_tc.cuh).
//
// The sinks' and the window's pages are packed into one line of columns, so KV tiles hold pages of both and none that
// no row sees; each CTA finds its item by a scan of cu_seqlens, so no plan kernel runs in front.  Measured: a tile
// pair takes 1.9 us of an SM (16.8 MFLOP: 1.3 PFLOP/s over the device), an item 9 us more for its start and end.
// 8 chunks of 128 to 2048 tokens, 16/8 heads x 128, window 1024 (104 GFLOP): 181 us = 0.57 PFLOP/s (216 with whole
// tiles of sinks and window and a plan kernel in front).
#include "prefill_tc.cuh"

namespace fvb {
namespace {

template <typename T, int D>
cudaError_t dispatch(int nrep, const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                     int n_kv_heads, int num_seqs, int64_t q_len_flatten, const int32_t* cu_seqlens,
                     const int32_t* block_tables, int max_blocks_per_seq, const int32_t* kv_lens, int kv_cap,
                     const int32_t* positions, const PrefillPlan& plan, const QOLayout& lay, void* ws, int* err,
                     cudaStream_t stream, const DecodeExtra& ex) {
#define FVB_TW_ARGS q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, q_len_flatten, cu_seqlens, block_tables, \
                    max_blocks_per_seq, kv_lens, kv_cap, positions, plan, lay, nrep, \
                    plan.single_rows_apart ? -1 : 0, 1, nullptr, nullptr, ws, err, stream, ex
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
#undef FVB_TW_ARGS
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
  DecodeExtra ex;
  ex.window = window;
  ex.sinks = sinks;
#define FVB_WP_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, q_len_flatten, cu_seqlens, \
                    block_tables, max_blocks_per_seq, kv_lens, kv_cap, positions, plan, lay, workspace, err, \
                    stream, ex
  cudaError_t ce;
  if (dtype == FVB_DTYPE_BF16) {
    ce = head_dim == 128 ? dispatch<__nv_bfloat16, 128>(FVB_WP_ARGS)
                         : dispatch<__nv_bfloat16, 64>(FVB_WP_ARGS);
  } else {
    ce = head_dim == 128 ? dispatch<__half, 128>(FVB_WP_ARGS) : dispatch<__half, 64>(FVB_WP_ARGS);
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

}  // namespace fvb
