// Decode paged attention with a sliding window and sinks: the split plan over the pages a
// window can touch, and the dispatch of the split-KV kernel's window form (decode_split.cuh).
#include "decode_split.cuh"

namespace fvb {
namespace {

template <typename T, int D>
cudaError_t dispatch(int nrep, const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                     int n_kv_heads, int num_seqs, const int32_t* block_tables, int max_blocks_per_seq,
                     const int32_t* kv_lens, int max_kv_len, const DecodePlan& plan, const QOLayout& lay, void* ws,
                     int* err, cudaStream_t stream, const int32_t* q_index, const int32_t* q_pos,
                     const DecodeExtra& ex) {
#define FVB_DW_ARGS q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, block_tables, max_blocks_per_seq, \
                    kv_lens, max_kv_len, plan, lay, nrep, ws, err, stream, q_index, q_pos, ex
  switch (decode_tile_heads(nrep)) {
    case 1:
      return launch_decode_t<T, D, 1, kDecodeWindow>(FVB_DW_ARGS);
    case 2:
      return launch_decode_t<T, D, 2, kDecodeWindow>(FVB_DW_ARGS);
    case 4:
      return launch_decode_t<T, D, 4, kDecodeWindow>(FVB_DW_ARGS);
    default:
      return launch_decode_t<T, D, 8, kDecodeWindow>(FVB_DW_ARGS);
  }
#undef FVB_DW_ARGS
}

}  // namespace

int window_max_units(int max_kv_len, int window, int sinks, int unit) {
  const int64_t all = (int64_t(max_kv_len) + unit - 1) / unit;
  // `window` consecutive keys touch at most ceil((window - 1) / unit) + 1 units
  const int64_t near = (int64_t(window) - 1 + unit - 1) / unit + 1;
  const int64_t head = (std::min<int64_t>(sinks, max_kv_len) + unit - 1) / unit;
  return int(std::max<int64_t>(1, std::min(all, near + head)));
}

DecodePlan plan_window_decode(int num_seqs, int n_heads, int n_kv_heads, int head_dim, int max_kv_len, int window,
                              int sinks, int num_sms) {
  const int pages = window_max_units(max_kv_len, window, sinks, kPageSize);
  DecodePlan p = plan_decode(num_seqs, n_heads, n_kv_heads, head_dim, pages * kPageSize, num_sms);
  // Eight pages are one stage for each consumer warp: a shorter split saves no time and may cost the combine
  // (4 short fp32 sequences, window 64: 6.6 us with splits of 4 pages and a combine, 5.4 without).
  constexpr int kOneRound = 8;
  if (p.pages_per_split < kOneRound) {
    p.pages_per_split = kOneRound;
    p.max_splits = (pages + kOneRound - 1) / kOneRound;
    const size_t rows = size_t(num_seqs) * n_heads * p.max_splits;
    p.ws_bytes = p.max_splits > 1 ? ((rows * head_dim * 4 + 255) & ~size_t(255)) + rows * 4 : 0;
  }
  return p;
}

cudaError_t launch_window_decode(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                                 int n_heads, int n_kv_heads, int head_dim, int num_seqs, const int32_t* block_tables,
                                 int max_blocks_per_seq, const int32_t* kv_lens, int max_kv_len, int window, int sinks,
                                 int dtype, const DecodePlan& plan, const QOLayout& lay, void* workspace, int* err,
                                 cudaStream_t stream, const int32_t* q_index, const int32_t* q_pos, DecodeExtra ex) {
  if (num_seqs == 0) return cudaSuccess;
  const int nrep = n_heads / n_kv_heads;
  ex.window = window;
  ex.sinks = sinks;
#define FVB_DW_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, block_tables, \
                    max_blocks_per_seq, kv_lens, max_kv_len, plan, lay, workspace, err, stream, q_index, q_pos, ex
  if (dtype == FVB_DTYPE_BF16)
    return head_dim == 128 ? dispatch<__nv_bfloat16, 128>(FVB_DW_ARGS) : dispatch<__nv_bfloat16, 64>(FVB_DW_ARGS);
  if (dtype == FVB_DTYPE_F16)
    return head_dim == 128 ? dispatch<__half, 128>(FVB_DW_ARGS) : dispatch<__half, 64>(FVB_DW_ARGS);
  return head_dim == 128 ? dispatch<float, 128>(FVB_DW_ARGS) : dispatch<float, 64>(FVB_DW_ARGS);
#undef FVB_DW_ARGS
}

}  // namespace fvb
