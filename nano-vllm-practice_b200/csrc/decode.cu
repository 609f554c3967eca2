// Decode paged attention over block tables with GQA: the split plan and the dispatch of the
// split-KV kernel and its combine (decode_split.cuh).
#include "decode_split.cuh"

namespace fvb {
namespace {

template <typename T, int D>
cudaError_t dispatch_nrep(int nrep, const void* q, void* out, const void* k_pool, const void* v_pool,
                          int64_t num_blocks, int n_kv_heads, int num_seqs, const int32_t* block_tables,
                          int max_blocks_per_seq, const int32_t* kv_lens, int max_kv_len, const DecodePlan& plan,
                          const QOLayout& lay, void* ws, int* err, cudaStream_t stream, const int32_t* q_index,
                          const int32_t* q_pos) {
#define FVB_DT_ARGS q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, block_tables, max_blocks_per_seq, \
                    kv_lens, max_kv_len, plan, lay, nrep, ws, err, stream, q_index, q_pos
  switch (decode_tile_heads(nrep)) {
    case 1:
      return launch_decode_t<T, D, 1>(FVB_DT_ARGS);
    case 2:
      return launch_decode_t<T, D, 2>(FVB_DT_ARGS);
    case 4:
      return launch_decode_t<T, D, 4>(FVB_DT_ARGS);
    default:
      return launch_decode_t<T, D, 8>(FVB_DT_ARGS);
  }
#undef FVB_DT_ARGS
}

}  // namespace

DecodePlan plan_decode(int num_seqs, int n_heads, int n_kv_heads, int head_dim, int max_kv_len, int num_sms) {
  DecodePlan p{};
  const int max_pages = std::max(1, (max_kv_len + kPageSize - 1) / kPageSize);
  const int group = n_kv_heads > 0 ? n_heads / n_kv_heads : 1;
  const int tile = decode_tile_heads(group);
  const int64_t units = int64_t(num_seqs) * n_kv_heads * ((group + tile - 1) / tile);
  // Splits of up to 256 pages (4096 tokens): each CTA start costs a pipeline fill
  // and drain, which at 1024-token splits held 32k-131k-token contexts 5-8 %
  // below the longer splits.  The longest sequence keeps at least 4 splits down to
  // 64 pages (contexts of 512-4096 tokens keep 1024-token splits, whose shorter
  // tail measured 0.6 % faster there), and splits halve (down to 4 pages) until
  // there are enough CTAs for ~4 waves of 3 resident CTAs per SM.
  const int64_t target = int64_t(num_sms) * 3 * 4;
  int pps = 256;
  while (pps > 64 && max_pages < 4 * pps) pps /= 2;
  while (pps > 4 && units * ((max_pages + pps - 1) / pps) < target) pps /= 2;
  p.pages_per_split = pps;
  p.max_splits = (max_pages + pps - 1) / pps;
  if (p.max_splits > 1) {
    const size_t o_bytes = size_t(num_seqs) * n_heads * p.max_splits * head_dim * 4;
    const size_t lse_bytes = size_t(num_seqs) * n_heads * p.max_splits * 4;
    p.ws_bytes = ((o_bytes + 255) & ~size_t(255)) + lse_bytes;
  } else {
    p.ws_bytes = 0;
  }
  return p;
}

cudaError_t launch_decode(const void* q, void* out, const void* k_pool, const void* v_pool, int64_t num_blocks,
                          int n_heads, int n_kv_heads, int head_dim, int num_seqs, const int32_t* block_tables,
                          int max_blocks_per_seq, const int32_t* kv_lens, int max_kv_len, int dtype,
                          const DecodePlan& plan, const QOLayout& lay, void* workspace, int* err,
                          cudaStream_t stream, const int32_t* q_index, const int32_t* q_pos) {
  if (num_seqs == 0) return cudaSuccess;
  const int nrep = n_heads / n_kv_heads;
#define FVB_DECODE_ARGS nrep, q, out, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, block_tables, \
                        max_blocks_per_seq, kv_lens, max_kv_len, plan, lay, workspace, err, stream, q_index, q_pos
  if (dtype == FVB_DTYPE_BF16) {
    return head_dim == 128 ? dispatch_nrep<__nv_bfloat16, 128>(FVB_DECODE_ARGS)
                           : dispatch_nrep<__nv_bfloat16, 64>(FVB_DECODE_ARGS);
  } else if (dtype == FVB_DTYPE_F16) {
    return head_dim == 128 ? dispatch_nrep<__half, 128>(FVB_DECODE_ARGS) : dispatch_nrep<__half, 64>(FVB_DECODE_ARGS);
  } else {
    return head_dim == 128 ? dispatch_nrep<float, 128>(FVB_DECODE_ARGS) : dispatch_nrep<float, 64>(FVB_DECODE_ARGS);
  }
#undef FVB_DECODE_ARGS
}


cudaError_t launch_decode_combine(const float* ws_o, const float* ws_lse, void* out, const int32_t* kv_lens,
                                  int kv_cap, int num_seqs, int n_heads, int head_dim, int pages_per_split,
                                  int max_splits, int dtype, const QOLayout& lay, cudaStream_t stream) {
  if (num_seqs == 0 || max_splits <= 1) return cudaSuccess;
#define FVB_CMB_ARGS ws_o, ws_lse, out, kv_lens, kv_cap, num_seqs, n_heads, pages_per_split, max_splits, lay, stream
  if (dtype == FVB_DTYPE_BF16) {
    return head_dim == 128 ? launch_combine_t<__nv_bfloat16, 128>(FVB_CMB_ARGS)
                           : launch_combine_t<__nv_bfloat16, 64>(FVB_CMB_ARGS);
  } else if (dtype == FVB_DTYPE_F16) {
    return head_dim == 128 ? launch_combine_t<__half, 128>(FVB_CMB_ARGS) : launch_combine_t<__half, 64>(FVB_CMB_ARGS);
  }
  return head_dim == 128 ? launch_combine_t<float, 128>(FVB_CMB_ARGS) : launch_combine_t<float, 64>(FVB_CMB_ARGS);
#undef FVB_CMB_ARGS
}

}  // namespace fvb
