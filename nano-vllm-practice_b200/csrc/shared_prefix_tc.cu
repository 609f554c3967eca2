// The shared prefixes of a decode batch on the tensor cores (prefix form of the kernel in
// prefill_tc.cuh): the 16-bit part of shared_prefix.cu.
#include "prefill_tc.cuh"

namespace fvb {
namespace {

template <typename T, int D, bool kIlv>
cudaError_t dispatch(int nrep, const void* q, const void* k_pool, const void* v_pool, int64_t num_blocks,
                     int n_kv_heads, int num_seqs, const int32_t* block_tables, int max_blocks_per_seq,
                     const int32_t* kv_lens, const PrefillPlan& items, const QOLayout& lay, int tiles_per_split,
                     int splits, float* ws_o, float* ws_lse, int* err, cudaStream_t stream, const DecodeExtra& ex) {
#define FVB_PT_ARGS q, nullptr, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, int64_t(num_seqs), nullptr, \
                    block_tables, max_blocks_per_seq, kv_lens, ex.prefix_cap, nullptr, items, lay, nrep,      \
                    tiles_per_split, splits, ws_o, ws_lse, nullptr, err, stream, ex
  switch (tc_tile_heads(nrep)) {
    case 1:
      return launch_tc<T, D, 1, kIlv, kTcPrefix>(FVB_PT_ARGS);
    case 2:
      return launch_tc<T, D, 2, kIlv, kTcPrefix>(FVB_PT_ARGS);
    case 4:
      return launch_tc<T, D, 4, kIlv, kTcPrefix>(FVB_PT_ARGS);
    case 8:
      return launch_tc<T, D, 8, kIlv, kTcPrefix>(FVB_PT_ARGS);
    default:
      return launch_tc<T, D, 16, kIlv, kTcPrefix>(FVB_PT_ARGS);
  }
#undef FVB_PT_ARGS
}

}  // namespace

cudaError_t launch_prefix_tc(const void* q, const void* k_pool, const void* v_pool, int64_t num_blocks, int n_heads,
                             int n_kv_heads, int head_dim, int num_seqs, const int32_t* block_tables,
                             int max_blocks_per_seq, const int32_t* kv_lens, int dtype, const SharedPrefixPlan& plan,
                             const QOLayout& lay, float* ws_o, float* ws_lse, const DecodeExtra& ex, int* err,
                             cudaStream_t stream) {
  const int nrep = n_heads / n_kv_heads;
  const int item_tok = kTileM / tc_tile_heads(nrep) * (plan.single_tiles ? 1 : 2);
  PrefillPlan items{};  // at most one partial item per group
  items.max_tiles = num_seqs / item_tok + ex.num_groups;
#define FVB_PT_ARGS nrep, q, k_pool, v_pool, num_blocks, n_kv_heads, num_seqs, block_tables, max_blocks_per_seq, \
                    kv_lens, items, lay, plan.keys_per_split / kTileN, plan.prefix_splits, ws_o, ws_lse, err,   \
                    stream, ex
#define FVB_PT_TYPE(T, D) \
  plan.single_tiles ? dispatch<T, D, true>(FVB_PT_ARGS) : dispatch<T, D, false>(FVB_PT_ARGS)
  if (dtype == FVB_DTYPE_BF16)
    return head_dim == 128 ? (FVB_PT_TYPE(__nv_bfloat16, 128)) : (FVB_PT_TYPE(__nv_bfloat16, 64));
  return head_dim == 128 ? (FVB_PT_TYPE(__half, 128)) : (FVB_PT_TYPE(__half, 64));
#undef FVB_PT_TYPE
#undef FVB_PT_ARGS
}

}  // namespace fvb
