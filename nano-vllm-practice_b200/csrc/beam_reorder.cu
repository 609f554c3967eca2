// Beam search's state follows the chosen beams: block tables and paged K/V of every layer,
// one launch.
//
// The reference has no beams; its block manager shares full pages between requests and
// copies none (femtovllm/engine/core_engine.py:140-162 lays out the pools).  All beams of a
// request hold kv_len tokens: `full` = kv_len / block_size full pages, which beams share by
// reference, and from table column `full` on the open pages, of which every row owns its
// own (the first holds the kv_len % block_size newest tokens).  Row r of the next step
// continues row p = parents[r] of this one:
//
//   table columns < full    p's: the pages are shared;
//   open pages              p's for the first of p's children, which carries on in them;
//                           every further child takes those of a row that has no child and
//                           gets a copy of p's newest tokens.  There are as many further
//                           children as rows without a child, so no page has to be allocated
//                           or freed, and no page that is copied from is copied to.
//
// The matching needs only the request's parents: every CTA (row, layer) derives its own row's
// part of it from two 64-bit masks, and CTAs of rows with nothing to copy end there.
//
// Bound by HBM where much is copied: 32 requests x 8 beams, 28 layers, 8 heads x 128 bf16, 173 MB read and written,
// 32.6 us = 5.3 TB/s (open pages of 1 to 15 tokens: runs of 256 bytes to 3.75 KB a head).  One request's 4 beams, 4
// layers: 4.1 us, which is a launch and three dependent loads.
#include "common.cuh"
#include "kernels.h"

namespace fvb {
namespace {

constexpr int kThreads = 128;
constexpr int kLayersPerLaunch = 64;

struct Layers {
  const void* k[kLayersPerLaunch];
  const void* v[kLayersPerLaunch];
};

__global__ void __launch_bounds__(kThreads) beam_reorder_kernel(
    const __grid_constant__ Layers layers, int64_t num_blocks, int n_kv_heads, int row_bytes, int block_size,
    const int32_t* __restrict__ tables, int32_t* __restrict__ new_tables, int width,
    const int32_t* __restrict__ kv_lens, const int64_t* __restrict__ parents, int num_beams, bool first_launch,
    int* __restrict__ err) {
  const int W = num_beams;
  const int64_t row0 = int64_t(blockIdx.x) / W * W;  // the request's first row
  const int r = int(blockIdx.x - row0);
  const int lane = threadIdx.x & 31;
  // ---- parents of the request, two a lane (every warp for itself) ----
  int p[2];
  bool bad = false;
  const int kv = __ldg(kv_lens + row0);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + 32 * j;
    p[j] = -1;
    if (i < W) {
      const int64_t x = __ldg(parents + row0 + i);
      bad = bad || x < 0 || x >= W || __ldg(kv_lens + row0 + i) != kv;
      p[j] = int(x);
    }
  }
  const int full = kv / block_size, fill = kv - full * block_size;
  bad = bad || kv < 0 || full + (fill > 0) > width;
  const bool skip = __any_sync(0xffffffffu, bad);  // malformed: the request's rows stay as they are
  if (skip && threadIdx.x == 0 && r == 0 && blockIdx.y == 0) record_error(err, FVB_ERR_INVALID_ARGUMENT, int(row0));
  int parent = r, donor = r;
  if (!skip) {
    // rows that have a child, and rows that are not their parent's first child
    uint64_t child[2], surplus = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __reduce_or_sync(0xffffffffu, p[j] >= 0 && p[j] < 32 ? 1u << p[j] : 0u);
      const uint32_t hi = __reduce_or_sync(0xffffffffu, p[j] >= 32 ? 1u << (p[j] - 32) : 0u);
      child[j] = uint64_t(hi) << 32 | lo;
      const uint32_t same = __match_any_sync(0xffffffffu, p[j]);
      bool later = (same & ((1u << lane) - 1)) != 0;
      if (j == 1) later = later || (p[1] >= 0 && ((child[0] >> p[1]) & 1));
      surplus |= uint64_t(__ballot_sync(0xffffffffu, p[j] >= 0 && later)) << (32 * j);
    }
    const uint64_t rows = W == 64 ? ~uint64_t(0) : (uint64_t(1) << W) - 1;
    uint64_t idle = rows & ~(child[0] | child[1]);
    parent = __shfl_sync(0xffffffffu, r < 32 ? p[0] : p[1], r & 31);
    donor = parent;
    if ((surplus >> r) & 1) {
      for (int n = __popcll(surplus & ((uint64_t(1) << r) - 1)); n > 0; --n) idle &= idle - 1;
      donor = __ffsll(idle) - 1;
    }
  }
  const int32_t* from = tables + (row0 + parent) * width;  // shared pages and newest tokens
  const int32_t* open = tables + (row0 + donor) * width;   // open pages
  if (first_launch && blockIdx.y == 0) {
    int32_t* to = new_tables + (row0 + r) * width;
    for (int c = threadIdx.x; c < width; c += kThreads) to[c] = __ldg((c < full ? from : open) + c);
  }
  if (parent == donor || fill == 0) return;
  const int src = __ldg(from + full), dst = __ldg(open + full);
  if (src < 0 || src >= num_blocks || dst < 0 || dst >= num_blocks) {
    if (threadIdx.x == 0) record_error(err, FVB_ERR_BAD_PAGE, int(row0) + r);
    return;
  }
  // ---- the filled tokens of every kv head: fill * row_bytes contiguous bytes at a page-head pitch ----
  const int per_head = fill * (row_bytes >> 4);  // 16-byte vectors
  const int pitch = block_size * (row_bytes >> 4);
  const int total = n_kv_heads * per_head;
  const int64_t src0 = int64_t(src) * n_kv_heads * pitch, dst0 = int64_t(dst) * n_kv_heads * pitch;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    uint4* pool = static_cast<uint4*>(const_cast<void*>(which ? layers.v[blockIdx.y] : layers.k[blockIdx.y]));
    constexpr int kUnroll = 4;
    for (int i0 = threadIdx.x; i0 < total; i0 += kThreads * kUnroll) {
      uint4 x[kUnroll];
      int64_t at[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = i0 + u * kThreads;
        const int h = i / per_head;
        at[u] = int64_t(h) * pitch + (i - h * per_head);
        if (i < total) x[u] = pool[src0 + at[u]];
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (i0 + u * kThreads < total) pool[dst0 + at[u]] = x[u];
      }
    }
  }
}

}  // namespace

cudaError_t launch_beam_reorder(const void* const* k_pools, const void* const* v_pools, int num_layers,
                                int64_t num_blocks, int n_kv_heads, int head_dim, int block_size, int esize,
                                const int32_t* block_tables, int32_t* new_tables, int max_blocks_per_seq,
                                const int32_t* kv_lens, const int64_t* parents, int num_requests, int num_beams,
                                int* err, cudaStream_t stream) {
  for (int done = 0; done < num_layers; done += kLayersPerLaunch) {
    Layers layers{};
    const int n = num_layers - done < kLayersPerLaunch ? num_layers - done : kLayersPerLaunch;
    for (int i = 0; i < n; ++i) {
      layers.k[i] = k_pools[done + i];
      layers.v[i] = v_pools[done + i];
    }
    beam_reorder_kernel<<<dim3(unsigned(num_requests) * num_beams, n), kThreads, 0, stream>>>(
        layers, num_blocks, n_kv_heads, head_dim * esize, block_size, block_tables, new_tables, max_blocks_per_seq,
        kv_lens, parents, num_beams, done == 0, err);
    const cudaError_t ce = cudaGetLastError();
    if (ce != cudaSuccess) return ce;
  }
  return cudaSuccess;
}

}  // namespace fvb
