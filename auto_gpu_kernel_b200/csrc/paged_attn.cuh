// What the kernels of the dense paged attention share: the requests' tiles, their even split over the CTAs, and
// the places of the partial results.
//
// A request of `len` cached tokens is max(1, ceil(len / 64)) tiles of one page each (the one tile of an empty
// request holds nothing and writes its zero output).  The tiles of all requests, one after the other, are cut into
// equal ranges, one per CTA of a row block; where a request is cut, every CTA that has a part of it (a "segment")
// leaves a partial result.  Lengths live on the device, so every CTA works the split out for itself.
#pragma once

#include "common.cuh"

namespace dsa {

struct PagedArgs {
  const __nv_bfloat16* q_nope;
  const __nv_bfloat16* q_pe;
  const int32_t* seq_lens;
  const int32_t* block_table;
  int64_t table_stride;
  __nv_bfloat16* out;
  float* lse;
  float* part;      // partial results of cut requests
  float* logits;    // base-2 logits [batch][max_pages][row blocks][rows of a block][64], or null
  int32_t* status;
  float scale_log2;
  int batch, max_pages, num_pages;
  int rows;         // query rows of a request: its new tokens x heads
  int heads, tokens;
  int block_rows;   // query rows that a CTA takes at once (a row block)
  int grid_x;       // ranges the tiles are cut into
};

constexpr int kPagedMaxRanges = 512;

// Query rows that a CTA takes at once, from the rows of a request: 16 or 32 by warp-level products (one or two row
// groups per page), 64 by tcgen05.
inline int paged_block_rows(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

__host__ __device__ inline int paged_len(int len, int max_pages) {
  const int64_t most = (int64_t)max_pages * kPage;
  return len < 0 ? 0 : ((int64_t)len > most ? (int)most : len);
}
__host__ __device__ inline int paged_tiles(int len, int max_pages) {
  const int n = (paged_len(len, max_pages) + kPage - 1) / kPage;
  return n < 1 ? 1 : n;
}

// Partial results: per (row block, range, which) a [rows of the block][512] fp32 accumulator ([512][64] for blocks of
// 64 rows), then its running maxima and sums.  `which` is 1 for the segment a request begins with and 0 for the ones that follow: a range
// holds at most one of each.
__host__ __device__ inline size_t paged_part_floats(int block_rows) { return (size_t)block_rows * (kCkv + 2); }
__device__ __forceinline__ float* paged_part(const PagedArgs& a, int block_rows, int rb, int range, int which) {
  return a.part + (((size_t)rb * a.grid_x + range) * 2 + which) * paged_part_floats(block_rows);
}

// Sum of all requests' tiles, and the tiles in front of this thread's share of the requests (requests
// [lo, hi) of equal contiguous shares).  By all threads of the CTA; `sums` has one entry per warp.
template <int kThreads>
__device__ __forceinline__ long long paged_scan(const int32_t* seq_lens, int batch, int max_pages, long long* sums,
                                                int& lo, int& hi, long long& before) {
  const int share = (batch + kThreads - 1) / kThreads;
  lo = min((int)threadIdx.x * share, batch);
  hi = min(lo + share, batch);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += paged_tiles(__ldg(seq_lens + b), max_pages);
  long long upto = mine;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sums[w] = upto;
  __syncthreads();
  long long front = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    if (i < w) front += sums[i];
    total += sums[i];
  }
  before = front + upto - mine;
  return total;
}

}  // namespace dsa
