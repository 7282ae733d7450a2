// What the kernels of the dense paged attention share: the requests' tiles, their even split over the CTAs, and
// the places of the partial results.
//
// A request of `len` cached tokens is max(1, ceil(len / 64)) tiles of one page each (the one tile of an empty
// request holds nothing and writes its zero output).  The tiles of all requests, one after the other and each request
// with `switch_cost` units of nothing in front, are cut into equal ranges, one per CTA of a row block: taking up a
// request (its q, its output) costs about that many tiles, and a CTA with ten short requests would otherwise end
// long after one that is inside a long one.  Where a request is cut, every CTA that has a part of it (a "segment")
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
  int2* segments;   // [batch] first range and number of the ranges that a request is cut into
  float* part;      // partial results of cut requests
  float* logits;    // base-2 logits [batch][max_pages][row blocks][rows of a block][64], or null
  int32_t* status;
  float scale_log2;
  int batch, max_pages, num_pages;
  int rows;         // query rows of a request: its new tokens x heads
  int heads, tokens;
  int block_rows;   // query rows that a CTA takes at once (a row block)
  int grid_x;       // ranges the tiles are cut into
  int whole;        // PagedSplit: whether and how requests stay whole
  int switch_cost;  // what taking up a request costs, in tiles
};

// Short requests are better left whole: nothing is written for a join, and the join's launch goes.
enum PagedSplit {
  kPagedCut = 0,    // ranges cut requests
  kPagedOne = 1,    // range r is request r
  kPagedSnap = 2,   // a range takes the requests that begin in it
};

// Query rows that a CTA takes at once, from the rows of a request: 16 by warp-level products, 64 by tcgen05.  At 16 rows the
// first keeps three pages in shared memory where the second has room for two beside its q (64 x 32768 tokens 363 us
// against 411 us in runs of a few ms, 1 x 131071 37 us against 53 us); from 17 rows on the second reads the cache once where
// the first would read it for every 16 (32 rows, 64 x 8192 tokens: 118 us, and 154 us for warp-level products with two row
// groups).
inline int paged_block_rows(int rows) { return rows <= 16 ? 16 : 64; }
// What taking up a request costs, in tiles (48 requests of 1 to 16384 tokens, 16 rows: cost 0 / 1 / 2 / 3 / 4 60 / 45 / 41.5 /
// 40.9 / 43.3 us; 64 rows are flat from 2 on, 200 short requests best at 2).
inline int paged_switch_cost(int rows) { return rows <= 16 ? 3 : 2; }

__host__ __device__ inline int paged_len(int len, int max_pages) {
  const int64_t most = (int64_t)max_pages * kPage;
  return len < 0 ? 0 : ((int64_t)len > most ? (int)most : len);
}
__host__ __device__ inline int paged_tiles(int len, int max_pages) {
  const int n = (paged_len(len, max_pages) + kPage - 1) / kPage;
  return n < 1 ? 1 : n;
}

// Partial results: per (row block, range, which) a [rows of the block][512] fp32 accumulator ([16][512][4] for blocks of
// 64 rows: four rows, column, row of the four), then its running maxima and sums.  `which` is 1 for the segment a
// request begins with and 0 for the ones that follow: a range holds at most one of each.
__host__ __device__ inline size_t paged_part_floats(int block_rows) { return (size_t)block_rows * (kCkv + 2); }
__device__ __forceinline__ float* paged_part(const PagedArgs& a, int block_rows, int rb, int range, int which) {
  return a.part + (((size_t)rb * a.grid_x + range) * 2 + which) * paged_part_floats(block_rows);
}

// Sum of all requests' tiles, and the tiles in front of this thread's share of the requests (requests
// [lo, hi) of equal contiguous shares).  By all threads of the CTA; `sums` has one entry per warp.
template <int kThreads>
__device__ __forceinline__ long long paged_scan(const PagedArgs& a, long long* sums, int& lo, int& hi, long long& before) {
  const int share = (a.batch + kThreads - 1) / kThreads;
  lo = min((int)threadIdx.x * share, a.batch);
  hi = min(lo + share, a.batch);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += paged_tiles(__ldg(a.seq_lens + b), a.max_pages);
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

// Units of a range, and the unit that request b's tiles begin at when `tiles` tiles lie in front of it.
// (64-bit divisions are hundreds of instructions, and every thread of a small kernel would make them)
__device__ __forceinline__ long long paged_div(long long x, long long y) {
  return x <= 0x7fffffffll && y <= 0x7fffffffll ? (long long)((uint32_t)x / (uint32_t)y) : x / y;
}
__device__ __forceinline__ long long paged_units(const PagedArgs& a, long long total) {
  return paged_div(total + (long long)a.batch * a.switch_cost + a.grid_x - 1, a.grid_x);
}
__device__ __forceinline__ long long paged_first_unit(const PagedArgs& a, int b, long long tiles) {
  return tiles + (long long)(b + 1) * a.switch_cost;
}

// The tiles of range `range`: from tile start_j of request start_b on, end - begin in number (tiles counted over
// all requests).  By all threads of the CTA; a __syncthreads must follow before the words are read.
struct PagedRange {
  long long begin, end;
  long long unit, per;      // the first tile's unit, units of a range
  int start_b, start_j;
};
template <int kThreads>
__device__ __forceinline__ void paged_find_range(const PagedArgs& a, int range, long long* sums, PagedRange* out) {
  if (a.whole == kPagedOne) {
    if (threadIdx.x == 0) *out = {0, paged_tiles(__ldg(a.seq_lens + range), a.max_pages), 0, 1, range, 0};
    return;
  }
  if (threadIdx.x == 0) out->begin = out->end = 0;      // a range without a request (the scan holds a barrier)
  int lo, hi;
  long long before;
  const long long total = paged_scan<kThreads>(a, sums, lo, hi, before);
  const long long per = paged_units(a, total), v0 = range * per, v1 = v0 + per;
  if (a.whole == kPagedSnap) {
    int ahead = lo > 0 ? paged_tiles(__ldg(a.seq_lens + lo - 1), a.max_pages) : 0;    // tiles of the request before
    for (int b = lo; b < hi; ++b) {
      const int k = paged_tiles(__ldg(a.seq_lens + b), a.max_pages);
      const long long first = paged_first_unit(a, b, before);
      if (first >= v0 && first < v1) {
        if (b == 0 || first - a.switch_cost - ahead < v0) {
          out->begin = before;
          out->start_b = b;
          out->start_j = 0;
        }
        if (b == a.batch - 1 || first + k + a.switch_cost >= v1) out->end = before + k;
      }
      before += k;
      ahead = k;
    }
    return;
  }
  if (threadIdx.x == 0) {
    out->per = per;
    // (a range behind the last unit has no tiles)
    if (v0 >= total + (long long)a.batch * a.switch_cost) out->begin = total;
    if (v1 >= total + (long long)a.batch * a.switch_cost) out->end = total;
  }
  for (int b = lo; b < hi; ++b) {
    const int k = paged_tiles(__ldg(a.seq_lens + b), a.max_pages);
    const long long first = paged_first_unit(a, b, before), begin = first - a.switch_cost, end = first + k;
    if (v0 >= begin && v0 < end) {
      const int j = v0 > first ? (int)(v0 - first) : 0;
      out->begin = before + j;
      out->unit = first + j;
      out->start_b = b;
      out->start_j = j;
    }
    if (v1 >= begin && v1 < end) out->end = before + (v1 > first ? v1 - first : 0);
    before += k;
  }
}

// By the CTA of the first row block that has a request's first tile, its tile `i`: what the join needs to know of it.
__device__ __forceinline__ void paged_tell_segments(const PagedArgs& a, const PagedRange& r, int range, int i, int b, int len) {
  const long long first = r.unit + i + (long long)(b - r.start_b) * a.switch_cost;
  a.segments[b] = make_int2(range, (int)paged_div(first + paged_tiles(len, a.max_pages) - 1, r.per) - range + 1);
}

}  // namespace dsa
