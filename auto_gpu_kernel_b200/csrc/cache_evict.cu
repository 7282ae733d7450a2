// Eviction from the paged caches by accumulated attention weight.
//
//   kept(b) = the first F positions, the last L positions and, of the others, the budget - F - L heaviest (equal weights:
//             the lower position), in ascending order; every position where a request is within the budget
//   token j of the request moves from position kept(b)[j] of its old pages to position j of its new pages.
//
// Two kernels.  The choice is a radix selection over the order-preserving 32-bit keys of the weights (11 + 11 + 10 bits),
// then one sweep that writes the kept positions in order; a row is read four times, from L2 after the first.  The
// move is bound by memory: 1152 B (+ 132 B of an index key and its scale) in and out per kept token.
#include "common.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace dsa {

namespace {

constexpr int kEvThreads = 1024;
constexpr int kEvBins = 2048;

struct EvictArgs {
  const float* weights;
  int64_t weights_stride;
  const int32_t* seq_lens;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* new_table;
  int64_t new_table_stride;
  uint4* ckv;
  uint4* kpe;
  uint8_t* index;
  int32_t* new_lens;
  float* new_weights;
  int64_t new_weights_stride;
  int32_t* kept;
  int64_t kept_stride;
  int32_t* status;
  int batch, max_pages, num_pages, budget, keep_first, keep_last;
};

__device__ __forceinline__ int ev_len(const EvictArgs& a, int b) {
  const int n = __ldg(a.seq_lens + b);
  const int64_t most = (int64_t)a.max_pages * kPage;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}
// -inf and NaN rank lowest, -0 as +0.
__device__ __forceinline__ uint32_t ev_key(float w) {
  return float_to_ordered(w > kScoreFloor ? w + 0.f : kScoreFloor);
}

// Sum of `v` over the threads in front of this one, and over all of them.
__device__ __forceinline__ uint32_t ev_scan(uint32_t v, uint32_t* sums, uint32_t& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) sums[w] = upto;
  __syncthreads();
  if (w == 0) {
    uint32_t s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    sums[lane] = s;
  }
  __syncthreads();
  total = sums[31];
  const uint32_t r = (w ? sums[w - 1] : 0u) + upto - v;
  __syncthreads();
  return r;
}

__global__ void __launch_bounds__(kEvThreads)
evict_choose_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[kEvBins];
  __shared__ uint32_t sums[32];
  __shared__ uint32_t pick[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int n = ev_len(a, b);
  const float* w = a.weights + (int64_t)b * a.weights_stride;
  float* nw = a.new_weights + (int64_t)b * a.new_weights_stride;
  int32_t* kept = a.kept + (int64_t)b * a.kept_stride;
  const int m = n < a.budget ? n : a.budget;
  if (tid == 0) a.new_lens[b] = m;
  for (int j = m + tid; j < a.budget; j += kEvThreads) {
    kept[j] = -1;
    nw[j] = 0.f;
  }
  if (n <= a.budget) {
    for (int j = tid; j < n; j += kEvThreads) {
      kept[j] = j;
      nw[j] = w[j];
    }
    return;
  }
  const int lo = a.keep_first, hi = n - a.keep_last;      // budget < n: the ends do not meet
  const uint32_t want = (uint32_t)(a.budget - a.keep_first - a.keep_last);
  for (int j = tid; j < lo; j += kEvThreads) {
    kept[j] = j;
    nw[j] = w[j];
  }
  for (int j = hi + tid; j < n; j += kEvThreads) {
    kept[a.budget - n + j] = j;
    nw[a.budget - n + j] = w[j];
  }
  if (want == 0) return;

  // ---- the want-th largest key of positions lo .. hi-1, eleven, eleven and ten bits at a time ----
  uint32_t prefix = 0, rest = want;      // keys that begin with `prefix` are still in question; `rest` of them are kept
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kEvThreads) {
      const uint32_t k = ev_key(w[j]);
      if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // bins from the top: thread t has bins 2047 - 2t and 2046 - 2t
    const uint32_t c0 = hist[kEvBins - 1 - 2 * tid], c1 = hist[kEvBins - 2 - 2 * tid];
    uint32_t all;
    const uint32_t above = ev_scan(c0 + c1, sums, all);
    if (above < rest && above + c0 >= rest) {
      pick[0] = kEvBins - 1 - 2 * tid;
      pick[1] = rest - above;
    } else if (above + c0 < rest && above + c0 + c1 >= rest) {
      pick[0] = kEvBins - 2 - 2 * tid;
      pick[1] = rest - above - c0;
    }
    __syncthreads();
    prefix = (prefix << bits) | pick[0];
    rest = pick[1];
    __syncthreads();
  }
  // ---- keys above `prefix` are kept, and the first `rest` that equal it ----
  uint32_t out = (uint32_t)lo, equal = 0;
  for (int j0 = lo; j0 < hi; j0 += 4 * kEvThreads) {
    uint32_t k[4];
    float v[4];
    uint32_t mine = 0;                   // above in the low half, equal in the high half (4096 at most)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + 4 * tid + e;
      v[e] = j < hi ? w[j] : 0.f;
      k[e] = ev_key(v[e]);
      if (j < hi) mine += k[e] > prefix ? 1u : k[e] == prefix ? 0x10000u : 0u;
    }
    uint32_t all;
    const uint32_t front = ev_scan(mine, sums, all);
    uint32_t gt = front & 0xffffu, eq = equal + (front >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + 4 * tid + e;
      if (j < hi) {
        const bool above = k[e] > prefix, same = k[e] == prefix;
        if (above || (same && eq < rest)) {
          const uint32_t at = out + gt + min(eq, rest) - min(equal, rest);
          kept[at] = j;
          nw[at] = v[e];
        }
        gt += above;
        eq += same;
      }
    }
    const uint32_t eq_all = equal + (all >> 16);
    out += (all & 0xffffu) + min(eq_all, rest) - min(equal, rest);
    equal = eq_all;
  }
}

// One warp per kRows kept tokens, all loads of a round in front of its stores.
constexpr int kMvThreads = 256;
constexpr int kMvRows = 4;

template <bool kIndex>
__global__ void __launch_bounds__(kMvThreads)
evict_move_kernel(const EvictArgs a) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const int j0 = (blockIdx.x * (kMvThreads / 32) + (threadIdx.x >> 5)) * kMvRows;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int n = ev_len(a, b), m = n < a.budget ? n : a.budget;
  if (j0 >= m) return;
  // lane r < kMvRows works out the slots of the warp's row r
  int64_t src = -1, dst = -1;
  if (lane < kMvRows && j0 + lane < m) {
    const int j = j0 + lane;
    const int from = __ldcg(a.kept + (int64_t)b * a.kept_stride + j);
    const int p = __ldg(a.table + (int64_t)b * a.table_stride + from / kPage);
    const int q = __ldg(a.new_table + (int64_t)b * a.new_table_stride + j / kPage);
    if (p < 0 || p >= a.num_pages || q < 0 || q >= a.num_pages) {
      raise_status(a.status, DSA_STATUS_BAD_PAGE);
    } else {
      src = (int64_t)p * kPage + from % kPage;
      dst = (int64_t)q * kPage + j % kPage;
      if (src == dst) src = -1;          // keeps its place
    }
  }
  uint4 c0[kMvRows], c1[kMvRows], e[kMvRows];
  uint32_t sc[kMvRows];
  int64_t s[kMvRows], d[kMvRows];
#pragma unroll
  for (int r = 0; r < kMvRows; ++r) {
    s[r] = __shfl_sync(0xffffffffu, src, r);
    d[r] = __shfl_sync(0xffffffffu, dst, r);
    if (s[r] < 0) continue;
    const uint4* row = a.ckv + s[r] * (kCkv * 2 / 16);
    c0[r] = row[lane];
    c1[r] = row[lane + 32];
    // lanes 0-7: kpe row; lanes 8-15: index key; lane 16: its scale
    if (lane < 8) e[r] = a.kpe[s[r] * 8 + lane];
    if (kIndex) {
      const uint8_t* page = a.index + (s[r] / kPage) * kPageBytes;
      const int pos = (int)(s[r] % kPage);
      if (lane >= 8 && lane < 16) e[r] = *reinterpret_cast<const uint4*>(page + pos * kIdxDim + (lane - 8) * 16);
      if (lane == 16) sc[r] = *reinterpret_cast<const uint32_t*>(page + kPageDataBytes + pos * 4);
    }
  }
#pragma unroll
  for (int r = 0; r < kMvRows; ++r) {
    if (s[r] < 0) continue;
    uint4* row = a.ckv + d[r] * (kCkv * 2 / 16);
    row[lane] = c0[r];
    row[lane + 32] = c1[r];
    if (lane < 8) a.kpe[d[r] * 8 + lane] = e[r];
    if (kIndex) {
      uint8_t* page = a.index + (d[r] / kPage) * kPageBytes;
      const int pos = (int)(d[r] % kPage);
      if (lane >= 8 && lane < 16) *reinterpret_cast<uint4*>(page + pos * kIdxDim + (lane - 8) * 16) = e[r];
      if (lane == 16) *reinterpret_cast<uint32_t*>(page + kPageDataBytes + pos * 4) = sc[r];
    }
  }
}

}  // namespace

cudaError_t launch_cache_evict(const float* weights, int64_t weights_stride, const int32_t* seq_lens, const int32_t* table,
                               int64_t table_stride, const int32_t* new_table, int64_t new_table_stride, void* ckv, void* kpe,
                               void* index, int32_t* new_lens, float* new_weights, int64_t new_weights_stride, int32_t* kept,
                               int64_t kept_stride, int batch, int max_pages, int num_pages, int budget, int keep_first,
                               int keep_last, int32_t* status, cudaStream_t stream) {
  EvictArgs a = {weights, weights_stride, seq_lens, table, table_stride, new_table, new_table_stride, static_cast<uint4*>(ckv),
                 static_cast<uint4*>(kpe), static_cast<uint8_t*>(index), new_lens, new_weights, new_weights_stride, kept,
                 kept_stride, status, batch, max_pages, num_pages, budget, keep_first, keep_last};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)batch);
  cfg.blockDim = dim3(kEvThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, evict_choose_kernel, a);
  if (e != cudaSuccess) return e;
  const int64_t most = (int64_t)max_pages * kPage < budget ? (int64_t)max_pages * kPage : budget;
  const int per = kMvThreads / 32 * kMvRows;
  cfg.gridDim = dim3((unsigned)((most + per - 1) / per), (unsigned)batch);
  cfg.blockDim = dim3(kMvThreads);
  return index ? cudaLaunchKernelEx(&cfg, evict_move_kernel<true>, a) : cudaLaunchKernelEx(&cfg, evict_move_kernel<false>, a);
}

}  // namespace dsa
