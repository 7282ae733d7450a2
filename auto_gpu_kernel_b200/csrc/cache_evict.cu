// Eviction from the paged caches by accumulated attention weight.
//
//   kept(b) = the first F positions, the last L positions and, of the others, the budget - F - L heaviest (equal weights:
//             the lower position), in ascending order; every position where a request is within the budget
//   token j of the request moves from position kept(b)[j] of its old pages to position j of its new pages.
//
// Two kernels.  The choice is a radix selection over the order-preserving 32-bit keys of the weights (11 + 11 + 10 bits):
// a cluster of CTAs per request, each with a slice of the row as keys in shared memory, adds its three histograms up
// through distributed shared memory; then every thread counts what it keeps of a run of its own, one scan gives the
// places, and the positions are written in order.  The move is bound by memory: 1152 B (+ 132 B of an index key and
// its scale) in and out per kept token; the kept weights go along with it.
#include <cooperative_groups.h>

#include "common.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace dsa {

namespace cg = cooperative_groups;

namespace {

constexpr int kEvThreads = 512;
constexpr int kEvBins = 2048;
constexpr int kEvMine = kEvBins / kEvThreads;
static_assert(kEvMine == 4, "one 16-byte read per thread and histogram");
constexpr int kEvStaged = 40960;      // keys of a slice that fit in shared memory; longer slices are read again

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
  const int n = __ldcg(a.seq_lens + b);
  const int64_t most = (int64_t)a.max_pages * kPage;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}
// -inf and NaN rank lowest, -0 as +0.
__device__ __forceinline__ uint32_t ev_key(float w) {
  return float_to_ordered(w > kScoreFloor ? w + 0.f : kScoreFloor);
}

// Sum of `v` over the threads in front of this one, and over all of them.
template <typename T>
__device__ __forceinline__ T ev_scan(T v, T* sums, T& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  T upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) sums[w] = upto;
  __syncthreads();
  T front = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kEvThreads / 32; ++i) {
    const T u = sums[i];
    if (i < w) front += u;
    total += u;
  }
  return front + upto - v;
}

__global__ void __launch_bounds__(kEvThreads)
evict_choose_kernel(const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ alignas(16) uint32_t hist[2][kEvBins];
  __shared__ uint32_t sums[3][kEvThreads / 32];
  __shared__ uint64_t sums64[kEvThreads / 32];
  __shared__ uint32_t pick[2];
  __shared__ uint64_t slice_counts;         // of this CTA's slice: above the threshold, and (high half) equal to it
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / csize, tid = threadIdx.x;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int n = ev_len(a, b);
  const float* w = a.weights + (int64_t)b * a.weights_stride;
  float* nw = a.new_weights + (int64_t)b * a.new_weights_stride;
  int32_t* kept = a.kept + (int64_t)b * a.kept_stride;
  const int m = n < a.budget ? n : a.budget;
  const int t0 = rank * kEvThreads + tid, step = csize * kEvThreads;
  if (t0 == 0) a.new_lens[b] = m;
  for (int j = m + t0; j < a.budget; j += step) {
    kept[j] = -1;
    nw[j] = 0.f;
  }
  if (n <= a.budget) {
    for (int j = t0; j < n; j += step) kept[j] = j;
    return;
  }
  const int lo = a.keep_first, hi = n - a.keep_last;      // budget < n: the ends do not meet
  const uint32_t want = (uint32_t)(a.budget - a.keep_first - a.keep_last);
  for (int j = t0; j < lo; j += step) kept[j] = j;
  for (int j = hi + t0; j < n; j += step) kept[a.budget - n + j] = j;
  if (want == 0) return;

  // this CTA's slice of the positions in question
  const int per = (hi - lo + csize - 1) / csize;
  const int s0 = min(lo + rank * per, hi), cnt = min(s0 + per, hi) - s0;
  const bool staged = cnt <= kEvStaged;
  // ---- the want-th largest key of positions lo .. hi-1, eleven, eleven and ten bits at a time ----
  uint32_t prefix = 0, rest = want;      // keys that begin with `prefix` are still in question; `rest` of them are kept
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    uint32_t* h = hist[pass & 1];        // the other one may still be read by the cluster
    for (int i = tid; i < kEvBins; i += kEvThreads) h[i] = 0;
    __syncthreads();
    for (int j = tid; j < cnt; j += 8 * kEvThreads) {
      uint32_t k[8];
      if (pass == 0 || !staged) {
        float v[8];                      // eight loads in flight
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = j + e * kEvThreads < cnt ? __ldg(w + s0 + j + e * kEvThreads) : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          k[e] = ev_key(v[e]);
          if (staged && j + e * kEvThreads < cnt) keys[j + e * kEvThreads] = k[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = j + e * kEvThreads < cnt ? keys[j + e * kEvThreads] : 0u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e * kEvThreads < cnt && (pass == 0 || (k[e] >> (shift + bits)) == prefix))
          atomicAdd(&h[(k[e] >> shift) & ((1u << bits) - 1u)], 1u);
    }
    if (csize > 1) cluster.sync();
    else __syncthreads();
    // bins from the top, of all slices: thread t has the kEvMine below 2048 - kEvMine t
    uint32_t c[kEvMine];
    const int top = kEvBins - kEvMine * tid;
    for (int r = 0; r < csize; ++r) {
      const uint4 v = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(h, r) + top - kEvMine);
      if (r == 0) c[0] = c[1] = c[2] = c[3] = 0;
      c[0] += v.w;
      c[1] += v.z;
      c[2] += v.y;
      c[3] += v.x;
    }
    uint32_t all;
    uint32_t above = ev_scan(c[0] + c[1] + c[2] + c[3], sums[pass], all);
#pragma unroll
    for (int k = 0; k < kEvMine; ++k) {
      if (above < rest && above + c[k] >= rest) {
        pick[0] = top - 1 - k;
        pick[1] = rest - above;
      }
      above += c[k];
    }
    __syncthreads();
    prefix = (prefix << bits) | pick[0];
    rest = pick[1];
    __syncthreads();                     // before the next pass picks
  }
  // ---- keys above `prefix` are kept, and the first `rest` that equal it ----
  // thread t has the run [t * run, (t + 1) * run) of the slice; an odd run keeps the banks apart
  const int run = ((cnt + kEvThreads - 1) / kEvThreads) | 1;
  const int j0 = min(tid * run, cnt), j1 = min(j0 + run, cnt);
  uint64_t mine = 0, all64;
  for (int j = j0; j < j1; ++j) {
    const uint32_t k = staged ? keys[j] : ev_key(w[s0 + j]);
    mine += k > prefix ? 1ull : k == prefix ? 1ull << 32 : 0ull;
  }
  mine = ev_scan(mine, sums64, all64);
  if (csize > 1) {
    if (tid == 0) slice_counts = all64;
    cluster.sync();
    for (int r = 0; r < rank; ++r) mine += *cluster.map_shared_rank(&slice_counts, r);
  }
  uint32_t gt = (uint32_t)mine, eq = (uint32_t)(mine >> 32);
  for (int j = j0; j < j1; ++j) {
    const uint32_t k = staged ? keys[j] : ev_key(w[s0 + j]);
    if (k > prefix || (k == prefix && eq < rest)) kept[(uint32_t)lo + gt + min(eq, rest)] = s0 + j;
    gt += k > prefix;
    eq += k == prefix;
  }
  if (csize > 1) cluster.sync();         // nobody leaves while its counts may be read
}

// CTAs per request: up to four while the SMs hold them at once and a slice stays 4096 keys, eight while it stays 16384 (a
// cluster of eight needs its SMs inside one GPC, and fewer fit); less is not worth the cluster's barriers.  Whole call with
// 512 or 1024 kept tokens, 1 / 2 / 4 CTAs: 1 x 4096 tokens 12.3 / 14.3 / 14.4 us, 4 x 8192 16.4 / 14.9 / 16.4, 64 x 16384
// 36.4 / 32.3 / 34.9, 128 x 8192 42.1 / 44.4 / 60.1, 16 x 32768 32.8 / 24.6 / 21.1, 32 x 32768 39.9 / 30.7 / 26.7; 4 / 8 CTAs:
// 8 x 65536 26.7 / 26.6, 14 x 131072 43.1 / 36.9, 1 x 1000000 307 / 169.
int ev_cluster(int batch, int64_t longest, int sms) {
  int c = 1;
  while (c < 8 && longest / (2 * c) >= (c < 4 ? 4096 : 16384) && (int64_t)batch * 2 * c <= (c < 4 ? sms * 9 / 10 : sms * 8 / 10))
    c *= 2;
  return c;
}

// One warp per four kept tokens: their slots are looked up together, then one row after the other moves.  More rows in
// flight per warp cost registers and with them warps, and were slower (32 x 8192 rows with index keys: one row at a time
// 117 us = 5.7 TB/s, two 125, four 156, eight 191 us; one lookup for every row 126 us).
constexpr int kMvThreads = 256;
constexpr int kMvRows = 4;

template <bool kIndex>
__global__ void __launch_bounds__(kMvThreads)
evict_move_kernel(const EvictArgs a) {
  const int lane = threadIdx.x & 31, b = blockIdx.y;
  const int j0 = (blockIdx.x * (kMvThreads / 32) + (threadIdx.x >> 5)) * kMvRows;
  const int n = ev_len(a, b), m = n < a.budget ? n : a.budget;    // older than the choice, which waits for its predecessor
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (j0 >= m) return;
  int64_t src = -1, dst = -1;              // lane r: row r
  if (lane < kMvRows && j0 + lane < m) {
    const int j = j0 + lane;
    const int from = __ldcg(a.kept + (int64_t)b * a.kept_stride + j);
    // (a caller whose outputs overlap has written over the choice: nothing out of bounds is read for it)
    const bool known = from >= 0 && from < n;
    if (known) a.new_weights[(int64_t)b * a.new_weights_stride + j] = __ldg(a.weights + (int64_t)b * a.weights_stride + from);
    const int p = known ? __ldg(a.table + (int64_t)b * a.table_stride + from / kPage) : -1;
    const int q = __ldg(a.new_table + (int64_t)b * a.new_table_stride + j / kPage);
    if (p < 0 || p >= a.num_pages || q < 0 || q >= a.num_pages) {
      raise_status(a.status, DSA_STATUS_BAD_PAGE);
    } else {
      src = (int64_t)p * kPage + from % kPage;
      dst = (int64_t)q * kPage + j % kPage;
      if (src == dst) src = -1;            // keeps its place
    }
  }
#pragma unroll 1
  for (int r = 0; r < kMvRows; ++r) {
    const int64_t s = __shfl_sync(0xffffffffu, src, r), d = __shfl_sync(0xffffffffu, dst, r);
    if (s < 0) continue;
    const uint4* from = a.ckv + s * (kCkv * 2 / 16);
    uint4* to = a.ckv + d * (kCkv * 2 / 16);
    const uint4 c0 = from[lane], c1 = from[lane + 32];
    // lanes 0-7: kpe row; lanes 8-15: index key; lane 16: its scale
    uint4 e = make_uint4(0, 0, 0, 0);
    if (lane < 8) e = a.kpe[s * 8 + lane];
    if (kIndex) {
      const uint8_t* page = a.index + (s / kPage) * kPageBytes;
      const int pos = (int)(s % kPage);
      if (lane >= 8 && lane < 16) e = *reinterpret_cast<const uint4*>(page + pos * kIdxDim + (lane - 8) * 16);
      if (lane == 16) e.x = *reinterpret_cast<const uint32_t*>(page + kPageDataBytes + pos * 4);
    }
    to[lane] = c0;
    to[lane + 32] = c1;
    if (lane < 8) a.kpe[d * 8 + lane] = e;
    if (kIndex) {
      uint8_t* page = a.index + (d / kPage) * kPageBytes;
      const int pos = (int)(d % kPage);
      if (lane >= 8 && lane < 16) *reinterpret_cast<uint4*>(page + pos * kIdxDim + (lane - 8) * 16) = e;
      if (lane == 16) *reinterpret_cast<uint32_t*>(page + kPageDataBytes + pos * 4) = e.x;
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
  const int64_t longest = (int64_t)max_pages * kPage;
  const int csize = ev_cluster(batch, longest, sm_count());
  const int64_t slice = (longest + csize - 1) / csize;
  const size_t staged = (size_t)(slice < kEvStaged ? slice : kEvStaged) * sizeof(uint32_t);
  static std::atomic<uint64_t> opted{0};
  cudaError_t e = opt_in_dynamic_smem(reinterpret_cast<const void*>(evict_choose_kernel), kEvStaged * sizeof(uint32_t), opted);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * csize));
  cfg.blockDim = dim3(kEvThreads);
  cfg.dynamicSmemBytes = staged;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)csize;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = csize > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, evict_choose_kernel, a);
  if (e != cudaSuccess) return e;
  const int64_t most = longest < budget ? longest : budget;
  const int per = kMvThreads / 32 * kMvRows;
  cfg.gridDim = dim3((unsigned)((most + per - 1) / per), (unsigned)batch);
  cfg.blockDim = dim3(kMvThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return index ? cudaLaunchKernelEx(&cfg, evict_move_kernel<true>, a) : cudaLaunchKernelEx(&cfg, evict_move_kernel<false>, a);
}

}  // namespace dsa
