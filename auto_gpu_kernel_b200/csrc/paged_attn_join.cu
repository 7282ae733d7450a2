// What follows the dense paged attention: the join of the partial results of cut requests, and the accumulated
// attention weight of every cached token.
//
// join:     out[r] = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s over the segments s of the request in order, M the
//           largest m_s; lse[r] = M + log2 of the sum below.  No atomics: every sum has one order.
// weights:  w'[b,pos] = w[b,pos] + sum_r 2^(x[r,pos] - lse[r]), the logits x as the attention left them.
// Both are bound by L2 reads (a segment is 2 KB per row, a cached token 4 B per row).
#include "paged_attn.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace dsa {

namespace {

// A partial result is an accumulator u, its running maximum and its sum; an empty one has maximum -inf and sum 0, one
// of NaNs a NaN sum.
template <int kN>
__device__ __forceinline__ void join_add(float& m, float& l, float (&v)[kN], float m2, float l2, const float (&u)[kN]) {
  const float mx = fmaxf(m, m2);
  const float c = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - mx);
  const float f = m2 == -INFINITY ? (l2 == 0.f ? 0.f : 1.f) : exp2f(m2 - mx);
  m = mx;
  l = l * c + l2 * f;
#pragma unroll
  for (int k = 0; k < kN; ++k) v[k] = v[k] * c + u[k] * f;
}

// Threads share a row's segments out in kSplit groups, each group with a running maximum of its own, and the first
// adds the groups up through shared memory.  A group's loads do not wait for one another (four segments of them are
// in flight), so a request with a hundred segments costs a few trips to L2 when enough groups share them.
//   kColumns false: partial results [row][512]; a CTA has one row and 128 of its columns, a thread four of these
//   kColumns true:  partial results [512][64] (row blocks of 64); a CTA has 64 rows and eight columns, a thread a row
template <bool kColumns, int kSplit>
__global__ void __launch_bounds__(kSplit * (kColumns ? 64 : 32))
paged_join_kernel(const PagedArgs a) {
  constexpr int kGroup = kColumns ? 64 : 32, kN = kColumns ? 8 : 4, kThreads = kSplit * kGroup;
  __shared__ long long sums[kThreads / 32];
  __shared__ PagedSegments seg;
  __shared__ float acc_sh[kSplit > 1 ? kSplit : 1][kN + 2][kGroup];
  const int tid = threadIdx.x, c = tid % kGroup, grp = tid / kGroup;
  const int items = kColumns ? (a.rows + 63) / 64 : a.rows;
  const int b = (int)(blockIdx.x / items), item = (int)(blockIdx.x % items);
  // lengths are older than the attention kernel, which waits for its own predecessor before it lets this one start
  paged_find_segments<kThreads>(a, b, sums, &seg);
  __syncthreads();
  const int x0 = seg.first, n_seg = seg.count;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (n_seg == 1) return;               // the attention wrote this request itself
  const int rb = kColumns ? item : item / a.block_rows, br = kColumns ? c : item - rb * a.block_rows;
  const int col = blockIdx.y * (kColumns ? 8 : 128) + (kColumns ? 0 : 4 * c);
  float m = -INFINITY, l = 0.f, v[kN];
#pragma unroll
  for (int k = 0; k < kN; ++k) v[k] = 0.f;
#pragma unroll 4
  for (int s = grp; s < n_seg; s += kSplit) {
    const float* p = paged_part(a, a.block_rows, rb, x0 + s, s == 0 ? 1 : 0);
    float u[kN];
    if (kColumns) {
#pragma unroll
      for (int k = 0; k < kN; ++k) u[k] = __ldcg(p + (size_t)(col + k) * 64 + br);
    } else {
      const float4 t = __ldcg(reinterpret_cast<const float4*>(p + (size_t)br * kCkv + col));
      u[0] = t.x;
      u[1] = t.y;
      u[2] = t.z;
      u[3] = t.w;
    }
    const float m2 = __ldcg(p + (size_t)a.block_rows * kCkv + br), l2 = __ldcg(p + (size_t)a.block_rows * (kCkv + 1) + br);
    join_add(m, l, v, m2, l2, u);
  }
  if (kSplit > 1) {
#pragma unroll
    for (int k = 0; k < kN; ++k) acc_sh[grp][k][c] = v[k];
    acc_sh[grp][kN][c] = m;
    acc_sh[grp][kN + 1][c] = l;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll 4
    for (int s = 1; s < kSplit; ++s) {
      float u[kN];
#pragma unroll
      for (int k = 0; k < kN; ++k) u[k] = acc_sh[s][k][c];
      join_add(m, l, v, acc_sh[s][kN][c], acc_sh[s][kN + 1][c], u);
    }
  }
  const int r = kColumns ? rb * 64 + c : item;
  if (r >= a.rows) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t h[kN / 2];
#pragma unroll
  for (int k = 0; k < kN / 2; ++k) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k] * inv, v[2 * k + 1] * inv);
    h[k] = *reinterpret_cast<const uint32_t*>(&t);
  }
  const size_t row = (size_t)b * a.rows + r;
  if constexpr (kColumns) *reinterpret_cast<uint4*>(a.out + row * kCkv + col) = make_uint4(h[0], h[1], h[2], h[3]);
  else *reinterpret_cast<uint2*>(a.out + row * kCkv + col) = make_uint2(h[0], h[1]);
  if (blockIdx.y == 0 && (kColumns || c == 0)) a.lse[row] = l == 0.f ? -INFINITY : m + log2f(l);
}

// Four cached tokens per thread, 1024 of one request per CTA; a row's 64 logits of a page are one coalesced 256-byte
// read, and the rows are added in ascending order.
constexpr int kWeighThreads = 256;
constexpr int kWeighTokens = 4 * kWeighThreads;
__global__ void __launch_bounds__(kWeighThreads)
paged_weights_kernel(const PagedArgs a, const float* weights, int64_t stride, float* out, int64_t out_stride) {
  __shared__ float lse_sh[kWeighThreads];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int len = paged_len(__ldg(a.seq_lens + b), a.max_pages);      // older than the attention, as above
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if ((int64_t)blockIdx.x * kWeighTokens >= len) return;
  const int pos = blockIdx.x * kWeighTokens + 4 * tid;
  const bool held = pos < len;
  const int blocks = (a.rows + a.block_rows - 1) / a.block_rows;
  const float* lg = a.logits +
                    ((size_t)b * a.max_pages + (held ? pos / kPage : 0)) * blocks * (size_t)(a.block_rows * kPage) + pos % kPage;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < a.rows; r0 += kWeighThreads) {
    const int n = min(kWeighThreads, a.rows - r0);
    __syncthreads();
    if (tid < n) {
      const float v = __ldcg(a.lse + (size_t)b * a.rows + r0 + tid);
      lse_sh[tid] = v == -INFINITY ? INFINITY : v;      // a row that saw nothing gives nothing
    }
    __syncthreads();
    if (held) {
#pragma unroll 8
      for (int r = 0; r < n; ++r) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(lg + (size_t)(r0 + r) * kPage));
        sum[0] += exp2f(x.x - lse_sh[r]);
        sum[1] += exp2f(x.y - lse_sh[r]);
        sum[2] += exp2f(x.z - lse_sh[r]);
        sum[3] += exp2f(x.w - lse_sh[r]);
      }
    }
  }
  if (!held) return;
  const float* w = weights ? weights + (int64_t)b * stride + pos : nullptr;
  float* dst = out + (int64_t)b * out_stride + pos;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (pos + e < len) dst[e] = (w ? w[e] : 0.f) + sum[e];
}

template <typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

cudaError_t launch_paged_join(const PagedArgs& a, cudaStream_t stream) {
  // about ranges / requests segments to a request; four loads in flight per group are one trip to L2
  const int seg = a.grid_x / a.batch;
  if (a.block_rows == 64) {
    const dim3 grid((unsigned)a.batch * (unsigned)((a.rows + 63) / 64), kCkv / 8);
    if (seg > 16) return launch_after(paged_join_kernel<true, 16>, grid, 16 * 64, stream, a);
    return launch_after(paged_join_kernel<true, 4>, grid, 4 * 64, stream, a);
  }
  const dim3 grid((unsigned)a.batch * (unsigned)a.rows, kCkv / 128);
  if (seg > 16) return launch_after(paged_join_kernel<false, 32>, grid, 32 * 32, stream, a);
  if (seg > 4) return launch_after(paged_join_kernel<false, 4>, grid, 4 * 32, stream, a);
  return launch_after(paged_join_kernel<false, 1>, grid, 32, stream, a);
}

cudaError_t launch_paged_weights(const PagedArgs& a, const float* weights, int64_t stride, float* out, int64_t out_stride,
                                 cudaStream_t stream) {
  const unsigned chunks = (unsigned)(((int64_t)a.max_pages * kPage + kWeighTokens - 1) / kWeighTokens);
  return launch_after(paged_weights_kernel, dim3(chunks, (unsigned)a.batch), kWeighThreads, stream, a, weights, stride, out,
                      out_stride);
}

}  // namespace dsa
