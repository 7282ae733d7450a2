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
// of NaNs a NaN sum.  What the two accumulators (m, l) and (m2, l2) are multiplied by when they are added:
__device__ __forceinline__ void join_factors(float& m, float& l, float m2, float l2, float& c, float& f) {
  const float mx = fmaxf(m, m2);
  c = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - mx);
  f = m2 == -INFINITY ? (l2 == 0.f ? 0.f : 1.f) : exp2f(m2 - mx);
  m = mx;
  l = l * c + l2 * f;
}

// 32 threads to a group; kSplit groups share the segments out, each with a running maximum of its
// own, and are then added up, every value by a thread of its own.  A group's loads do not wait for one another (kDepth
// segments of them are in flight), so a request with a hundred segments costs a few trips to L2 when enough groups
// share them.
//   kQuads false: partial results [row][512]; a CTA has one row and 128 of its columns, a thread four of these
//   kQuads true:  partial results [16][512][4] (row blocks of 64: four rows, column, row of the four); a CTA has four
//                 rows and 128 columns, a thread four of these, 32 apart
template <bool kQuads, int kSplit>
__global__ void __launch_bounds__(kSplit * 32)
paged_join_kernel(const PagedArgs a) {
  constexpr int kThreads = kSplit * 32, kDepth = kQuads ? 2 : 5;
  constexpr int kM = kQuads ? 4 : 1;               // rows of a thread
  constexpr int kV = 4 * kM;                       // values of a thread: of row k % kM
  __shared__ float acc_sh[kSplit > 1 ? kSplit : 1][kV][32];      // the groups' values
  __shared__ float sum_sh[kSplit > 1 ? kSplit : 1][kM];         // their rows' sums and maxima
  __shared__ float max_sh[kSplit > 1 ? kSplit : 1][kM];
  const int tid = threadIdx.x, c = tid & 31, grp = tid >> 5;
  const int items = kQuads ? (a.rows + 3) / 4 : a.rows;
  const int b = (int)(blockIdx.x / items), item = (int)(blockIdx.x % items);
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int2 seg = __ldcg(a.segments + b);
  const int x0 = seg.x, n_seg = seg.y;
  // The attention wrote a request of one segment itself; a word that it never wrote (a wait of its that ran out)
  // may say anything.
  if (x0 < 0 || x0 >= a.grid_x || n_seg < 2 || n_seg > a.grid_x - x0) return;
  const int row0 = kQuads ? 4 * item : item, rb = row0 / a.block_rows, br = row0 - rb * a.block_rows;
  const int col = blockIdx.y * 128 + (kQuads ? c : 4 * c);
  const size_t place = kQuads ? ((size_t)(br >> 2) * kCkv + col) * 4 : (size_t)br * kCkv + col;
  float m[kM], l[kM], v[kV];
#pragma unroll
  for (int k = 0; k < kV; ++k) v[k] = 0.f;
#pragma unroll
  for (int k = 0; k < kM; ++k) {
    m[k] = -INFINITY;
    l[k] = 0.f;
  }
  for (int s0 = grp; s0 < n_seg; s0 += kSplit * kDepth) {
    float u[kDepth][kV], m2[kDepth][kM], l2[kDepth][kM];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int s = s0 + d * kSplit;
#pragma unroll
      for (int k = 0; k < kV; ++k) u[d][k] = 0.f;
#pragma unroll
      for (int k = 0; k < kM; ++k) {
        m2[d][k] = -INFINITY;
        l2[d][k] = 0.f;
      }
      if (s < n_seg) {
        const float* p = paged_part(a, a.block_rows, rb, x0 + s, s == 0 ? 1 : 0);
        const float* stat = p + (size_t)a.block_rows * kCkv + br;
#pragma unroll
        for (int q = 0; q < kM; ++q)               // (quads: 32 columns on is 128 floats on)
          *reinterpret_cast<float4*>(u[d] + 4 * q) = __ldcg(reinterpret_cast<const float4*>(p + place + 128 * q));
        if constexpr (kQuads) {
          *reinterpret_cast<float4*>(m2[d]) = __ldcg(reinterpret_cast<const float4*>(stat));
          *reinterpret_cast<float4*>(l2[d]) = __ldcg(reinterpret_cast<const float4*>(stat + a.block_rows));
        } else {
          m2[d][0] = __ldcg(stat);
          l2[d][0] = __ldcg(stat + a.block_rows);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      float f0[kM], f1[kM];
#pragma unroll
      for (int k = 0; k < kM; ++k) join_factors(m[k], l[k], m2[d][k], l2[d][k], f0[k], f1[k]);
#pragma unroll
      for (int k = 0; k < kV; ++k) v[k] = v[k] * f0[k % kM] + u[d][k] * f1[k % kM];
    }
  }
  if (kSplit > 1) {
    if (c == 0) {
#pragma unroll
      for (int k = 0; k < kM; ++k) max_sh[grp][k] = m[k];
    }
    __syncthreads();
    float f[kM];
#pragma unroll
    for (int k = 0; k < kM; ++k) {
      float top = m[k];
#pragma unroll
      for (int s = 0; s < kSplit; ++s) top = fmaxf(top, max_sh[s][k]);
      f[k] = m[k] == -INFINITY ? (l[k] == 0.f ? 0.f : 1.f) : exp2f(m[k] - top);
      m[k] = top;
      if (c == 0) sum_sh[grp][k] = l[k] * f[k];
    }
#pragma unroll
    for (int k = 0; k < kV; ++k) acc_sh[grp][k][c] = v[k] * f[k % kM];
    __syncthreads();
    // in the order of the groups, back into the first group's place
    for (int i = tid; i < 32 * kV; i += kThreads) {
      float t = acc_sh[0][i >> 5][i & 31];
#pragma unroll
      for (int s = 1; s < kSplit; ++s) t += acc_sh[s][i >> 5][i & 31];
      acc_sh[0][i >> 5][i & 31] = t;
    }
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = acc_sh[0][k][c];
#pragma unroll
    for (int k = 0; k < kM; ++k) {
      l[k] = sum_sh[0][k];
#pragma unroll
      for (int s = 1; s < kSplit; ++s) l[k] += sum_sh[s][k];
    }
  }
  float inv[kM];
#pragma unroll
  for (int k = 0; k < kM; ++k) inv[k] = l[k] == 0.f ? 0.f : 1.f / l[k];
  const size_t row = (size_t)b * a.rows + row0;
  if constexpr (kQuads) {
#pragma unroll
    for (int k = 0; k < kV; ++k)
      if (row0 + k % 4 < a.rows) a.out[(row + k % 4) * kCkv + col + 32 * (k / 4)] = __float2bfloat16_rn(v[k] * inv[k % 4]);
  } else {
    const __nv_bfloat162 p0 = __floats2bfloat162_rn(v[0] * inv[0], v[1] * inv[0]);
    const __nv_bfloat162 p1 = __floats2bfloat162_rn(v[2] * inv[0], v[3] * inv[0]);
    *reinterpret_cast<uint2*>(a.out + row * kCkv + col) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
  }
  if (blockIdx.y == 0 && c == 0) {
#pragma unroll
    for (int k = 0; k < kM; ++k)
      if (row0 + k < a.rows) a.lse[row + k] = l[k] == 0.f ? -INFINITY : m[k] + log2f(l[k]);
  }
}

// Four cached tokens per thread, 1024 of one request per CTA; a row's 64 logits of a page are one coalesced 256-byte
// read, and the rows are added in ascending order.  64 x 16384 tokens, 16 rows (67 MB of logits just written, so most of them
// from L2, 4 MB of weights in and out): 16 us.
constexpr int kWeighThreads = 256;
constexpr int kWeighTokens = 4 * kWeighThreads;
__global__ void __launch_bounds__(kWeighThreads)
paged_weights_kernel(const PagedArgs a, const float* weights, int64_t stride, float* out, int64_t out_stride) {
  __shared__ float lse_sh[kWeighThreads];
  const int b = blockIdx.y, tid = threadIdx.x;
  // lengths are older than the attention, which waits for its own predecessor before it lets a successor start
  const int len = paged_len(__ldcg(a.seq_lens + b), a.max_pages);
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
  // About ranges / requests segments to a request.  More groups and more loads in flight shorten a CTA's chain but cost
  // resident CTAs: 16 x 8192 tokens x 64 rows (19 MB of partial results), whole call, with 2 groups and 1 / 2 / 3 / 4
  // segments in flight 51.1 / 47.4 / 51.3 / 53.7 us, with 4 groups 47.7 / 57, with 8 62; one request of 131071 tokens and
  // 16 rows, 16 groups and 3 / 5 / 8 segments 39.7 / 37.0 / 38.0 us; 64 x 16384 tokens, 4 groups 202 us, 1 group 193.
  const int seg = a.grid_x / a.batch;
  if (a.block_rows == 64) {
    const dim3 grid((unsigned)a.batch * (unsigned)((a.rows + 3) / 4), kCkv / 128);
    if (seg > 32) return launch_after(paged_join_kernel<true, 16>, grid, 16 * 32, stream, a);
    if (seg > 2) return launch_after(paged_join_kernel<true, 2>, grid, 2 * 32, stream, a);
    return launch_after(paged_join_kernel<true, 1>, grid, 32, stream, a);
  }
  const dim3 grid((unsigned)a.batch * (unsigned)a.rows, kCkv / 128);
  if (seg > 64) return launch_after(paged_join_kernel<false, 16>, grid, 16 * 32, stream, a);
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
