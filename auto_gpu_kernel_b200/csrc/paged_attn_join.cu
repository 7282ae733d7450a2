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

// One row and kCols of its 512 output columns per CTA, four columns per thread; kSplit groups of threads share the
// segments out among them.  <1, 512> where there are rows enough to fill the machine, <16, 128> where one request's
// hundred segments are the work.
template <int kSplit, int kCols>
__global__ void __launch_bounds__(kSplit * kCols / 4)
paged_join_kernel(const PagedArgs a) {
  constexpr int kGroup = kCols / 4, kThreads = kSplit * kGroup;
  __shared__ long long sums[kThreads / 32];
  __shared__ long long base_sh;
  __shared__ float factor[kPagedMaxRanges];
  __shared__ float red[2][kThreads / 32];
  __shared__ float4 acc_sh[kSplit > 1 ? kSplit : 1][kGroup];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int b = (int)(blockIdx.x / a.rows), r = (int)(blockIdx.x % a.rows);
  // lengths are older than the attention kernel, which waits for its own predecessor before it lets this one start
  int lo, hi;
  long long before;
  const long long total = paged_scan<kThreads>(a.seq_lens, a.batch, a.max_pages, sums, lo, hi, before);
  for (int k = lo; k < hi; ++k) {
    if (k == b) base_sh = before;
    before += paged_tiles(__ldg(a.seq_lens + k), a.max_pages);
  }
  __syncthreads();
  const long long per = (total + a.grid_x - 1) / a.grid_x;
  const long long first = base_sh, last = first + paged_tiles(__ldg(a.seq_lens + b), a.max_pages) - 1;
  const int x0 = (int)(first / per), n_seg = (int)(last / per) - x0 + 1;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (n_seg == 1) return;               // the attention wrote this request itself
  const int rb = r / a.block_rows, br = r - rb * a.block_rows;
  const size_t stat = (size_t)a.block_rows * kCkv + br;
  auto part = [&](int s) { return paged_part(a, a.block_rows, rb, x0 + s, s == 0 ? 1 : 0); };

  float mx = -INFINITY;
  for (int s = tid; s < n_seg; s += kThreads) {
    const float m = __ldcg(part(s) + stat);
    factor[s] = m;
    mx = fmaxf(mx, m);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) red[0][w] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) mx = fmaxf(mx, red[0][i]);
  float sum = 0.f;
  for (int s = tid; s < n_seg; s += kThreads) {
    const float m = factor[s], l = __ldcg(part(s) + stat + a.block_rows);
    // a segment whose logits were all NaN has a NaN sum and no maximum
    const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - mx);
    factor[s] = f;
    sum += f * l;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[1][w] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) sum += red[1][i];

  const int grp = tid / kGroup, c = tid % kGroup;
  const int col = blockIdx.y * kCols + 4 * c;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = grp; s < n_seg; s += kSplit) {
    const float f = factor[s];
    const float4 u = __ldcg(reinterpret_cast<const float4*>(part(s) + (size_t)br * kCkv + col));
    v.x += f * u.x;
    v.y += f * u.y;
    v.z += f * u.z;
    v.w += f * u.w;
  }
  if (kSplit > 1) {
    acc_sh[grp][c] = v;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 1; k < kSplit; ++k) {
      const float4 u = acc_sh[k][c];
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const size_t row = (size_t)b * a.rows + r;
  __nv_bfloat162 p0 = __floats2bfloat162_rn(v.x * inv, v.y * inv), p1 = __floats2bfloat162_rn(v.z * inv, v.w * inv);
  *reinterpret_cast<uint2*>(a.out + row * kCkv + col) =
      make_uint2(*reinterpret_cast<uint32_t*>(&p0), *reinterpret_cast<uint32_t*>(&p1));
  if (blockIdx.y == 0 && tid == 0) a.lse[row] = sum == 0.f ? -INFINITY : mx + log2f(sum);
}

// The same for row blocks of 64, whose partial accumulators lie [column][row]: 64 threads have a row and eight columns
// each, kSplit groups of them share the segments out, each with a running maximum of its own.
constexpr int kJoinRows = 64, kJoinCols = 8;
template <int kSplit>
__global__ void __launch_bounds__(kSplit * kJoinRows)
paged_join_columns_kernel(const PagedArgs a) {
  constexpr int kThreads = kSplit * kJoinRows;
  __shared__ long long sums[kThreads / 32];
  __shared__ long long base_sh;
  __shared__ float acc_sh[kSplit][kJoinCols + 2][kJoinRows];
  const int tid = threadIdx.x, row = tid % kJoinRows, grp = tid / kJoinRows;
  const int blocks = (a.rows + kJoinRows - 1) / kJoinRows;
  const int b = (int)(blockIdx.x / blocks), rb = (int)(blockIdx.x % blocks);
  // lengths are older than the attention kernel, which waits for its own predecessor before it lets this one start
  int lo, hi;
  long long before;
  const long long total = paged_scan<kThreads>(a.seq_lens, a.batch, a.max_pages, sums, lo, hi, before);
  for (int k = lo; k < hi; ++k) {
    if (k == b) base_sh = before;
    before += paged_tiles(__ldg(a.seq_lens + k), a.max_pages);
  }
  __syncthreads();
  const long long per = (total + a.grid_x - 1) / a.grid_x;
  const long long first = base_sh, last = first + paged_tiles(__ldg(a.seq_lens + b), a.max_pages) - 1;
  const int x0 = (int)(first / per), n_seg = (int)(last / per) - x0 + 1;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (n_seg == 1) return;
  const int col = blockIdx.y * kJoinCols;
  float m = -INFINITY, l = 0.f, v[kJoinCols];
#pragma unroll
  for (int k = 0; k < kJoinCols; ++k) v[k] = 0.f;
  // one more partial result (m2, l2, u) into (m, l, v); an empty one has m2 = -inf and l2 = 0, one of NaNs l2 = NaN
  auto add = [&](float m2, float l2, const float (&u)[kJoinCols]) {
    const float mx = fmaxf(m, m2);
    const float c = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - mx);
    const float f = m2 == -INFINITY ? (l2 == 0.f ? 0.f : 1.f) : exp2f(m2 - mx);
    m = mx;
    l = l * c + l2 * f;
#pragma unroll
    for (int k = 0; k < kJoinCols; ++k) v[k] = v[k] * c + u[k] * f;
  };
#pragma unroll 4
  for (int s = grp; s < n_seg; s += kSplit) {
    const float* p = paged_part(a, kJoinRows, rb, x0 + s, s == 0 ? 1 : 0);
    float u[kJoinCols];
#pragma unroll
    for (int k = 0; k < kJoinCols; ++k) u[k] = __ldcg(p + (size_t)(col + k) * kJoinRows + row);
    const float m2 = __ldcg(p + (size_t)kJoinRows * kCkv + row), l2 = __ldcg(p + (size_t)kJoinRows * (kCkv + 1) + row);
    add(m2, l2, u);
  }
  if (kSplit > 1) {
#pragma unroll
    for (int k = 0; k < kJoinCols; ++k) acc_sh[grp][k][row] = v[k];
    acc_sh[grp][kJoinCols][row] = m;
    acc_sh[grp][kJoinCols + 1][row] = l;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll 1
    for (int s = 1; s < kSplit; ++s) {
      float u[kJoinCols];
#pragma unroll
      for (int k = 0; k < kJoinCols; ++k) u[k] = acc_sh[s][k][row];
      add(acc_sh[s][kJoinCols][row], acc_sh[s][kJoinCols + 1][row], u);
    }
  }
  const int r = rb * kJoinRows + row;
  if (r >= a.rows) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t h[kJoinCols / 2];
#pragma unroll
  for (int k = 0; k < kJoinCols / 2; ++k) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k] * inv, v[2 * k + 1] * inv);
    h[k] = *reinterpret_cast<const uint32_t*>(&t);
  }
  *reinterpret_cast<uint4*>(a.out + ((size_t)b * a.rows + r) * kCkv + col) = make_uint4(h[0], h[1], h[2], h[3]);
  if (blockIdx.y == 0) a.lse[(size_t)b * a.rows + r] = l == 0.f ? -INFINITY : m + log2f(l);
}

// One thread per cached token, 256 tokens of one request per CTA; a row's 64 logits of a page are one coalesced
// 256-byte read, and the rows are added in ascending order.
constexpr int kWeighThreads = 256;
__global__ void __launch_bounds__(kWeighThreads)
paged_weights_kernel(const PagedArgs a, const float* weights, int64_t stride, float* out, int64_t out_stride) {
  __shared__ float lse_sh[kWeighThreads];
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int b = blockIdx.y, tid = threadIdx.x;
  const int len = paged_len(__ldg(a.seq_lens + b), a.max_pages);
  if ((int64_t)blockIdx.x * kWeighThreads >= len) return;
  const int pos = blockIdx.x * kWeighThreads + tid;
  const bool held = pos < len;
  const int blocks = (a.rows + a.block_rows - 1) / a.block_rows;
  const float* lg = a.logits +
                    ((size_t)b * a.max_pages + (held ? pos / kPage : 0)) * blocks * (size_t)(a.block_rows * kPage) + pos % kPage;
  float sum = 0.f;
  for (int r0 = 0; r0 < a.rows; r0 += kWeighThreads) {
    const int n = min(kWeighThreads, a.rows - r0);
    __syncthreads();
    if (tid < n) {
      const float v = __ldcg(a.lse + (size_t)b * a.rows + r0 + tid);
      lse_sh[tid] = v == -INFINITY ? INFINITY : v;      // a row that saw nothing gives nothing
    }
    __syncthreads();
    if (held) {
#pragma unroll 16
      for (int r = 0; r < n; ++r) sum += exp2f(__ldcg(lg + (size_t)(r0 + r) * kPage) - lse_sh[r]);
    }
  }
  if (held) out[(int64_t)b * out_stride + pos] = (weights ? weights[(int64_t)b * stride + pos] : 0.f) + sum;
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
  const unsigned rows = (unsigned)a.batch * (unsigned)a.rows;
  if (a.block_rows == kJoinRows) {
    const unsigned n = (unsigned)a.batch * (unsigned)((a.rows + kJoinRows - 1) / kJoinRows);
    // segments per request: about ranges / (requests x row blocks)
    if (n <= 4) return launch_after(paged_join_columns_kernel<16>, dim3(n, kCkv / kJoinCols), 16 * kJoinRows, stream, a);
    return launch_after(paged_join_columns_kernel<4>, dim3(n, kCkv / kJoinCols), 4 * kJoinRows, stream, a);
  }
  if (rows <= 160) return launch_after(paged_join_kernel<16, 128>, dim3(rows, 4), 512, stream, a);
  return launch_after(paged_join_kernel<1, 512>, dim3(rows), 128, stream, a);
}

cudaError_t launch_paged_weights(const PagedArgs& a, const float* weights, int64_t stride, float* out, int64_t out_stride,
                                 cudaStream_t stream) {
  const unsigned chunks = (unsigned)(((int64_t)a.max_pages * kPage + kWeighThreads - 1) / kWeighThreads);
  return launch_after(paged_weights_kernel, dim3(chunks, (unsigned)a.batch), kWeighThreads, stream, a, weights, stride, out,
                      out_stride);
}

}  // namespace dsa
