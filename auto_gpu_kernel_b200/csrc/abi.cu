// extern "C" boundary of libdsa_b200.so: argument checks on the host, then kernel launches on the
// caller's stream.  No allocation, no synchronisation, no exceptions cross this boundary.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "common.cuh"
#include "paged_attn.cuh"
#include "tmap.cuh"

namespace dsa {
cudaError_t launch_indexer_score_simt(const void*, const void*, const float*, const int32_t*,
                                      const int32_t*, int64_t, float*, int64_t, int, int, int,
                                      int32_t*, cudaStream_t);
cudaError_t launch_indexer_score_tc(const void*, const void*, const float*, const int32_t*,
                                    const int32_t*, int64_t, float*, int64_t, int, int, int, int,
                                    uint32_t*, uint32_t*, int32_t*, cudaStream_t);
cudaError_t launch_topk_select_hist(const float*, int64_t, const int32_t*, const int32_t*, int64_t,
                                    int32_t*, int64_t, int, int, uint32_t*, const RowSend*, int32_t*,
                                    cudaStream_t);
bool topk_select_hist_supports(int batch, int max_pages);
cudaError_t launch_topk_select(const float*, int64_t, const int32_t*, const int32_t*, int64_t,
                               int32_t*, int64_t, int, int, uint32_t*, int32_t*, cudaStream_t);
cudaError_t launch_sparse_attn_simt(const void*, const void*, const void*, const void*,
                                    const int32_t*, int64_t, float, void*, float*, int, int, int64_t,
                                    int, void*, int32_t*, cudaStream_t);
cudaError_t launch_sparse_attn_tc(const void*, const void*, const void*, const void*,
                                  const int32_t*, int64_t, float, void*, float*, int, int, int64_t,
                                  void*, int32_t*, cudaStream_t);
size_t at_tc_workspace_bytes_auto(int tokens, int topk);
cudaError_t launch_index_rows_exchange(int32_t*, const RowSend&, int, int, int64_t, int, uint64_t, int32_t*,
                                       cudaStream_t);
cudaError_t launch_sparse_attn_mma(const void*, const void*, const void*, const void*,
                                   const int32_t*, int64_t, float, void*, float*, int, int, int64_t,
                                   void*, int32_t*, cudaStream_t);
int att_pick_splits(int tokens, int topk);
cudaError_t launch_indexer_score_prefill(const void*, const void*, const float*, const int32_t*,
                                         const int32_t*, float*, int64_t, int, int, int, int,
                                         int32_t*, cudaStream_t);
constexpr int kPrefillMinRows = 16;   // below this the per-row streaming kernel is as fast
cudaError_t launch_index_cache_write(const void*, int, int64_t, const int32_t*, void*, int, int64_t,
                                     int32_t*, cudaStream_t);
cudaError_t launch_kv_cache_append(const void*, int64_t, const void*, int64_t, const int32_t*, void*,
                                   void*, int, int64_t, int32_t*, cudaStream_t);
size_t att_workspace_bytes(int tokens, int splits);
cudaError_t launch_paged_attn_mma(const PagedArgs&, const void*, const void*, cudaStream_t);
cudaError_t launch_paged_attn_tc(const PagedArgs&, const void*, const void*, cudaStream_t);
cudaError_t launch_paged_join(const PagedArgs&, cudaStream_t);
cudaError_t launch_paged_weights(const PagedArgs&, const float*, int64_t, float*, int64_t, cudaStream_t);
cudaError_t launch_cache_evict(const float*, int64_t, const int32_t*, const int32_t*, int64_t, const int32_t*, int64_t, void*,
                               void*, void*, int32_t*, float*, int64_t, int32_t*, int64_t, int, int, int, int, int, int,
                               int32_t*, cudaStream_t);
cudaError_t launch_rotary_append(const void*, int64_t, int64_t, const void*, int64_t, const void*, int64_t, const int32_t*,
                                 int64_t, const float*, uint64_t, int, const int32_t*, void*, void*, void*, int, int, int64_t,
                                 int32_t*, cudaStream_t);
}  // namespace dsa

namespace {
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Memory of an argument: `rows` rows of `row` bytes, `stride` bytes apart.
struct Region {
  const void* at;
  size_t row, stride, rows;
};
// Whether two arguments may share a byte.  Exact for rows of one pitch (column ranges of one buffer are apart although their
// spans meet); for others it goes by the spans.
inline bool meet(const Region& a, const Region& b) {
  if (a.at == nullptr || b.at == nullptr || a.row == 0 || b.row == 0 || a.rows == 0 || b.rows == 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.at), pb = reinterpret_cast<uintptr_t>(b.at);
  if (pa + (a.rows - 1) * a.stride + a.row <= pb || pb + (b.rows - 1) * b.stride + b.row <= pa) return false;
  const size_t pitch = a.rows > 1 ? a.stride : b.stride;
  if (pitch == 0 || (a.rows > 1 && b.rows > 1 && a.stride != b.stride)) return true;
  const Region &lo = pa <= pb ? a : b, &hi = pa <= pb ? b : a;
  const size_t off = (pa <= pb ? pb - pa : pa - pb) % pitch;
  return off < lo.row || off + hi.row > pitch;
}
// Whether one of the first `outputs` regions meets any other one.
template <int kN>
inline bool outputs_meet(const Region (&r)[kN], int outputs) {
  for (int i = 0; i < outputs; ++i)
    for (int j = i + 1; j < kN; ++j)
      if (meet(r[i], r[j])) return true;
  return false;
}
// score rows are padded to a multiple of 128 tokens so a 2-page tile never crosses rows
inline int64_t score_row_stride(int max_pages) { return ((int64_t)max_pages * dsa::kPage + 127) / 128 * 128; }
}  // namespace

extern "C" {

int dsa_b200_version(void) { return DSA_B200_ABI_VERSION; }

const char* dsa_b200_error_string(int code) {
  switch (code) {
    case DSA_OK: return "ok";
    case DSA_ERR_NULL_POINTER: return "dsa_b200: null pointer argument";
    case DSA_ERR_BAD_SHAPE: return "dsa_b200: unsupported or inconsistent shape";
    case DSA_ERR_WORKSPACE_TOO_SMALL: return "dsa_b200: workspace too small";
    case DSA_ERR_MISALIGNED: return "dsa_b200: pointer or stride not 16-byte aligned";
    case DSA_ERR_UNSUPPORTED: return "dsa_b200: variant not available";
    case DSA_ERR_SCRATCH_TOO_SMALL:
      return "dsa_b200: batch x context exceeds the built-in scratch of dsa_indexer_topk_noalloc";
    case DSA_ERR_OVERLAP: return "dsa_b200: outputs must not overlap the inputs or one another";
    default: break;
  }
  if (code > 0) return cudaGetErrorString(static_cast<cudaError_t>(code));
  return "dsa_b200: unknown error code";
}

// [ per request: max of the ordered score keys, max of their complements | per-request score
//   histograms | fp32 score rows ]
// The first two regions must be zero between calls (the kernels put back what they use), so each
// has one fixed size for every shape: no call's score rows ever land on another call's words.
constexpr size_t kMinmaxRegionBytes = 65536 * 2 * sizeof(uint32_t);   // batch <= 65535
constexpr size_t kScoreRowsOffset = kMinmaxRegionBytes + dsa::kHistRegionBytes;
size_t dsa_indexer_workspace_bytes(int batch, int max_pages) {
  if (batch <= 0 || max_pages <= 0) return 256;
  return kScoreRowsOffset + round256((size_t)batch * score_row_stride(max_pages) * sizeof(float));
}

// How dsa_indexer_topk scores and selects long rows (decode shapes, batch <= 1024):
//   "hist"   (default) the scorer also builds every request's score histogram; the selection
//            kernel starts from it (boundary bin, one counting and one writing sweep);
//   "minmax" the scorer hands over each row's min / max, the selection builds its own histogram
//            over the linear map of that range (also what larger batches and the shared-pages
//            scorer use).
// DSA_INDEXER_PATH in the environment picks one; read on every call so that a test can compare
// the paths in one process.
enum IndexerPath { kPathHist, kPathMinmax };
static IndexerPath indexer_path() {
  const char* e = getenv("DSA_INDEXER_PATH");
  return (e != nullptr && e[0] == 'm') ? kPathMinmax : kPathHist;
}

static int scores_impl(const void* q_fp8, const void* k_cache, const float* weights,
                       const int32_t* seq_lens, const int32_t* block_table,
                       int64_t block_table_stride, float* scores, int64_t score_stride, int batch,
                       int num_pages, int max_pages, int variant, int skip_short, uint32_t* minmax,
                       uint32_t* ghist, int32_t* status_dev, void* stream) {
  if (batch == 0) return DSA_OK;
  if (!q_fp8 || !k_cache || !weights || !seq_lens || !block_table || !scores)
    return DSA_ERR_NULL_POINTER;
  if (batch < 0 || batch > 65535 || num_pages <= 0 || max_pages <= 0 || block_table_stride < 0 ||
      score_stride < (int64_t)max_pages * dsa::kPage)
    return DSA_ERR_BAD_SHAPE;
  if (!aligned16(q_fp8) || !aligned16(k_cache) || !aligned16(scores) || (score_stride & 3))
    return DSA_ERR_MISALIGNED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (variant == 1) {
    e = dsa::launch_indexer_score_simt(q_fp8, k_cache, weights, seq_lens, block_table,
                                       block_table_stride, scores, score_stride, batch, num_pages,
                                       max_pages, status_dev, s);
  } else if (variant == 0 && block_table_stride == 0 && batch >= dsa::kPrefillMinRows) {
    // every row reads the same pages (chunked prefill): four rows share each tcgen05.mma
    e = dsa::launch_indexer_score_prefill(q_fp8, k_cache, weights, seq_lens, block_table, scores,
                                          score_stride, batch, num_pages, max_pages, skip_short,
                                          status_dev, s);
  } else if (variant == 0 || variant == 2) {
    e = dsa::launch_indexer_score_tc(q_fp8, k_cache, weights, seq_lens, block_table,
                                     block_table_stride, scores, score_stride, batch, num_pages,
                                     max_pages, skip_short, minmax, ghist, status_dev, s);
  } else {
    return DSA_ERR_UNSUPPORTED;
  }
  return static_cast<int>(e);
}

int dsa_indexer_scores(const void* q_fp8, const void* k_cache, const float* weights,
                       const int32_t* seq_lens, const int32_t* block_table,
                       int64_t block_table_stride, float* scores, int64_t score_stride, int batch,
                       int num_pages, int max_pages, int variant, int32_t* status_dev,
                       void* stream) {
  return scores_impl(q_fp8, k_cache, weights, seq_lens, block_table, block_table_stride, scores,
                     score_stride, batch, num_pages, max_pages, variant, 0, nullptr, nullptr, status_dev,
                     stream);
}

int dsa_topk_select(const float* scores, int64_t score_stride, const int32_t* seq_lens,
                    const int32_t* block_table, int64_t block_table_stride, int32_t* topk_out,
                    int64_t topk_stride, int batch, int max_pages, int32_t* status_dev,
                    void* stream) {
  if (batch == 0) return DSA_OK;
  if (!scores || !seq_lens || !block_table || !topk_out) return DSA_ERR_NULL_POINTER;
  if (batch < 0 || max_pages <= 0 || topk_stride < dsa::kTopK || block_table_stride < 0)
    return DSA_ERR_BAD_SHAPE;
  return static_cast<int>(dsa::launch_topk_select(scores, score_stride, seq_lens, block_table,
                                                  block_table_stride, topk_out, topk_stride, batch,
                                                  max_pages, nullptr, status_dev,
                                                  static_cast<cudaStream_t>(stream)));
}

// `send` (may be null): where finished rows go in a head-sharded layer.  *sent tells whether the
// selection kernel has sent them itself (the histogram path) or the caller still has to.
static int indexer_topk_impl(const void* q_fp8, const void* k_cache, const float* weights,
                             const int32_t* seq_lens, const int32_t* block_table,
                             int64_t block_table_stride, int32_t* topk_out, int64_t topk_stride, int batch,
                             int num_pages, int max_pages, void* workspace, size_t workspace_bytes,
                             int32_t* status_dev, void* stream, const dsa::RowSend* send, bool* sent) {
  if (sent) *sent = false;
  if (batch == 0) return DSA_OK;
  if (!workspace) return DSA_ERR_NULL_POINTER;
  if (workspace_bytes < dsa_indexer_workspace_bytes(batch, max_pages))
    return DSA_ERR_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return DSA_ERR_MISALIGNED;
  if (batch > 65535) return DSA_ERR_BAD_SHAPE;
  float* scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + kScoreRowsOffset);
  const int64_t stride = score_row_stride(max_pages);
  // The streaming scorer leaves every row's min / max in front of the score rows (the words start
  // at zero and the selection puts them back to zero); the shared-pages scorer does not.
  const bool shared_pages = block_table_stride == 0 && batch >= dsa::kPrefillMinRows;
  uint32_t* minmax = shared_pages ? nullptr : static_cast<uint32_t*>(workspace);
  const bool long_rows = (int64_t)max_pages * dsa::kPage > dsa::kTopK;
  const IndexerPath path = indexer_path();
  uint32_t* ghist = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kMinmaxRegionBytes);
  // rows of at most 2048 tokens are emitted whole by the selection: their scores are skipped, and
  // when no row can be longer (max_pages <= 32) the scorer is not launched at all (the reference's
  // GPU dispatch takes the same shortcut from the shape alone, indexer_fused.py:358-380)
  if (long_rows && !shared_pages && path != kPathMinmax &&
      dsa::topk_select_hist_supports(batch, max_pages)) {
    if (!topk_out) return DSA_ERR_NULL_POINTER;
    if (topk_stride < dsa::kTopK) return DSA_ERR_BAD_SHAPE;
    int rc = scores_impl(q_fp8, k_cache, weights, seq_lens, block_table, block_table_stride, scores,
                         stride, batch, num_pages, max_pages, 0, 1, nullptr, ghist, status_dev, stream);
    if (rc != DSA_OK) return rc;
    if (sent) *sent = send != nullptr;
    return static_cast<int>(dsa::launch_topk_select_hist(
        scores, stride, seq_lens, block_table, block_table_stride, topk_out, topk_stride, batch,
        max_pages, ghist, send, status_dev, static_cast<cudaStream_t>(stream)));
  }
  if (long_rows) {
    int rc = scores_impl(q_fp8, k_cache, weights, seq_lens, block_table, block_table_stride, scores,
                         stride, batch, num_pages, max_pages, 0, 1, minmax, nullptr, status_dev, stream);
    if (rc != DSA_OK) return rc;
  } else if (!q_fp8 || !k_cache || !weights || !seq_lens || !block_table) {
    return DSA_ERR_NULL_POINTER;
  }
  if (!seq_lens || !block_table || !topk_out) return DSA_ERR_NULL_POINTER;
  if (max_pages <= 0 || topk_stride < dsa::kTopK || block_table_stride < 0) return DSA_ERR_BAD_SHAPE;
  return static_cast<int>(dsa::launch_topk_select(scores, stride, seq_lens, block_table,
                                                  block_table_stride, topk_out, topk_stride, batch,
                                                  max_pages, minmax, status_dev,
                                                  static_cast<cudaStream_t>(stream)));
}

int dsa_indexer_topk(const void* q_fp8, const void* k_cache, const float* weights,
                     const int32_t* seq_lens, const int32_t* block_table,
                     int64_t block_table_stride, int32_t* topk_out, int64_t topk_stride, int batch,
                     int num_pages, int max_pages, void* workspace, size_t workspace_bytes,
                     int32_t* status_dev, void* stream) {
  return indexer_topk_impl(q_fp8, k_cache, weights, seq_lens, block_table, block_table_stride, topk_out,
                           topk_stride, batch, num_pages, max_pages, workspace, workspace_bytes,
                           status_dev, stream, nullptr, nullptr);
}

static int fill_row_send(dsa::RowSend* xs, void* const* peer_stage, int world, int rank, int row_offset,
                         int row_width, uint32_t epoch) {
  if (!peer_stage) return DSA_ERR_NULL_POINTER;
  if (world < 1 || world > dsa::kRowSendMaxWorld || rank < 0 || rank >= world || row_offset < 0 ||
      row_width <= 0 || row_width % 2 != 0 || epoch == 0)
    return DSA_ERR_BAD_SHAPE;
  *xs = dsa::RowSend{};
  for (int p = 0; p < world; ++p) {
    if (!peer_stage[p]) return DSA_ERR_NULL_POINTER;
    if (!aligned16(peer_stage[p])) return DSA_ERR_MISALIGNED;
    xs->stage[p] = static_cast<uint2*>(peer_stage[p]);
  }
  xs->world = world;
  xs->rank = rank;
  xs->row_offset = row_offset;
  xs->row_width = row_width;
  xs->epoch = epoch;
  return DSA_OK;
}

int dsa_indexer_topk_send(const void* q_fp8, const void* k_cache, const float* weights,
                          const int32_t* seq_lens, const int32_t* block_table,
                          int64_t block_table_stride, int32_t* topk_out, int64_t topk_stride, int batch,
                          int num_pages, int max_pages, void* workspace, size_t workspace_bytes,
                          void* const* peer_stage, int world, int rank, int row_offset, uint32_t epoch,
                          int32_t* status_dev, void* stream) {
  dsa::RowSend xs;
  int rc = fill_row_send(&xs, peer_stage, world, rank, row_offset, dsa::kTopK, epoch);
  if (rc != DSA_OK) return rc;
  if (topk_stride % 2 != 0 || (reinterpret_cast<uintptr_t>(topk_out) & 7u)) return DSA_ERR_MISALIGNED;
  bool sent = false;
  rc = indexer_topk_impl(q_fp8, k_cache, weights, seq_lens, block_table, block_table_stride, topk_out,
                         topk_stride, batch, num_pages, max_pages, workspace, workspace_bytes, status_dev,
                         stream, &xs, &sent);
  if (rc != DSA_OK || sent || batch == 0 || world == 1) return rc;
  // the other selection kernels do not send: a push-only pass over the finished rows
  int32_t* base = topk_out - (int64_t)row_offset * topk_stride;   // row i of the exchange = base + i * stride
  return static_cast<int>(dsa::launch_index_rows_exchange(base, xs, batch, row_offset + batch, topk_stride, 1,
                                                          1, status_dev, static_cast<cudaStream_t>(stream)));
}

size_t dsa_sparse_attn_workspace_bytes(int tokens, int heads, int topk) {
  if (tokens <= 0 || heads != dsa::kHeads || topk <= 0) return 256;
  size_t a = dsa::att_workspace_bytes(tokens, dsa::att_pick_splits(tokens, topk));
  size_t b = dsa::at_tc_workspace_bytes_auto(tokens, topk);
  return round256(a > b ? a : b);
}

static int attn_impl(const void* q_nope, const void* q_pe, const void* ckv, const void* kpe,
                     const int32_t* sparse_indices, int64_t index_stride, float sm_scale, void* out,
                     float* lse, int tokens, int heads, int topk, int64_t num_slots, void* workspace,
                     size_t workspace_bytes, int32_t* status_dev, void* stream, int variant) {
  if (tokens == 0) return DSA_OK;
  if (!q_nope || !q_pe || !ckv || !kpe || !sparse_indices || !out || !lse || !workspace)
    return DSA_ERR_NULL_POINTER;
  if (tokens < 0 || heads != dsa::kHeads || topk <= 0 || num_slots <= 0 || index_stride < topk)
    return DSA_ERR_BAD_SHAPE;
  if (!aligned16(q_nope) || !aligned16(q_pe) || !aligned16(ckv) || !aligned16(kpe) ||
      !aligned16(out) || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return DSA_ERR_MISALIGNED;
  if (workspace_bytes < dsa_sparse_attn_workspace_bytes(tokens, heads, topk))
    return DSA_ERR_WORKSPACE_TOO_SMALL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (variant == 1) {
    const int splits = dsa::att_pick_splits(tokens, topk);
    return static_cast<int>(dsa::launch_sparse_attn_simt(q_nope, q_pe, ckv, kpe, sparse_indices,
                                                         index_stride, sm_scale, out, lse, tokens,
                                                         topk, num_slots, splits, workspace,
                                                         status_dev, s));
  }
  if (variant == 2) {
    return static_cast<int>(dsa::launch_sparse_attn_tc(q_nope, q_pe, ckv, kpe, sparse_indices,
                                                       index_stride, sm_scale, out, lse, tokens,
                                                       topk, num_slots, workspace, status_dev, s));
  }
  return static_cast<int>(dsa::launch_sparse_attn_mma(q_nope, q_pe, ckv, kpe, sparse_indices,
                                                      index_stride, sm_scale, out, lse, tokens, topk,
                                                      num_slots, workspace, status_dev, s));
}

int dsa_sparse_attn(const void* q_nope, const void* q_pe, const void* ckv, const void* kpe,
                    const int32_t* sparse_indices, int64_t index_stride, float sm_scale, void* out,
                    float* lse, int tokens, int heads, int topk, int64_t num_slots, void* workspace,
                    size_t workspace_bytes, int32_t* status_dev, void* stream) {
  return attn_impl(q_nope, q_pe, ckv, kpe, sparse_indices, index_stride, sm_scale, out, lse, tokens,
                   heads, topk, num_slots, workspace, workspace_bytes, status_dev, stream, 0);
}

int dsa_sparse_attn_cuda_core(const void* q_nope, const void* q_pe, const void* ckv,
                              const void* kpe, const int32_t* sparse_indices, int64_t index_stride,
                              float sm_scale, void* out, float* lse, int tokens, int heads, int topk,
                              int64_t num_slots, void* workspace, size_t workspace_bytes,
                              int32_t* status_dev, void* stream) {
  return attn_impl(q_nope, q_pe, ckv, kpe, sparse_indices, index_stride, sm_scale, out, lse, tokens,
                   heads, topk, num_slots, workspace, workspace_bytes, status_dev, stream, 1);
}

int dsa_sparse_attn_tcgen05(const void* q_nope, const void* q_pe, const void* ckv, const void* kpe,
                            const int32_t* sparse_indices, int64_t index_stride, float sm_scale,
                            void* out, float* lse, int tokens, int heads, int topk,
                            int64_t num_slots, void* workspace, size_t workspace_bytes,
                            int32_t* status_dev, void* stream) {
  return attn_impl(q_nope, q_pe, ckv, kpe, sparse_indices, index_stride, sm_scale, out, lse, tokens,
                   heads, topk, num_slots, workspace, workspace_bytes, status_dev, stream, 2);
}

// ---- buffers that the GPUs of one host can address in each other's memory (CUDA IPC) ----------
int dsa_peer_slab_create(size_t bytes, void** ptr, void* handle64) {
  if (!ptr || !handle64 || bytes == 0) return DSA_ERR_NULL_POINTER;
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, bytes);
  if (e != cudaSuccess) return static_cast<int>(e);
  e = cudaMemset(p, 0, bytes);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  cudaIpcMemHandle_t h;
  if (e == cudaSuccess) e = cudaIpcGetMemHandle(&h, p);
  if (e != cudaSuccess) {
    cudaFree(p);
    return static_cast<int>(e);
  }
  static_assert(sizeof(cudaIpcMemHandle_t) == 64, "handle size");
  memcpy(handle64, &h, 64);
  *ptr = p;
  return DSA_OK;
}

int dsa_peer_slab_open(const void* handle64, void** ptr) {
  if (!ptr || !handle64) return DSA_ERR_NULL_POINTER;
  cudaIpcMemHandle_t h;
  memcpy(&h, handle64, 64);
  // opened with the CALLER's device current: peer access from it to the owner is enabled with it
  return static_cast<int>(cudaIpcOpenMemHandle(ptr, h, cudaIpcMemLazyEnablePeerAccess));
}

int dsa_peer_slab_close(void* ptr) {
  return ptr ? static_cast<int>(cudaIpcCloseMemHandle(ptr)) : DSA_OK;
}

int dsa_peer_slab_destroy(void* ptr) { return ptr ? static_cast<int>(cudaFree(ptr)) : DSA_OK; }

int dsa_index_rows_exchange(int32_t* rows, void* const* peer_stage, int world, int rank, int rows_local,
                            int row_offset, int rows_total, int64_t row_stride, int row_width,
                            uint32_t epoch, int mode, uint64_t wait_limit_ns, int32_t* status_dev,
                            void* stream) {
  if (!rows) return DSA_ERR_NULL_POINTER;
  dsa::RowSend xs;
  int rc = fill_row_send(&xs, peer_stage, world, rank, row_offset, row_width, epoch);
  if (rc != DSA_OK) return rc;
  if (rows_local < 0 || rows_total < row_offset + rows_local || row_stride < row_width ||
      row_stride % 2 != 0 || mode < 1 || mode > 3 || wait_limit_ns == 0 ||
      wait_limit_ns > 10000000000ull)
    return DSA_ERR_BAD_SHAPE;
  if (reinterpret_cast<uintptr_t>(rows) & 7u) return DSA_ERR_MISALIGNED;
  if (rows_total == 0) return DSA_OK;
  return static_cast<int>(dsa::launch_index_rows_exchange(rows, xs, rows_local, rows_total, row_stride,
                                                          mode, wait_limit_ns, status_dev,
                                                          static_cast<cudaStream_t>(stream)));
}

int dsa_index_cache_write(const void* keys, int key_dtype, int64_t key_stride, const int32_t* slots,
                          void* k_cache, int tokens, int num_pages, int32_t* status_dev,
                          void* stream) {
  if (tokens == 0) return DSA_OK;
  if (!keys || !slots || !k_cache) return DSA_ERR_NULL_POINTER;
  if (tokens < 0 || num_pages <= 0 || key_stride < dsa::kIdxDim || (key_dtype != 0 && key_dtype != 1))
    return DSA_ERR_BAD_SHAPE;
  const int64_t elem = key_dtype == 0 ? 4 : 2;
  if (!aligned16(keys) || (key_stride * elem) % 16 != 0 || !aligned16(k_cache))
    return DSA_ERR_MISALIGNED;
  return static_cast<int>(dsa::launch_index_cache_write(
      keys, key_dtype, key_stride, slots, k_cache, tokens,
      static_cast<int64_t>(num_pages) * dsa::kPage, status_dev, static_cast<cudaStream_t>(stream)));
}

int dsa_kv_cache_append(const void* ckv, int64_t ckv_stride, const void* kpe, int64_t kpe_stride,
                        const int32_t* slots, void* ckv_cache, void* kpe_cache, int tokens,
                        int64_t num_slots, int32_t* status_dev, void* stream) {
  if (tokens == 0) return DSA_OK;
  if (!ckv || !kpe || !slots || !ckv_cache || !kpe_cache) return DSA_ERR_NULL_POINTER;
  if (tokens < 0 || num_slots <= 0 || ckv_stride < dsa::kCkv || kpe_stride < dsa::kKpe)
    return DSA_ERR_BAD_SHAPE;
  if (!aligned16(ckv) || !aligned16(kpe) || !aligned16(ckv_cache) || !aligned16(kpe_cache) ||
      ckv_stride % 8 != 0 || kpe_stride % 8 != 0)
    return DSA_ERR_MISALIGNED;
  return static_cast<int>(dsa::launch_kv_cache_append(ckv, ckv_stride, kpe, kpe_stride, slots,
                                                      ckv_cache, kpe_cache, tokens, num_slots,
                                                      status_dev, static_cast<cudaStream_t>(stream)));
}

// ---- dense attention over the paged caches, eviction from them, rotary append to them ----------
static bool paged_shape_ok(int batch, int tokens, int heads, int max_pages) {
  return batch >= 0 && batch <= 65535 && tokens >= 1 && heads >= 1 && heads <= 128 && (int64_t)tokens * heads <= 65536 &&
         max_pages >= 1 && max_pages <= DSA_PAGED_MAX_PAGES;
}
// Whether requests stay whole, from the batch and the width of the block table (the lengths are on the device).  Whole ones
// save a launch, the partial results and their join; cut ones spread the pages evenly.  The widest table that is better left
// whole grows with the requests (times row blocks) per SM: 3 pages and 13.5 more for each while every one has an SM of
// its own, 2 and 8.5 more beyond, where the last turn leaves SMs idle.  Fitted to the geometric mean over three kinds of
// lengths (all of the table, evenly spread over 1 .. table, spread over its logarithm), 227 pairs of batch and table
// of 16, 64 and 128 rows; the rule takes the slower side by more than 4 % twice (7 % at most: 64 rows, 8 x 4 pages).
// Measured, cut / whole in us, calls in a graph, caches larger than L2; all of the table, even, logarithm:
//   left whole  16 rows:   32 x 4 pages  13.3/11.2  12.8/11.2  11.8/11.0     64 rows:   32 x 4   19.2/14.6  17.7/14.6  15.2/14.5
//                         100 x 12       31.5/25.2  25.8/24.5  20.4/22.4               100 x 12  38.6/31.0  30.3/30.4  23.9/27.6
//                         160 x 8        36.8/35.4  30.9/27.3  27.6/21.8               160 x 8   45.7/44.6  37.3/32.9  32.1/27.4
//                         300 x 16       87.8/88.4  61.5/57.4  48.5/41.3               300 x 16   101/102   76.8/71.2  57.3/48.1
//                         700 x 16        191/147    136/105   95.9/61.7               700 x 16   223/170    168/132    116/79.6
//   cut         16 rows:   32 x 8 pages  15.4/17.3  13.7/17.4  11.0/12.7     64 rows:   64 x 12  29.2/29.2  24.1/28.9  21.2/26.9
//                         100 x 16       35.0/31.3  27.5/30.8  22.0/28.8               100 x 16  45.3/37.5  34.9/37.1  25.9/34.6
//                         160 x 12       44.5/47.7  34.3/33.7  27.6/30.1               160 x 12  54.9/58.1  41.7/43.8  32.4/36.2
//                         300 x 24        113/126   75.7/85.1  51.0/55.6               300 x 24   129/143   91.7/94.6  60.2/60.0
static int paged_split(int batch, int blocks, int max_pages) {
  const int64_t sms = dsa::sm_count(), ctas = (int64_t)batch * blocks;
  const int64_t widest = ctas <= sms ? (6 * sms + 27 * ctas) / (2 * sms) : (4 * sms + 17 * ctas) / (2 * sms);
  if (max_pages > widest) return dsa::kPagedCut;
  return ctas <= sms ? dsa::kPagedOne : dsa::kPagedSnap;
}
// Ranges that the tiles are cut into: a CTA per SM over all row blocks, so that the blocks of one request walk its
// pages at the same time and share them through L2.
static int paged_ranges(int batch, int blocks, int max_pages) {
  if (paged_split(batch, blocks, max_pages) == dsa::kPagedOne) return batch;
  int x = dsa::sm_count() / blocks;
  const int64_t tiles = (int64_t)batch * max_pages;
  if (x > tiles) x = (int)tiles;
  return x < 1 ? 1 : x;
}
static int paged_blocks(int rows) { return (rows + dsa::paged_block_rows(rows) - 1) / dsa::paged_block_rows(rows); }
// [ segments of the requests | partial results | logits ]
static size_t paged_segment_bytes(int batch) { return round256((size_t)batch * sizeof(int2)); }
static size_t paged_part_bytes(int batch, int rows, int max_pages) {
  const int blocks = paged_blocks(rows), ranges = paged_ranges(batch, blocks, max_pages);
  if (ranges == 1 || paged_split(batch, blocks, max_pages) != dsa::kPagedCut) return paged_segment_bytes(batch);
  return paged_segment_bytes(batch) +
         round256((size_t)ranges * blocks * 2 * dsa::paged_part_floats(dsa::paged_block_rows(rows)) * sizeof(float));
}

size_t dsa_paged_attn_workspace_bytes(int batch, int tokens_per_request, int heads, int max_pages, int with_weights) {
  if (batch <= 0 || !paged_shape_ok(batch, tokens_per_request, heads, max_pages)) return 256;
  const int rows = tokens_per_request * heads;
  size_t n = paged_part_bytes(batch, rows, max_pages);
  if (with_weights)
    n += (size_t)batch * max_pages * paged_blocks(rows) * dsa::paged_block_rows(rows) * dsa::kPage * sizeof(float);
  return n;
}

int dsa_paged_attn(const void* q_nope, const void* q_pe, const void* ckv, const void* kpe, const int32_t* seq_lens,
                   const int32_t* block_table, int64_t block_table_stride, float sm_scale, void* out, float* lse,
                   const float* token_weights, int64_t token_weights_stride, float* new_token_weights,
                   int64_t new_token_weights_stride, int batch, int tokens_per_request, int heads, int num_pages,
                   int max_pages, void* workspace, size_t workspace_bytes, int32_t* status_dev, void* stream) {
  if (batch == 0) return DSA_OK;
  if (!q_nope || !q_pe || !ckv || !kpe || !seq_lens || !block_table || !out || !lse || !workspace)
    return DSA_ERR_NULL_POINTER;
  if (!paged_shape_ok(batch, tokens_per_request, heads, max_pages) || num_pages <= 0 ||
      num_pages > DSA_PAGED_MAX_PAGES || block_table_stride < 0 || (token_weights && !new_token_weights))
    return DSA_ERR_BAD_SHAPE;
  const int64_t width = (int64_t)max_pages * dsa::kPage;
  if (new_token_weights && (new_token_weights_stride < width || (token_weights && token_weights_stride < width)))
    return DSA_ERR_BAD_SHAPE;
  if (!aligned16(q_nope) || !aligned16(q_pe) || !aligned16(ckv) || !aligned16(kpe) || !aligned16(out) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return DSA_ERR_MISALIGNED;
  if (workspace_bytes < dsa_paged_attn_workspace_bytes(batch, tokens_per_request, heads, max_pages, new_token_weights != nullptr))
    return DSA_ERR_WORKSPACE_TOO_SMALL;
  const int rows = tokens_per_request * heads;
  const size_t all_rows = (size_t)batch * rows, slots = (size_t)num_pages * dsa::kPage, held = (size_t)width * sizeof(float);
  // weights that grow in place are one argument
  const bool in_place = token_weights == new_token_weights && (batch == 1 || token_weights_stride == new_token_weights_stride);
  const Region regions[] = {
      {out, all_rows * dsa::kCkv * 2, 0, 1},
      {lse, all_rows * sizeof(float), 0, 1},
      {new_token_weights, held, (size_t)new_token_weights_stride * sizeof(float), (size_t)batch},
      {workspace, workspace_bytes, 0, 1},
      {in_place ? nullptr : token_weights, held, (size_t)token_weights_stride * sizeof(float), (size_t)batch},
      {q_nope, all_rows * dsa::kCkv * 2, 0, 1},
      {q_pe, all_rows * dsa::kKpe * 2, 0, 1},
      {ckv, slots * dsa::kCkv * 2, 0, 1},
      {kpe, slots * dsa::kKpe * 2, 0, 1},
      {seq_lens, (size_t)batch * sizeof(int32_t), 0, 1},
      {block_table, (size_t)max_pages * sizeof(int32_t), (size_t)block_table_stride * sizeof(int32_t), (size_t)batch}};
  if (outputs_meet(regions, 4)) return DSA_ERR_OVERLAP;
  dsa::PagedArgs a = {};
  a.q_nope = static_cast<const __nv_bfloat16*>(q_nope);
  a.q_pe = static_cast<const __nv_bfloat16*>(q_pe);
  a.seq_lens = seq_lens;
  a.block_table = block_table;
  a.table_stride = block_table_stride;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.segments = static_cast<int2*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + paged_segment_bytes(batch));
  a.logits = new_token_weights ? reinterpret_cast<float*>(static_cast<char*>(workspace) + paged_part_bytes(batch, rows, max_pages))
                               : nullptr;
  a.status = status_dev;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.batch = batch;
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.rows = rows;
  a.heads = heads;
  a.tokens = tokens_per_request;
  a.block_rows = dsa::paged_block_rows(rows);
  a.grid_x = paged_ranges(batch, paged_blocks(rows), max_pages);
  a.whole = paged_split(batch, paged_blocks(rows), max_pages);
  a.switch_cost = dsa::paged_switch_cost(rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = a.block_rows == 64 ? dsa::launch_paged_attn_tc(a, ckv, kpe, s) : dsa::launch_paged_attn_mma(a, ckv, kpe, s);
  if (e == cudaSuccess && a.grid_x > 1 && a.whole == dsa::kPagedCut) e = dsa::launch_paged_join(a, s);
  if (e == cudaSuccess && new_token_weights)
    e = dsa::launch_paged_weights(a, token_weights, token_weights_stride, new_token_weights, new_token_weights_stride, s);
  return static_cast<int>(e);
}

int dsa_cache_evict(const float* token_weights, int64_t token_weights_stride, const int32_t* seq_lens,
                    const int32_t* block_table, int64_t block_table_stride, const int32_t* new_block_table,
                    int64_t new_block_table_stride, void* ckv, void* kpe, void* k_index_cache, int32_t* new_seq_lens,
                    float* new_token_weights, int64_t new_token_weights_stride, int32_t* kept, int64_t kept_stride, int batch,
                    int max_pages, int new_max_pages, int num_pages, int budget, int keep_first, int keep_last,
                    int32_t* status_dev, void* stream) {
  if (batch == 0) return DSA_OK;
  if (!token_weights || !seq_lens || !block_table || !new_block_table || !ckv || !kpe || !new_seq_lens || !new_token_weights ||
      !kept)
    return DSA_ERR_NULL_POINTER;
  const int64_t width = (int64_t)max_pages * dsa::kPage, most = width < budget ? width : budget;
  if (batch < 0 || batch > 65535 || max_pages < 1 || max_pages > DSA_PAGED_MAX_PAGES || num_pages <= 0 ||
      num_pages > DSA_PAGED_MAX_PAGES || budget < 1 || budget > DSA_EVICT_MAX_BUDGET || keep_first < 0 || keep_last < 0 ||
      (int64_t)keep_first + keep_last > budget || (int64_t)new_max_pages * dsa::kPage < most || token_weights_stride < width ||
      new_token_weights_stride < budget || kept_stride < budget || block_table_stride < 0 || new_block_table_stride < 0)
    return DSA_ERR_BAD_SHAPE;
  if (!aligned16(ckv) || !aligned16(kpe) || !aligned16(k_index_cache)) return DSA_ERR_MISALIGNED;
  const size_t slots = (size_t)num_pages * dsa::kPage, kept_row = (size_t)budget * sizeof(int32_t), n = (size_t)batch;
  const Region regions[] = {
      {ckv, slots * dsa::kCkv * 2, 0, 1},
      {kpe, slots * dsa::kKpe * 2, 0, 1},
      {k_index_cache, (size_t)num_pages * dsa::kPageBytes, 0, 1},
      {new_seq_lens, n * sizeof(int32_t), 0, 1},
      {new_token_weights, kept_row, (size_t)new_token_weights_stride * sizeof(float), n},
      {kept, kept_row, (size_t)kept_stride * sizeof(int32_t), n},
      {token_weights, (size_t)width * sizeof(float), (size_t)token_weights_stride * sizeof(float), n},
      {seq_lens, n * sizeof(int32_t), 0, 1},
      {block_table, (size_t)max_pages * sizeof(int32_t), (size_t)block_table_stride * sizeof(int32_t), n},
      {new_block_table, (size_t)new_max_pages * sizeof(int32_t), (size_t)new_block_table_stride * sizeof(int32_t), n}};
  if (outputs_meet(regions, 6)) return DSA_ERR_OVERLAP;
  return static_cast<int>(dsa::launch_cache_evict(
      token_weights, token_weights_stride, seq_lens, block_table, block_table_stride, new_block_table, new_block_table_stride,
      ckv, kpe, k_index_cache, new_seq_lens, new_token_weights, new_token_weights_stride, kept, kept_stride, batch, max_pages,
      num_pages, budget, keep_first, keep_last, status_dev, static_cast<cudaStream_t>(stream)));
}

int dsa_rotary_append(const void* q_pe, int64_t q_token_stride, int64_t q_head_stride, const void* ckv, int64_t ckv_stride,
                      const void* kpe, int64_t kpe_stride, const int32_t* positions, int64_t positions_stride, int axes,
                      const float* inv_freq, uint64_t pair_axes, int interleaved, const int32_t* slots, void* q_out,
                      void* ckv_cache, void* kpe_cache, int tokens, int heads, int64_t num_slots, int32_t* status_dev,
                      void* stream) {
  if (tokens == 0) return DSA_OK;
  if (!q_pe || !ckv || !kpe || !positions || !inv_freq || !slots || !q_out || !ckv_cache || !kpe_cache)
    return DSA_ERR_NULL_POINTER;
  if (tokens < 0 || heads < 1 || heads > 128 || axes < 1 || axes > 4 || num_slots <= 0 || positions_stride < 0 ||
      ckv_stride < dsa::kCkv || kpe_stride < dsa::kKpe || q_token_stride < dsa::kKpe || q_head_stride < dsa::kKpe)
    return DSA_ERR_BAD_SHAPE;
  for (int i = 0; i < dsa::kKpe / 2; ++i)
    if ((int)((pair_axes >> (2 * i)) & 3u) >= axes) return DSA_ERR_BAD_SHAPE;
  if (!aligned16(q_pe) || !aligned16(ckv) || !aligned16(kpe) || !aligned16(q_out) || !aligned16(ckv_cache) ||
      !aligned16(kpe_cache) || q_token_stride % 8 != 0 || q_head_stride % 8 != 0 || ckv_stride % 8 != 0 || kpe_stride % 8 != 0)
    return DSA_ERR_MISALIGNED;
  const size_t n = (size_t)tokens, q_row = ((size_t)(heads - 1) * q_head_stride + dsa::kKpe) * 2;
  const bool in_place = q_out == q_pe && (heads == 1 || q_head_stride == dsa::kKpe) &&
                        (tokens == 1 || q_token_stride == (int64_t)heads * dsa::kKpe);
  const Region q = {in_place ? nullptr : q_pe, q_row, (size_t)q_token_stride * 2, n};
  const Region turned = {q_out, n * heads * dsa::kKpe * 2, 0, 1};
  const Region regions[] = {
      {ckv_cache, (size_t)num_slots * dsa::kCkv * 2, 0, 1},
      {kpe_cache, (size_t)num_slots * dsa::kKpe * 2, 0, 1},
      turned,
      q,
      {positions, n * sizeof(int32_t), (size_t)positions_stride * sizeof(int32_t), (size_t)axes},
      {inv_freq, dsa::kKpe / 2 * sizeof(float), 0, 1},
      {slots, n * sizeof(int32_t), 0, 1}};
  // (ckv and kpe may lie in the caches, where rows of another place are stored again)
  if (outputs_meet(regions, 3) || meet(turned, {ckv, dsa::kCkv * 2, (size_t)ckv_stride * 2, n}) ||
      meet(turned, {kpe, dsa::kKpe * 2, (size_t)kpe_stride * 2, n}))
    return DSA_ERR_OVERLAP;
  return static_cast<int>(dsa::launch_rotary_append(q_pe, q_token_stride, q_head_stride, ckv, ckv_stride, kpe, kpe_stride,
                                                    positions, positions_stride, inv_freq, pair_axes, interleaved, slots, q_out,
                                                    ckv_cache, kpe_cache, tokens, heads, num_slots, status_dev,
                                                    static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
