// Dense attention of every request's newest tokens over its whole paged ckv / kpe cache, for requests of at most 16 query
// rows (one new token of 16 heads); paged_attn_tc.cu has the others.
//
//   x[r,k]  = (q_nope[r].ckv[k] + q_pe[r].kpe[k]) * sm_scale * log2 e        k < the positions row r sees
//   lse[r]  = log2 sum_k 2^x[r,k]        out[r] = sum_k 2^(x[r,k] - lse[r]) ckv[k]
// A request's rows r are its new tokens x heads; token i of n sees the positions below len - n + 1 + i.
//
// Bound by the one read of the cache (1152 B per cached token, 2 * 1088 flops per byte-row and query row): with 16
// rows the products of a 64-token page are 544 mma.sync.m16n8k16, 1.1 k cycles at the 2.0 cycles each that this part
// issues, against 3.2 k cycles in which an SM's share of the memory bandwidth delivers the page.
//
// One CTA of 8 warps per SM, three stages of one 64-token page each.  A page is nine [64 rows x 128 B] TMA boxes (8
// ckv column blocks and kpe) with the 128-byte swizzle, which keeps both ldmatrix patterns free of bank conflicts;
// nine lanes of warp 0 issue a page's boxes two pages ahead, into the stage that the page before the current one has
// just left, and look the page ids up 32 at a time, one batch ahead.
//   S = Q.K^T   warp w has tokens 8w .. 8w+7 of the page; q_nope stays in registers as 32 A fragments, q_pe in shared
//               memory (all 36 in registers left the loop none to schedule in);
//   softmax     base 2, the running maximum refreshed (and O rescaled) only when a logit exceeds it by more than 2^8;
//               P is rounded to bf16 for the second product, whose operands have one type and whose other one is the bf16
//               cache; sums are taken of the fp32 values.  The rounding is independent from key to key and of the size of
//               the output's own (rms error against 64 bits 0.0020 with both, 0.0017 with the output's alone: 1 x 1000 tokens).
//               P as a sum of two bf16 operands gives 0.0017 and makes 256 products more per page: 64 x 32768 tokens 424 -> 476 us,
//               48 ragged requests 34.7 -> 38.1, 1 x 131071 35.6 -> 38.8, so it is not done;
//   O += P.V    warp w has the output columns 64w .. 64w+63 = column block w of the same stage (ldmatrix.trans).
// Rows behind a request's length are put to zero in the stage before the second product: the cache may hold anything
// there, and 0 x NaN would get into the sum.
#include "mma.cuh"
#include "paged_attn.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace dsa {

namespace {

constexpr int kPaStages = 3;
constexpr int kPaBlockBytes = kPage * 128;           // 8192
constexpr int kPaStageBytes = 9 * kPaBlockBytes;     // 73728
constexpr int kPaThreads = 256;
constexpr int kPaRows = 16;                          // query rows of a block
constexpr int kPaQPitch = 1040;                      // 1024-byte q_nope rows, padded against bank conflicts
constexpr float kPaRescaleGap = 8.f;

struct PaTile {
  int b, j, len, live;
};
struct PaShared {
  uint64_t full[kPaStages];
  PaTile tile[kPaStages];
  float red[8][kPaRows];
  long long sums[kPaThreads / 32];
  PagedRange range;
};

constexpr size_t kPaDynBytes = 1024 + kPaStages * kPaStageBytes + 2 * kPaRows * 128 + sizeof(PaShared);
static_assert(kPaDynBytes <= 232448, "shared memory of one CTA");

template <bool kLogits>
__global__ void __launch_bounds__(kPaThreads, 1)
paged_attn_mma_kernel(const __grid_constant__ CUtensorMap map_ckv, const __grid_constant__ CUtensorMap map_kpe,
                      const PagedArgs a) {
  extern __shared__ unsigned char dyn_raw[];
  const uint32_t raw_addr = smem_u32(dyn_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t kv_addr = raw_addr + pad;
  unsigned char* kv_ptr = dyn_raw + pad;
  const uint32_t p_addr = kv_addr + kPaStages * kPaStageBytes;
  unsigned char* p_ptr = kv_ptr + kPaStages * kPaStageBytes;
  const uint32_t qpe_addr = p_addr + kPaRows * 128;
  PaShared& sh = *reinterpret_cast<PaShared*>(p_ptr + 2 * kPaRows * 128);

  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int rb = blockIdx.y, range = blockIdx.x;

  if (tid == 0) {
    ptx::prefetch_tensormap(&map_ckv);
    ptx::prefetch_tensormap(&map_kpe);
    for (int s = 0; s < kPaStages; ++s) ptx::mbar_init(smem_u32(&sh.full[s]), 1);
    ptx::fence_barrier_init();
  }
  ptx::grid_dependency_wait();
  ptx::launch_dependents();

  // ---------------- this CTA's range of tiles --------------------------------------------------------
  paged_find_range<kPaThreads>(a, range, sh.sums, &sh.range);
  __syncthreads();
  const int n = (int)(sh.range.end - sh.range.begin);
  if (n <= 0) return;

  // ---------------- tile issue (warp 0) --------------------------------------------------------------
  int issued = 0;
  int ib = sh.range.start_b, ij = sh.range.start_j, ilen = 0, itiles = 0, cbase = ij;
  int cur = -1, nb = 0, nc = 0, nxt = -1, nlen = 0;
  auto lookup = [&](int b, int c) {      // page ids of tiles c .. c+31 of request b, one per lane
    return b < a.batch && c + lane < a.max_pages ? __ldg(a.block_table + (int64_t)b * a.table_stride + c + lane) : -1;
  };
  auto look_ahead = [&]() {              // the 32 ids behind the current ones, and the length they belong to
    const bool same = cbase + 32 < itiles;
    nb = same ? ib : ib + 1;
    nc = same ? cbase + 32 : 0;
    nxt = lookup(nb, nc);
    nlen = nb < a.batch ? paged_len(__ldg(a.seq_lens + nb), a.max_pages) : 0;
  };
  if (w == 0) {
    ilen = paged_len(__ldg(a.seq_lens + ib), a.max_pages);
    itiles = paged_tiles(ilen, a.max_pages);
    cur = lookup(ib, cbase);
    look_ahead();
  }
  auto issue_tile = [&]() {
    if (issued < n) {
      if (ij == itiles || ij - cbase == 32) {
        if (nb != ib) {
          ib = nb;
          ij = 0;
          ilen = nlen;
          itiles = paged_tiles(ilen, a.max_pages);
        }
        cbase = nc;
        cur = nxt;
        look_ahead();
      }
      const int s = issued % kPaStages;
      const int page = __shfl_sync(0xffffffffu, cur, ij - cbase);
      const bool held = ilen > 0, live = held && page >= 0 && page < a.num_pages;
      const uint32_t bar = smem_u32(&sh.full[s]), dst = kv_addr + s * kPaStageBytes;
      if (lane == 0) {
        sh.tile[s] = {ib, ij, ilen, live ? 1 : 0};
        if (held && !live) raise_status(a.status, DSA_STATUS_BAD_PAGE);
        if (live) ptx::mbar_expect_tx(bar, kPaStageBytes);
        else ptx::mbar_arrive(bar);
      }
      __syncwarp();
      if (live) {
        if (lane < 8) ptx::tma_load_2d(dst + lane * kPaBlockBytes, &map_ckv, lane * 64, page * kPage, bar);
        else if (lane == 8) ptx::tma_load_2d(dst + 8 * kPaBlockBytes, &map_kpe, 0, page * kPage, bar);
      }
      ++ij;
    }
    ++issued;
  };

  // q rows of a request's block, padded rows as zeros
  auto stage_q = [&](int b, uint32_t qs) {
    for (int c = tid; c < kPaRows * 72; c += kPaThreads) {
      const int h = c / 72, jj = c - h * 72;
      const int r = rb * kPaRows + h;
      const size_t row = (size_t)b * a.rows + (r < a.rows ? r : 0);
      const __nv_bfloat16* src = jj < 64 ? a.q_nope + row * kCkv + jj * 8 : a.q_pe + row * kKpe + (jj - 64) * 8;
      const uint32_t dst = jj < 64 ? qs + h * kPaQPitch + jj * 16 : qpe_addr + h * 128 + (((jj - 64) ^ (h & 7)) << 4);
      ptx::cp_async16(dst, src, r < a.rows ? 16 : 0);
    }
    cp_async_commit();
  };
  stage_q(sh.range.start_b, kv_addr + 2 * kPaStageBytes);   // tile 2 gets the stage once q is in registers
  if (w == 0) {
    issue_tile();
    issue_tile();
  }

  // where the logits of a tile go (only where they are wanted; padding rows among them: leaving these out cost 3 % at
  // 64 x 16384 tokens x 16 rows, 223 us against 216, and gave nothing at 64 x 8192 x 5 rows)
  auto tile_logits = [&](const PaTile& t) {
    return a.logits + (((size_t)t.b * a.max_pages + t.j) * gridDim.y + rb) * (size_t)(kPaRows * kPage);
  };
  // token (of the request's new ones) of each row of this thread; rows behind the last see nothing
  int row_tok[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = rb * kPaRows + g + 8 * e;
    row_tok[e] = r < a.rows ? r / a.heads : -1;
  }

  uint32_t qa[32][4];           // A fragments of q_nope: k-step ks covers columns 16 ks .. 16 ks + 15
  float o[8][4];                // O[rows g / g+8][columns 64 w + 8 n + 2 t4, +1]
  float m0 = -INFINITY, m1 = -INFINITY;
  float l0 = 0.f, l1 = 0.f;     // row sums over this thread's tokens
  int cur_b = -1, first_j = 0, lim0 = 0, lim1 = 0;
  bool lost = false;

  for (int i = 0; i < n; ++i) {
    const int s = i % kPaStages;
    const bool landed = ptx::mbar_wait(smem_u32(&sh.full[s]), (i / kPaStages) & 1);
    // tile i has landed for every thread, and everyone is done with tile i-1
    if (__syncthreads_or(!landed)) {
      if (!landed && lane == 0) raise_status(a.status, DSA_STATUS_WAIT_TIMEOUT);
      lost = true;
      break;
    }
    const PaTile tile = sh.tile[s];
    if (tile.b != cur_b) {
      const uint32_t qs = kv_addr + ((i + 2) % kPaStages) * kPaStageBytes;
      if (i > 0) stage_q(tile.b, qs);
      cp_async_wait_group<0>();
      __syncthreads();
      const uint32_t qrow = qs + ((lane & 7) + ((lane >> 3) & 1) * 8) * kPaQPitch + (lane >> 4) * 16;
#pragma unroll
      for (int ks = 0; ks < 32; ++ks) ldsm_x4(qrow + ks * 32, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3]);
#pragma unroll
      for (int nn = 0; nn < 8; ++nn) o[nn][0] = o[nn][1] = o[nn][2] = o[nn][3] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
      cur_b = tile.b;
      first_j = tile.j;
      if (tid == 0 && rb == 0 && first_j == 0 && a.whole == kPagedCut)
        paged_tell_segments(a, sh.range, range, i, tile.b, tile.len);
      const int base = tile.len - a.tokens + 1;
      lim0 = row_tok[0] < 0 ? 0 : base + row_tok[0];
      lim1 = row_tok[1] < 0 ? 0 : base + row_tok[1];
      ptx::fence_proxy_async_smem();   // the stage now goes back from plain stores and reads to TMA
      __syncthreads();
    }
    if (w == 0) issue_tile();          // tile i+2 -> the stage tile i-1 used
    const int pos0 = tile.j * kPage;
    if (!tile.live) {
      if (kLogits && tile.len > 0) {
        float* lg = tile_logits(tile);
        for (int c = tid; c < kPaRows * kPage; c += kPaThreads) lg[c] = -INFINITY;
      }
    } else {
      const uint32_t sa = kv_addr + s * kPaStageBytes;
      const int filled = tile.len - pos0;
      if (filled < kPage) {            // last page of the request: what lies behind its tokens becomes zero
        for (int c = tid; c < (kPage - filled) * 64; c += kPaThreads) {
          const int r = filled + (c >> 6), k = c & 63;
          *reinterpret_cast<uint4*>(kv_ptr + s * kPaStageBytes + (k >> 3) * kPaBlockBytes + r * 128 + (k & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        ptx::fence_proxy_async_smem();   // TMA writes the stage next
      }
      // ---- S = Q . K^T for tokens 8w .. 8w+7; four accumulator chains --------------------------
      float acc[4][4];
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
      {
        const int tok = 8 * w + (lane & 7), rx = tok & 7, quad = lane >> 3;
        const uint32_t brow = sa + tok * 128;
#pragma unroll
        for (int kb = 0; kb < 9; ++kb) {
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            uint32_t r0, r1, r2, r3;
            ldsm_x4(brow + kb * kPaBlockBytes + (((kk * 4 + quad) ^ rx) << 4), r0, r1, r2, r3);
            if (kb < 8) {
              hmma_16816(acc[2 * kk], qa[kb * 4 + 2 * kk], r0, r1);
              hmma_16816(acc[2 * kk + 1], qa[kb * 4 + 2 * kk + 1], r2, r3);
            } else {                     // q_pe
              const int qr = (lane & 7) + ((lane >> 3) & 1) * 8;
              uint32_t qp[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h)
                ldsm_x4(qpe_addr + qr * 128 + (((4 * kk + 2 * h + (lane >> 4)) ^ (qr & 7)) << 4), qp[h][0], qp[h][1], qp[h][2],
                        qp[h][3]);
              hmma_16816(acc[2 * kk], qp[0], r0, r1);
              hmma_16816(acc[2 * kk + 1], qp[1], r2, r3);
            }
          }
        }
      }
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool seen = pos0 + 8 * w + 2 * t4 + (e & 1) < (e < 2 ? lim0 : lim1);
        const float v = (acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e]);
        x[e] = seen ? v * a.scale_log2 : -INFINITY;
      }
      // where this thread's P goes: [row][token], 16-byte chunks swizzled by the row
      uint32_t* pw0 = reinterpret_cast<uint32_t*>(p_ptr + g * 128 + ((w ^ (g & 7)) << 4) + t4 * 4);
      uint32_t* pw1 = reinterpret_cast<uint32_t*>(p_ptr + (g + 8) * 128 + ((w ^ (g & 7)) << 4) + t4 * 4);
      float v0 = fmaxf(x[0], x[1]), v1 = fmaxf(x[2], x[3]);
      const bool need = v0 > m0 + kPaRescaleGap || v1 > m1 + kPaRescaleGap;
      float p[4];
      auto publish = [&]() {
        const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
        p[0] = exp2f(x[0] - u0);
        p[1] = exp2f(x[1] - u0);
        p[2] = exp2f(x[2] - u1);
        p[3] = exp2f(x[3] - u1);
        *pw0 = pack_bf162(p[0], p[1]);
        *pw1 = pack_bf162(p[2], p[3]);
      };
      // P with the running maxima as they are; the barrier that makes it visible tells whether a logit exceeded
      // its maximum by more than 2^8 (rare)
      publish();
      if (__syncthreads_or(need)) {
        v0 = fmaxf(v0, __shfl_xor_sync(0xffffffffu, v0, 1));
        v0 = fmaxf(v0, __shfl_xor_sync(0xffffffffu, v0, 2));
        v1 = fmaxf(v1, __shfl_xor_sync(0xffffffffu, v1, 1));
        v1 = fmaxf(v1, __shfl_xor_sync(0xffffffffu, v1, 2));
        if (t4 == 0) {
          sh.red[w][g] = v0;
          sh.red[w][g + 8] = v1;
        }
        __syncthreads();
        float n0 = m0, n1 = m1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          n0 = fmaxf(n0, sh.red[k][g]);
          n1 = fmaxf(n1, sh.red[k][g + 8]);
        }
        const float c0 = n0 == -INFINITY ? 1.f : exp2f(m0 - n0), c1 = n1 == -INFINITY ? 1.f : exp2f(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= c0;
        l1 *= c1;
#pragma unroll
        for (int nn = 0; nn < 8; ++nn) {
          o[nn][0] *= c0;
          o[nn][1] *= c0;
          o[nn][2] *= c1;
          o[nn][3] *= c1;
        }
        publish();
        __syncthreads();
      }
      l0 += p[0] + p[1];
      l1 += p[2] + p[3];
      if (kLogits) {                    // behind the barrier that the other warps wait at
        float* lg = tile_logits(tile) + g * kPage + 8 * w + 2 * t4;
        *reinterpret_cast<float2*>(lg) = make_float2(x[0], x[1]);
        *reinterpret_cast<float2*>(lg + 8 * kPage) = make_float2(x[2], x[3]);
      }
      // ---- O += P . V for columns 64w .. 64w+63 (column block w of the tile) ---------------------
      {
        const int hrow = (lane & 7) + ((lane >> 3) & 1) * 8, half = lane >> 4;
        const uint32_t vbase = sa + w * kPaBlockBytes;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          uint32_t pf[4];
          ldsm_x4(p_addr + hrow * 128 + (((ks * 2 + half) ^ (hrow & 7)) << 4), pf[0], pf[1], pf[2], pf[3]);
          const int vrow = ks * 16 + hrow;
          const uint32_t va = vbase + vrow * 128;
#pragma unroll
          for (int np = 0; np < 4; ++np) {
            uint32_t r0, r1, r2, r3;
            ldsm_x4_trans(va + (((np * 2 + half) ^ (vrow & 7)) << 4), r0, r1, r2, r3);
            hmma_16816(o[2 * np], pf, r0, r1);
            hmma_16816(o[2 * np + 1], pf, r2, r3);
          }
        }
      }
    }
    const bool ends = tile.j == paged_tiles(tile.len, a.max_pages) - 1;
    if (ends || i == n - 1) {
      // ------------------ end of this CTA's segment of the request --------------------------------
      float s0 = l0, s1 = l1;
      s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
      s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
      s1 += __shfl_xor_sync(0xffffffffu, s1, 1);
      s1 += __shfl_xor_sync(0xffffffffu, s1, 2);
      __syncthreads();                 // sh.red may still be read by a slow warp of a refresh above
      if (t4 == 0) {
        sh.red[w][g] = s0;
        sh.red[w][g + 8] = s1;
      }
      __syncthreads();
      const bool whole = ends && first_j == 0;
      float* part = whole ? nullptr : paged_part(a, kPaRows, rb, range, first_j == 0 ? 1 : 0);
      const int col = 64 * w + 2 * t4;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int br = g + 8 * e, r = rb * kPaRows + br;
        const float m = e ? m1 : m0;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += sh.red[k][br];
        if (r >= a.rows) continue;
        if (whole) {
          // a row that sees nothing has output 0 and lse -inf; a NaN sum stays NaN
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          __nv_bfloat16* dst = a.out + ((size_t)tile.b * a.rows + r) * kCkv + col;
#pragma unroll
          for (int nn = 0; nn < 8; ++nn)
            *reinterpret_cast<uint32_t*>(dst + 8 * nn) = pack_bf162(o[nn][2 * e] * inv, o[nn][2 * e + 1] * inv);
          if (w == 0 && t4 == 0) a.lse[(size_t)tile.b * a.rows + r] = sum == 0.f ? -INFINITY : m + log2f(sum);
        } else {
          float* dst = part + (size_t)br * kCkv + col;
#pragma unroll
          for (int nn = 0; nn < 8; ++nn)
            *reinterpret_cast<float2*>(dst + 8 * nn) = make_float2(o[nn][2 * e], o[nn][2 * e + 1]);
          if (w == 0 && t4 == 0) {
            part[(size_t)kPaRows * kCkv + br] = sum == 0.f ? -INFINITY : m;
            part[(size_t)kPaRows * (kCkv + 1) + br] = sum;
          }
        }
      }
      __syncthreads();                 // sh.red may be written again
    }
  }
  cp_async_wait_group<0>();
  if (lost) {   // give the copies in flight a bounded time to land before the CTA's shared memory goes
    for (int k = 0; k < 64; ++k) __nanosleep(20000);
  }
}

}  // namespace

template <bool kLogits>
static cudaError_t launch_mma(const PagedArgs& a, const CUtensorMap& mc, const CUtensorMap& mk, cudaStream_t stream) {
  static std::atomic<uint64_t> opted{0};
  const cudaError_t e =
      opt_in_dynamic_smem(reinterpret_cast<const void*>(paged_attn_mma_kernel<kLogits>), kPaDynBytes, opted);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.grid_x, (unsigned)((a.rows + kPaRows - 1) / kPaRows));
  cfg.blockDim = dim3(kPaThreads);
  cfg.dynamicSmemBytes = kPaDynBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_mma_kernel<kLogits>, mc, mk, a);
}

cudaError_t launch_paged_attn_mma(const PagedArgs& a, const void* ckv, const void* kpe, cudaStream_t stream) {
  CUtensorMap mc, mk;
  const uint64_t slots = (uint64_t)a.num_pages * kPage;
  if (!make_tmap_2d_sw128(&mc, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ckv, kCkv, slots, 64, kPage) ||
      !make_tmap_2d_sw128(&mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kpe, kKpe, slots, 64, kPage))
    return cudaErrorInvalidValue;
  return a.logits ? launch_mma<true>(a, mc, mk, stream) : launch_mma<false>(a, mc, mk, stream);
}

}  // namespace dsa
