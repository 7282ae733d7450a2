// Dense attention of every request's newest tokens over its whole paged cache (the operator of paged_attn_mma.cu) for
// requests with many query rows -- drafted tokens, or all 128 heads on one GPU -- on the 5th-generation tensor cores.
//
// 64 query rows of a request per CTA.  A 64-token page is read once from memory for all of them:
//   S[64 rows, 64 tokens]  = Q[64,576] . K^T      A = q, K-major, resident; B = the page, K-major      (36 tcgen05.mma)
//   O^T[512, 64 rows]     += V^T[512,64] . P^T    A = the SAME page read MN-major; B = P, K-major       (16 tcgen05.mma)
// The first product has the rows as M: a softmax warp then holds 16 rows x 32 tokens in the fragment order of the warp-level
// products, and writes P as that order's 4-byte pairs without bank conflicts.  The second is transposed because the
// rows are too few for M: 512 output columns are four M = 128 blocks, and the accumulator is 256 of the 512 TMEM
// columns, which leaves room for two S buffers.  P is rounded to bf16, as in paged_attn_mma.cu (which has the error and what the
// remainder as a second operand costs; here that would be 16 more instructions of 49 cycles per page, and 8 KB of shared
// memory beside q and two pages, where less than 2 KB are left); the sums are taken of the fp32 values.
//
// Bounds: an instruction reads its operands from shared memory at 128 B per cycle, so the first product's cost 32 cycles
// (M = N = 64; measured 36 when a converged warp issues them, 55-160 from a branch of one lane, whose descriptors have
// to be moved to uniform registers each time) and the second's 48 (49): 2.1 k cycles per page, against the 3.2 k in
// which an SM's share of the memory bandwidth delivers it.  q (72 KB) and P leave shared memory for two pages only, so
// what counts is how long a page stays: every page travels as four column groups with barriers of their own -- the
// first product follows the groups as they land, the second hands each back as it is done -- the two products are
// issued by warps of their own, and L2 is asked for the pages that have no place yet.  Steady state 3.0 k cycles per
// page; 16 requests x 8192 tokens x 64 rows take 47 us, floor 23.4 us (memory): 8 us until the first page is there, 22 us
// of pages, 3 us to store the partial results, the rest the join.
//
// Roles (352 threads): warps 0-7 softmax and epilogue, warp 8 issues the first products and warp 9 the second ones (a
// second product is not to wait behind a first one whose page is still landing), warp 10 the TMA loads.  Every wait is
// bounded; a wait that runs out is told at the softmax warps' next barrier, so that all of them leave together, and
// to the other roles by a flag.
#include "paged_attn.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace dsa {

namespace {

constexpr int kTcRows = 64;
constexpr int kTcBlock = kPage * 128;            // one [64 x 128 B] block
constexpr int kTcPage = 9 * kTcBlock;            // 73728
constexpr int kTcSoftmax = 256;                 // threads of the softmax warps
constexpr int kTcThreads = kTcSoftmax + 96;
constexpr int kTcGroups = 4;                     // column groups of a page: ckv blocks 2c, 2c+1; the last also kpe
constexpr int kTcAhead = 2;                      // pages that L2 is asked for beyond the one being loaded
constexpr int kTcCols = 512;
constexpr int kTcSCol = 4 * kTcRows;             // O^T block c at column 64c, S buffer s at 256 + 64s
constexpr float kTcGap = 8.f;
constexpr uint32_t kTcIdescQK = ptx::idesc(ptx::kFmtBF16, ptx::kFmtBF16, false, false, kTcRows, kPage);
constexpr uint32_t kTcIdescPV = ptx::idesc(ptx::kFmtBF16, ptx::kFmtBF16, true, false, 128, kTcRows);

struct TcTile {
  int b, j, len;
  short live, last;     // has a page; is the request's last tile
};
struct TcShared {
  uint64_t full[2][kTcGroups], empty[2][kTcGroups], q_full, q_empty, s_full[2], s_empty[2], p_full, p_empty, told;
  TcTile tile[2];
  float corr[kTcRows], inv[kTcRows];   // of each row: what O^T is multiplied by in a refresh, and at the end
  float half[2][kTcRows];              // maxima, at the end sums, over the token halves
  long long sums[kTcThreads / 32];
  PagedRange range;
  alignas(16) int word[4][8];          // what the softmax warps tell each other at a barrier: 1 = refresh, 2 = a wait ran out
  uint32_t tmem_base;
  volatile int abort_flag;
};
constexpr size_t kTcDynBytes = 1024 + 3 * kTcPage + kTcRows * 128 + sizeof(TcShared);
static_assert(kTcDynBytes <= 232448, "shared memory of one CTA");

template <bool kLogits>
__global__ void __launch_bounds__(kTcThreads, 1)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap map_ckv, const __grid_constant__ CUtensorMap map_kpe,
                     const __grid_constant__ CUtensorMap map_qn, const __grid_constant__ CUtensorMap map_qp,
                     const __nv_bfloat16* ckv, const __nv_bfloat16* kpe, const PagedArgs a) {
  extern __shared__ unsigned char dyn_raw[];
  const uint32_t raw_addr = smem_u32(dyn_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t kv_addr = raw_addr + pad;              // two pages
  const uint32_t q_addr = kv_addr + 2 * kTcPage;
  const uint32_t p_addr = q_addr + kTcPage;
  unsigned char* kv_ptr = dyn_raw + pad;
  unsigned char* p_ptr = kv_ptr + 3 * kTcPage;
  TcShared& sh = *reinterpret_cast<TcShared*>(p_ptr + kTcRows * 128);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rb = blockIdx.y, range = blockIdx.x;

  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        for (int c = 0; c < kTcGroups; ++c) {
          ptx::mbar_init(smem_u32(&sh.full[s][c]), 1);
          ptx::mbar_init(smem_u32(&sh.empty[s][c]), c == 0 ? 9 : 1);   // the products; group 0 also the softmax warps
        }
        ptx::mbar_init(smem_u32(&sh.s_full[s]), 1);
        ptx::mbar_init(smem_u32(&sh.s_empty[s]), 8);
      }
      ptx::mbar_init(smem_u32(&sh.q_full), 1);
      ptx::mbar_init(smem_u32(&sh.q_empty), 1);
      ptx::mbar_init(smem_u32(&sh.p_full), 8);
      ptx::mbar_init(smem_u32(&sh.p_empty), 1);
      ptx::mbar_init(smem_u32(&sh.told), 8);
      sh.abort_flag = 0;
      ptx::fence_barrier_init();
    }
    __syncwarp();
    ptx::tmem_alloc(smem_u32(&sh.tmem_base), kTcCols);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  paged_find_range<kTcThreads>(a, range, sh.sums, &sh.range);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const int n = (int)(sh.range.end - sh.range.begin);
  const uint32_t tmem = sh.tmem_base;

  if (n > 0 && warp < 8) {
    // ============================ softmax and epilogue ============================
    // The rows lie in an M = 64 accumulator 16 to a quarter; warps q and q + 4 take the quarter's rows for 32 tokens
    // each.  Read as fragments, a thread has rows g and g + 8, and of each 8 tokens the two at 2 t4.
    const int g = lane >> 2, t4 = lane & 3, quarter = warp & 3, half = warp >> 2;
    const int row0 = quarter * 16 + g;
    int row_tok[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = rb * kTcRows + row0 + 8 * e;
      row_tok[e] = r < a.rows ? r / a.heads : -1;
    }
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    int pl = 0, seg_live = 0, cur_b = -1, first_j = 0, lim0 = 0, lim1 = 0, lost = 0;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    // a wait that runs out is remembered and told at the next barrier, where all warps leave together
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(smem_u32(&bar), parity) ? 1 : 0)) lost = 2;
    };
    auto words = [&](int which) {
      const int4 u = *reinterpret_cast<const int4*>(&sh.word[which][0]), v = *reinterpret_cast<const int4*>(&sh.word[which][4]);
      return (u.x | u.y | u.z | u.w) | (v.x | v.y | v.z | v.w);
    };
    auto tell = [&](int which) {
      if (lane == 0) sh.word[which][warp] = lost;
      ptx::named_bar_sync(1, kTcSoftmax);
      return words(which);
    };
    for (int i = 0; i < n; ++i) {
      const int s = i & 1, phase = (i >> 1) & 1;
      wait(sh.full[s][0], phase);
      wait(sh.s_full[s], phase);
      const TcTile tile = sh.tile[s];
      const bool live = !lost && tile.live;
      if (tile.b != cur_b) {
        cur_b = tile.b;
        first_j = tile.j;
        if (tid == 0 && rb == 0 && first_j == 0 && a.whole == kPagedCut)
          paged_tell_segments(a, sh.range, range, i, tile.b, tile.len);
        seg_live = 0;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
        lim0 = row_tok[0] < 0 ? 0 : tile.len - a.tokens + 1 + row_tok[0];
        lim1 = row_tok[1] < 0 ? 0 : tile.len - a.tokens + 1 + row_tok[1];
      }
      const int pos0 = tile.j * kPage;
      float* lg = nullptr;                           // (rows behind a request's last are not stored)
      if (kLogits)
        lg = a.logits + ((((size_t)tile.b * a.max_pages + tile.j) * gridDim.y + rb) * kTcRows + row0) * (size_t)kPage +
             32 * half + 2 * t4;
      float x[16];
      float v0 = -INFINITY, v1 = -INFINITY;
      if (live) {
        uint32_t raw[16];
        ptx::tc_fence_after();
        ptx::tmem_ld_frag32(tmem + lanes + kTcSCol + s * 64 + 32 * half, raw);
        ptx::tmem_wait_ld();
        ptx::tc_fence_before();
        const bool all_seen = pos0 + kPage <= min(lim0, lim1);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int pos = pos0 + 32 * half + 8 * (k >> 2) + 2 * t4 + (k & 1);
          const bool seen = all_seen || pos < ((k & 2) ? lim1 : lim0);
          x[k] = seen ? __uint_as_float(raw[k]) * a.scale_log2 : -INFINITY;
          if (k & 2) v1 = fmaxf(v1, x[k]);
          else v0 = fmaxf(v0, x[k]);
        }
      }
      __syncwarp();
      if (lane == 0) {                               // S buffer and tile word have been read by this warp
        ptx::mbar_arrive(smem_u32(&sh.s_empty[s]));
        ptx::mbar_arrive(smem_u32(&sh.empty[s][0]));
      }
      // whether a logit exceeds its row's maximum by more than 2^8 is told while the weights are being computed with the
      // maxima as they are; it is rare
      const bool need = __any_sync(0xffffffffu, v0 > m0 + kTcGap || v1 > m1 + kTcGap);
      if (lane == 0) {
        sh.word[i & 1][warp] = (need ? 1 : 0) | lost;
        ptx::mbar_arrive(smem_u32(&sh.told));
      }
      uint32_t pk[8];
      float s0, s1;
      auto weigh = [&]() {
        const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
        s0 = s1 = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p0 = ptx::exp2_ftz(x[4 * k] - u0), p1 = ptx::exp2_ftz(x[4 * k + 1] - u0);
          const float p2 = ptx::exp2_ftz(x[4 * k + 2] - u1), p3 = ptx::exp2_ftz(x[4 * k + 3] - u1);
          s0 += p0 + p1;
          s1 += p2 + p3;
          const __nv_bfloat162 ha = __floats2bfloat162_rn(p0, p1), hb = __floats2bfloat162_rn(p2, p3);
          pk[2 * k] = *reinterpret_cast<const uint32_t*>(&ha);
          pk[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&hb);
        }
      };
      if (live) weigh();
      // (every warp arrives within its own waits' limits, far below this one)
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(smem_u32(&sh.told), i & 1, 4000000000ull) ? 1 : 0)) {
        lost = 2;
        break;
      }
      const int told = words(i & 1);
      if (told & 2) break;
      if (!live) {
        if (kLogits && tile.len > 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (row_tok[0] >= 0) *reinterpret_cast<float2*>(lg + 8 * k) = make_float2(-INFINITY, -INFINITY);
            if (row_tok[1] >= 0) *reinterpret_cast<float2*>(lg + 8 * kPage + 8 * k) = make_float2(-INFINITY, -INFINITY);
          }
        }
      } else {
        const int filled = tile.len - pos0;
        if (filled < kPage) {                        // what lies behind the request's tokens becomes zero
          for (int c = tid; c < (kPage - filled) * 64; c += kTcSoftmax) {
            const int rr = filled + (c >> 6), k = c & 63;
            *reinterpret_cast<uint4*>(kv_ptr + s * kTcPage + (k >> 3) * kTcBlock + rr * 128 + (k & 7) * 16) =
                make_uint4(0, 0, 0, 0);
          }
        }
        if (kLogits) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (row_tok[0] >= 0) *reinterpret_cast<float2*>(lg + 8 * k) = make_float2(x[4 * k], x[4 * k + 1]);
            if (row_tok[1] >= 0) *reinterpret_cast<float2*>(lg + 8 * kPage + 8 * k) = make_float2(x[4 * k + 2], x[4 * k + 3]);
          }
        }
        if (told & 1) {
#pragma unroll
          for (int d = 1; d < 4; d <<= 1) {
            v0 = fmaxf(v0, __shfl_xor_sync(0xffffffffu, v0, d));
            v1 = fmaxf(v1, __shfl_xor_sync(0xffffffffu, v1, d));
          }
          if (t4 == 0) {
            sh.half[half][row0] = v0;
            sh.half[half][row0 + 8] = v1;
          }
          // the product of the tile before is complete once its P has been handed back
          if (seg_live > 0) wait(sh.p_empty, (pl - 1) & 1);
          if (tell(2) & 2) break;
          const float n0 = fmaxf(m0, fmaxf(sh.half[0][row0], sh.half[1][row0]));
          const float n1 = fmaxf(m1, fmaxf(sh.half[0][row0 + 8], sh.half[1][row0 + 8]));
          const float c0 = n0 == -INFINITY ? 1.f : exp2f(m0 - n0), c1 = n1 == -INFINITY ? 1.f : exp2f(m1 - n1);
          m0 = n0;
          m1 = n1;
          l0 *= c0;
          l1 *= c1;
          if (seg_live > 0) {
            if (t4 == 0 && half == 0) {
              sh.corr[row0] = c0;
              sh.corr[row0 + 8] = c1;
            }
            ptx::named_bar_sync(1, kTcSoftmax);
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c16 = 8 * half; c16 < 8 * half + 8; ++c16) {
              uint32_t o[16];
              ptx::tmem_ld16(tmem + lanes + c16 * 16, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k)
                o[k] = __float_as_uint(__uint_as_float(o[k]) * sh.corr[(c16 & 3) * 16 + k]);
              ptx::tmem_st16(tmem + lanes + c16 * 16, o);
            }
            ptx::tmem_wait_st();
            ptx::tc_fence_before();
          }
          weigh();
        }
        l0 += s0;
        l1 += s1;
        // the one P buffer is free once the product of the last tile has read it
        if (pl > 0) wait(sh.p_empty, (pl - 1) & 1);
        unsigned char* pr = p_ptr + row0 * 128 + 4 * t4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int chunk = ((4 * half + k) ^ (g & 7)) << 4;
          *reinterpret_cast<uint32_t*>(pr + chunk) = pk[2 * k];
          *reinterpret_cast<uint32_t*>(pr + 8 * 128 + chunk) = pk[2 * k + 1];
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(smem_u32(&sh.p_full));
        ++pl;
        ++seg_live;
      }
      const bool ends = tile.last != 0;
      if (ends || i == n - 1) {
        // ------------------ end of this CTA's segment of the request ------------------
        if (seg_live > 0) wait(sh.p_empty, (pl - 1) & 1);
        const bool whole = ends && first_j == 0;
        float* part = whole ? nullptr : paged_part(a, kTcRows, rb, range, first_j == 0 ? 1 : 0);
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, d);
          l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        if (t4 == 0) {
          sh.half[half][row0] = l0;
          sh.half[half][row0 + 8] = l1;
        }
        if (tell(3) & 2) break;
        if (t4 == 0 && half == 0) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = row0 + 8 * e, r = rb * kTcRows + row;
            const float l = sh.half[0][row] + sh.half[1][row], m = e ? m1 : m0;
            sh.inv[row] = l == 0.f ? 0.f : 1.f / l;         // a row that sees nothing: output 0, lse -inf
            if (r >= a.rows) continue;
            if (whole) {
              a.lse[(size_t)tile.b * a.rows + r] = l == 0.f ? -INFINITY : m + log2f(l);
            } else {
              part[(size_t)kTcRows * kCkv + row] = l == 0.f ? -INFINITY : m;
              part[(size_t)kTcRows * (kCkv + 1) + row] = l;
            }
          }
        }
        ptx::named_bar_sync(1, kTcSoftmax);
        ptx::tc_fence_after();
        const int rows_here = min(kTcRows, a.rows - rb * kTcRows);
        // a lane has an output column, a register a row: partial results are stored four rows at a time, [16][512][4]
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int block = 2 * half + (c >> 1), r0 = 32 * (c & 1);
          const int col = block * 128 + quarter * 32 + lane;
          uint32_t o[32];
          if (seg_live > 0) {
            ptx::tmem_ld32(tmem + lanes + block * kTcRows + r0, o);
            ptx::tmem_wait_ld();
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0u;
          }
          if (whole) {
            __nv_bfloat16* dst = a.out + ((size_t)tile.b * a.rows + rb * kTcRows + r0) * kCkv + col;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (r0 + k < rows_here) dst[(size_t)k * kCkv] = __float2bfloat16_rn(__uint_as_float(o[k]) * sh.inv[r0 + k]);
          } else {
            uint4* dst = reinterpret_cast<uint4*>(part) + (size_t)(r0 >> 2) * kCkv + col;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              dst[(size_t)k * kCkv] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        }
        ptx::tc_fence_before();
        ptx::named_bar_sync(1, kTcSoftmax);          // O^T and sh.inv may be written again
      }
    }
    if (lost) {
      sh.abort_flag = 1;
      if (lane == 0) raise_status(a.status, DSA_STATUS_WAIT_TIMEOUT);
    }
  } else if (n > 0 && warp == 8) {
    // ============================ first products ============================
    // The whole warp runs this, its lanes' descriptors in uniform registers; one lane issues.
    const uint32_t elected = ptx::elect_one();
    const uint64_t dq = ptx::smem_desc_sw128(q_addr, 16, 1024), dk = ptx::smem_desc_sw128(kv_addr, 16, 1024);
    int cur_b = -1, nq = 0;
    bool ok = true;
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(smem_u32(&bar), parity) ? 1 : 0);
    };
    for (int i = 0; i < n && ok; ++i) {
      const int s = i & 1, phase = (i >> 1) & 1;
      wait(sh.full[s][0], phase);
      if (!ok) break;
      const TcTile tile = sh.tile[s];
      if (tile.b != cur_b) {
        cur_b = tile.b;
        wait(sh.q_full, nq & 1);
        ++nq;
      }
      wait(sh.s_empty[s], phase ^ 1);
      if (!ok) break;
      if (tile.live) {
        const uint32_t d = tmem + kTcSCol + s * 64;
        const uint64_t ka = dk + (uint32_t)((s * kTcPage) >> 4);
        ptx::tc_fence_after();
#pragma unroll
        for (int g = 0; g < kTcGroups; ++g) {
          if (g > 0) wait(sh.full[s][g], phase);
#pragma unroll
          for (int k = 8 * g; k < (g == kTcGroups - 1 ? 36 : 8 * g + 8); ++k)
            ptx::mma_bf16_warp(elected, d, dq + (((k >> 2) * kTcBlock + (k & 3) * 32) >> 4),
                               ka + (((k >> 2) * kTcBlock + (k & 3) * 32) >> 4), kTcIdescQK, k ? 1u : 0u);
        }
        if (elected) ptx::tc_commit(smem_u32(&sh.s_full[s]));
      } else if (elected) {
        ptx::mbar_arrive(smem_u32(&sh.s_full[s]));   // nothing to multiply
      }
      if ((tile.last || i == n - 1) && elected) ptx::tc_commit(smem_u32(&sh.q_empty));
      __syncwarp();
    }
    if (!ok && lane == 0) {
      sh.abort_flag = 1;
      raise_status(a.status, DSA_STATUS_WAIT_TIMEOUT);
    }
    __syncwarp();
  } else if (n > 0 && warp == 9) {
    // ============================ second products ============================
    const uint32_t elected = ptx::elect_one();
    const uint64_t dv = ptx::smem_desc_sw128(kv_addr, kTcBlock, 1024), dp = ptx::smem_desc_sw128(p_addr, 16, 1024);
    int cur_b = -1, np = 0;
    uint32_t acc = 0;
    bool ok = true;
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(smem_u32(&bar), parity) ? 1 : 0);
    };
    for (int i = 0; i < n && ok; ++i) {
      const int s = i & 1, phase = (i >> 1) & 1;
      wait(sh.full[s][0], phase);
      if (!ok) break;
      const TcTile tile = sh.tile[s];
      if (tile.b != cur_b) {
        cur_b = tile.b;
        acc = 0;                                     // the request's first product overwrites O^T
      }
      if (tile.live) {
        wait(sh.p_full, np & 1);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint64_t va = dv + (uint32_t)((s * kTcPage) >> 4);
#pragma unroll
        for (int c = 0; c < kTcGroups; ++c) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            ptx::mma_bf16_warp(elected, tmem + c * kTcRows, va + ((2 * c * kTcBlock + ks * 2048) >> 4),
                               dp + ((ks * 32) >> 4), kTcIdescPV, ks == 0 ? acc : 1u);
          if (elected) ptx::tc_commit(smem_u32(&sh.empty[s][c]));
        }
        if (elected) ptx::tc_commit(smem_u32(&sh.p_empty));
        ++np;
        acc = 1;
      } else {
        // nothing to multiply; a group is handed back once the producer is past it, never before
        for (int c = 1; c < kTcGroups; ++c) wait(sh.full[s][c], phase);
        if (ok && elected)
          for (int c = 0; c < kTcGroups; ++c) ptx::mbar_arrive(smem_u32(&sh.empty[s][c]));
      }
      __syncwarp();
    }
    if (!ok && lane == 0) {
      sh.abort_flag = 1;
      raise_status(a.status, DSA_STATUS_WAIT_TIMEOUT);
    }
    __syncwarp();
  } else if (n > 0) {
    // ============================ TMA producer ============================
    int ib = sh.range.start_b, ij = sh.range.start_j, cbase = ij, qb = -1, nq = 0;
    int ilen = paged_len(__ldg(a.seq_lens + ib), a.max_pages), itiles = paged_tiles(ilen, a.max_pages);
    int cur, nb = 0, nc = 0, nxt = -1, nlen = 0;
    auto lookup = [&](int b, int c) {
      return b < a.batch && c + lane < a.max_pages ? __ldg(a.block_table + (int64_t)b * a.table_stride + c + lane) : -1;
    };
    auto look_ahead = [&]() {
      const bool same = cbase + 32 < itiles;
      nb = same ? ib : ib + 1;
      nc = same ? cbase + 32 : 0;
      nxt = lookup(nb, nc);
      nlen = nb < a.batch ? paged_len(__ldg(a.seq_lens + nb), a.max_pages) : 0;
    };
    auto ask_l2 = [&](int page) {
      if (page >= 0 && page < a.num_pages) {          // 4 KB per lane
        if (lane < 16) ptx::bulk_prefetch_l2(ckv + (size_t)page * (kPage * kCkv) + lane * 2048, 4096);
        else if (lane < 18) ptx::bulk_prefetch_l2(kpe + (size_t)page * (kPage * kKpe) + (lane - 16) * 2048, 4096);
      }
    };
    cur = lookup(ib, cbase);
    look_ahead();
    bool ok = true;
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      if (ok && !(!sh.abort_flag && ptx::mbar_wait(smem_u32(&bar), parity))) {
        if (!sh.abort_flag) {
          sh.abort_flag = 1;
          raise_status(a.status, DSA_STATUS_WAIT_TIMEOUT);
        }
        ok = false;
      }
      return ok;
    };
    for (int i = 0; i < n; ++i) {
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
      const int s = i & 1, phase = (i >> 1) & 1;
      const int page = __shfl_sync(0xffffffffu, cur, ij - cbase);
      const bool held = ilen > 0, live = held && page >= 0 && page < a.num_pages;
      if (lane == 0) {
        if (ok && ib != qb) {
          // q of the request, once the products of the one before are done with the buffer; rows behind the
          // request's last are another request's, or zeros behind the tensor's end, and see nothing
          if (wait(sh.q_empty, (nq & 1) ^ 1)) {
            const uint32_t bar = smem_u32(&sh.q_full);
            const int y = ib * a.rows + rb * kTcRows;
            ptx::mbar_expect_tx(bar, kTcPage);
#pragma unroll 1
            for (int kb = 0; kb < 8; ++kb) ptx::tma_load_2d(q_addr + kb * kTcBlock, &map_qn, kb * 64, y, bar);
            ptx::tma_load_2d(q_addr + 8 * kTcBlock, &map_qp, 0, y, bar);
            ++nq;
          }
        }
        for (int c = 0; c < kTcGroups; ++c) {
          if (!wait(sh.empty[s][c], phase ^ 1)) break;
          const uint32_t bar = smem_u32(&sh.full[s][c]);
          if (c == 0) {
            sh.tile[s] = {ib, ij, ilen, (short)(live ? 1 : 0), (short)(ij == itiles - 1 ? 1 : 0)};
            if (held && !live) raise_status(a.status, DSA_STATUS_BAD_PAGE);
          }
          if (!live) {
            ptx::mbar_arrive(bar);
            continue;
          }
          const uint32_t dst = kv_addr + s * kTcPage + 2 * c * kTcBlock;
          ptx::mbar_expect_tx(bar, (c == kTcGroups - 1 ? 3 : 2) * kTcBlock);
          ptx::tma_load_2d(dst, &map_ckv, 2 * c * 64, page * kPage, bar);
          ptx::tma_load_2d(dst + kTcBlock, &map_ckv, 2 * c * 64 + 64, page * kPage, bar);
          if (c == kTcGroups - 1) ptx::tma_load_2d(dst + 2 * kTcBlock, &map_kpe, 0, page * kPage, bar);
        }
      }
      if (i > 0 && i + kTcAhead < n) {               // a page that has no place yet
        const int k = ij + kTcAhead;
        const int later = k < itiles ? k - cbase : 32 + (nb != ib ? k - itiles : 0);
        const int v = later < 32 ? __shfl_sync(0xffffffffu, cur, later) : __shfl_sync(0xffffffffu, nxt, later - 32);
        if (k < itiles || (nb != ib && (k - itiles) * kPage < nlen)) ask_l2(v);
      }
      qb = ib;
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok) break;
      ++ij;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    if (sh.abort_flag) {                             // let the copies in flight land
      for (int k = 0; k < 64; ++k) __nanosleep(20000);
    }
    ptx::tmem_dealloc(tmem, kTcCols);
  }
}

}  // namespace

template <bool kLogits>
static cudaError_t launch_tc(const PagedArgs& a, const void* ckv, const void* kpe, const CUtensorMap (&maps)[4], cudaStream_t stream) {
  static std::atomic<uint64_t> opted{0};
  const cudaError_t e =
      opt_in_dynamic_smem(reinterpret_cast<const void*>(paged_attn_tc_kernel<kLogits>), kTcDynBytes, opted);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.grid_x, (unsigned)((a.rows + kTcRows - 1) / kTcRows));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = kTcDynBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_tc_kernel<kLogits>, maps[0], maps[1], maps[2], maps[3],
                            static_cast<const __nv_bfloat16*>(ckv), static_cast<const __nv_bfloat16*>(kpe), a);
}

cudaError_t launch_paged_attn_tc(const PagedArgs& a, const void* ckv, const void* kpe, cudaStream_t stream) {
  CUtensorMap maps[4];
  const uint64_t slots = (uint64_t)a.num_pages * kPage, rows = (uint64_t)a.batch * a.rows;
  const CUtensorMapDataType bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_tmap_2d_sw128(&maps[0], bf16, 2, ckv, kCkv, slots, 64, kPage) ||
      !make_tmap_2d_sw128(&maps[1], bf16, 2, kpe, kKpe, slots, 64, kPage) ||
      !make_tmap_2d_sw128(&maps[2], bf16, 2, a.q_nope, kCkv, rows, 64, kTcRows) ||
      !make_tmap_2d_sw128(&maps[3], bf16, 2, a.q_pe, kKpe, rows, 64, kTcRows))
    return cudaErrorInvalidValue;
  return a.logits ? launch_tc<true>(a, ckv, kpe, maps, stream) : launch_tc<false>(a, ckv, kpe, maps, stream);
}

}  // namespace dsa
