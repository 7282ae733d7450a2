// Rotary positions with several axes, and the append of the rotated keys to the paged cache.
//
//   angle[t,i] = positions[axis(i), t] * inv_freq[i]        i < 32 pairs of the 64 rope dimensions
//   (a, b) -> (a cos - b sin, b cos + a sin) for every pair of q_pe[t,h] and of kpe[t]
// A pair is two neighbours (2i, 2i+1) or two halves (i, i+32).  ckv[t] and the rotated kpe[t] go to slot slots[t].
//
// Bound by memory (64 * 2 * 2 B per head and token, 2304 B per token for the cache rows).  The angle is a product of up to
// 31 + 24 bits and is reduced in double precision: in fp32 a position of 10^5 would already be 10^-2 off.  One
// sine and cosine per pair and warp, by the lane of that number; the lanes that rotate get theirs by shuffle.
// 16384 tokens of 16 heads (105 MB in and out), per call in a graph of many: 18.0 us, 5.8 TB/s; 17 tokens 1.6 us.
#include "common.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace dsa {

namespace {

constexpr int kRoThreads = 128;
constexpr int kRoHeads = 16;      // heads that a warp rotates

struct RotaryArgs {
  const uint4* q;
  int64_t q_token, q_head;        // strides in 16-byte units
  const uint4* ckv;
  int64_t ckv_stride;
  const uint4* kpe;
  int64_t kpe_stride;
  const int32_t* positions;
  int64_t positions_stride;
  const float* inv_freq;
  uint64_t pair_axes;             // two bits per pair
  const int32_t* slots;
  uint4* q_out;
  uint4* ckv_cache;
  uint4* kpe_cache;
  int32_t* status;
  int64_t num_slots;
  int tokens, heads, groups;
};

__device__ __forceinline__ float2 unpack(uint32_t v) {
  const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&v);
  return make_float2(__low2float(h), __high2float(h));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// cos / sin of the pairs that this lane rotates: four neighbours' pairs 4c .. 4c+3 (c = lane & 7), or eight pairs
// 8c .. 8c+7 of halves (c = lane & 3).
template <int kPairs>
__device__ __forceinline__ void spread(float co, float si, int first, float (&c)[kPairs], float (&s)[kPairs]) {
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    c[k] = __shfl_sync(0xffffffffu, co, first + k);
    s[k] = __shfl_sync(0xffffffffu, si, first + k);
  }
}

__device__ __forceinline__ uint4 turn_neighbours(uint4 v, const float (&c)[4], const float (&s)[4]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = unpack(u[k]);
    u[k] = pack(x.x * c[k] - x.y * s[k], x.y * c[k] + x.x * s[k]);
  }
  return v;
}
__device__ __forceinline__ void turn_halves(uint4& lo, uint4& hi, const float (&c)[8], const float (&s)[8]) {
  uint32_t *a = reinterpret_cast<uint32_t*>(&lo), *b = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = unpack(a[k]), y = unpack(b[k]);
    a[k] = pack(x.x * c[2 * k] - y.x * s[2 * k], x.y * c[2 * k + 1] - y.y * s[2 * k + 1]);
    b[k] = pack(y.x * c[2 * k] + x.x * s[2 * k], y.y * c[2 * k + 1] + x.y * s[2 * k + 1]);
  }
}

// One warp per (token, 16 heads) and one per token for its cache rows.  A 64-wide row is 8 chunks of 16 bytes: a lane has one
// chunk of neighbours, or the chunks c and c + 4 of halves.
template <bool kNeighbours>
__global__ void __launch_bounds__(kRoThreads)
rotary_append_kernel(const RotaryArgs a) {
  constexpr int kPairs = kNeighbours ? 4 : 8, kLanes = kNeighbours ? 8 : 4, kAtOnce = 32 / kLanes;
  constexpr int kRounds = kRoHeads / kAtOnce;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kRoThreads / 32) + (threadIdx.x >> 5);
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  if (unit >= (int64_t)a.tokens * (a.groups + 1)) return;
  // units of the heads first, then those of the cache rows
  const bool cache = unit >= (int64_t)a.tokens * a.groups;
  const int64_t first = cache ? unit - (int64_t)a.tokens * a.groups : unit;
  const int t = (int)(cache ? first : first / a.groups), grp = (int)(cache ? 0 : first % a.groups);
  const int c = lane % kLanes, sub = lane / kLanes;
  float cs[kPairs], sn[kPairs];
  auto turns = [&]() {
    const int axis = (int)((a.pair_axes >> (2 * lane)) & 3u);
    // in half turns: the remainder of a whole number of turns is exact in double
    const double half = (double)__ldg(a.positions + axis * a.positions_stride + t) *
                        ((double)__ldg(a.inv_freq + lane) * 0.31830988618379067154);
    float co, si;
    sincospif((float)(half - 2.0 * rint(0.5 * half)), &si, &co);
    spread<kPairs>(co, si, kPairs * c, cs, sn);
  };
  if (!cache) {
    uint4 x[kRounds], y[kRounds];                  // all loads first
    const uint4* q = a.q + (int64_t)t * a.q_token;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int h = grp * kRoHeads + k * kAtOnce + sub;
      if (h < a.heads) {
        x[k] = q[(int64_t)h * a.q_head + c];
        if (!kNeighbours) y[k] = q[(int64_t)h * a.q_head + c + 4];
      }
    }
    turns();
    uint4* out = a.q_out + (int64_t)t * a.heads * 8;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int h = grp * kRoHeads + k * kAtOnce + sub;
      if (h >= a.heads) continue;
      if constexpr (kNeighbours) {
        out[h * 8 + c] = turn_neighbours(x[k], cs, sn);
      } else {
        turn_halves(x[k], y[k], cs, sn);
        out[h * 8 + c] = x[k];
        out[h * 8 + c + 4] = y[k];
      }
    }
    return;
  }
  const int slot = __ldg(a.slots + t);
  if (slot < 0) return;
  if (slot >= a.num_slots) {
    if (lane == 0) raise_status(a.status, DSA_STATUS_BAD_SLOT);
    return;
  }
  const uint4 r0 = a.ckv[(int64_t)t * a.ckv_stride + lane], r1 = a.ckv[(int64_t)t * a.ckv_stride + lane + 32];
  uint4 kx = make_uint4(0, 0, 0, 0), ky = kx;
  if (sub == 0) {
    kx = a.kpe[(int64_t)t * a.kpe_stride + c];
    if (!kNeighbours) ky = a.kpe[(int64_t)t * a.kpe_stride + c + 4];
  }
  turns();
  uint4* row = a.ckv_cache + (int64_t)slot * (kCkv * 2 / 16);
  row[lane] = r0;
  row[lane + 32] = r1;
  if (sub == 0) {
    uint4* key = a.kpe_cache + (int64_t)slot * 8;
    if constexpr (kNeighbours) {
      key[c] = turn_neighbours(kx, cs, sn);
    } else {
      turn_halves(kx, ky, cs, sn);
      key[c] = kx;
      key[c + 4] = ky;
    }
  }
}

}  // namespace

cudaError_t launch_rotary_append(const void* q, int64_t q_token, int64_t q_head, const void* ckv, int64_t ckv_stride,
                                 const void* kpe, int64_t kpe_stride, const int32_t* positions, int64_t positions_stride,
                                 const float* inv_freq, uint64_t pair_axes, int interleaved, const int32_t* slots, void* q_out,
                                 void* ckv_cache, void* kpe_cache, int tokens, int heads, int64_t num_slots, int32_t* status,
                                 cudaStream_t stream) {
  RotaryArgs a = {static_cast<const uint4*>(q), q_token / 8, q_head / 8, static_cast<const uint4*>(ckv), ckv_stride / 8,
                  static_cast<const uint4*>(kpe), kpe_stride / 8, positions, positions_stride, inv_freq, pair_axes, slots,
                  static_cast<uint4*>(q_out), static_cast<uint4*>(ckv_cache), static_cast<uint4*>(kpe_cache), status, num_slots,
                  tokens, heads, (heads + kRoHeads - 1) / kRoHeads};
  const int64_t units = (int64_t)tokens * (a.groups + 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units + kRoThreads / 32 - 1) / (kRoThreads / 32)));
  cfg.blockDim = dim3(kRoThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return interleaved ? cudaLaunchKernelEx(&cfg, rotary_append_kernel<true>, a)
                     : cudaLaunchKernelEx(&cfg, rotary_append_kernel<false>, a);
}

}  // namespace dsa
