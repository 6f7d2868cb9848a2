// Attention of a step's new tokens over the key/value cache in 4 bits (gfa_kv4.h), gfx950: few query rows
// per request (single tokens, drafted tokens), split over the keys.
//
// Rows: the G query heads of a KV head for every new token of a request, row r = token r / G, head r % G;
// ROWS = 16 of them are a row block. Work item: (request, row block, chunk of the request's key tiles); a
// workgroup takes one item of one KV head, its waves take the chunk's 32-token tiles in turn.
//  * S^T = K Q^T (v_mfma_f32_16x16x32): A = 16 tokens of K decoded in registers from the 16 bytes a lane
//    loads (one tile ahead), B = the wave's resident Q rows. Rows sit on lanes, so softmax statistics are
//    per-lane values, and a lane's scores are in the B layout of O^T += V^T P^T for the token order
//    4 g + r, 16 + 4 g + r, in which V is stored. No LDS and no barrier until the end.
//  * Every wave keeps its own running maximum m, row sum l and O^T; they are joined once through LDS,
//    and the chunks' results by the join kernels from fp32 partial sums, in a fixed order.
// Bound: memory for batches (64 requests of 16k, 32:8 D = 128: 822 MB in 142 us, 5.8 TB/s), at D = 512 the decoding of
// one wave per SIMD (32 ragged requests, 32:4: 371 MB in 88 us, 4.2 TB/s), latency for one request (16k, D = 512: 13 us).
#pragma once
#include "gfa_kv4_sched.h"

namespace gfa {

namespace {

template <bool IS_BF16>
__device__ __forceinline__ f32x4 mma16(i16x8 a, i16x8 b, f32x4 c) {
  if constexpr (IS_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// Over the four lanes that hold one column of a 16 x 16 result (16 apart).
__device__ __forceinline__ float quad_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

constexpr int kRows = kSplitRows;
constexpr int kWaves = 4;

// 16 bytes of codes; ONCE: non-temporal, for tiles that no other workgroup reads, or few (gfa_kv4_shared.hip).
template <bool ONCE>
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  typedef unsigned vec __attribute__((ext_vector_type(4)));
  if constexpr (ONCE) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const vec*>(p)));
  return *reinterpret_cast<const uint4*>(p);
}

// What a lane holds of a 32-token tile.
template <int D>
struct TileRegs {
  static constexpr int NJ = D == 64 ? 1 : D / 128;
  uint4 k[D == 64 ? 1 : 2 * NJ], v[D == 64 ? 1 : 2 * NJ];  // D = 64: k holds both halves' 8 bytes
  unsigned ks[2];
  uint2 vs;
  bool held;
};

// Workgroup `extra` of n_extra without an item: tokens ahead of the first request's and behind the last one's are zeros, they
// take them in turn.
template <int D>
__device__ __forceinline__ void zero_rows(const Kv4AttnParams& p, int tid, int64_t extra, int64_t n_extra) {
  const int lead = min(max(p.cu[0], 0), p.T), n0 = min(max(p.cu[p.B], 0), p.T);
  const int64_t pieces = ((int64_t)lead + p.T - n0) * p.Hq * (D / 8);
  for (int64_t i = extra * (kWaves * 64) + tid; i < pieces; i += n_extra * (kWaves * 64)) {
    const int64_t hd = i / (D / 8), n = hd / p.Hq;
    const int t = (int)(n < lead ? n : n0 + (n - lead));
    uint16_t* at = p.o + p.n.quot(t) * p.osb + hd % p.Hq * p.osh + p.n.rem(t) * p.osn + i % (D / 8) * 8;
    *reinterpret_cast<i16x8*>(at) = i16x8{};
  }
}

}  // namespace

}  // namespace gfa
