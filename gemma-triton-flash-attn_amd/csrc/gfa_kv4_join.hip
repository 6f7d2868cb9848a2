// The chunks' results of attention over the key/value cache, joined row by row, gfx950.
#include "gfa_kv4_sched.h"
#include "gfa_launch.h"

namespace gfa {

// A workgroup takes rows of one row block and head, LPR lanes of four channels a row, its GR groups of lanes the
// chunks in turn: fp32 sums in a fixed order. Bound: latency. A single token over 16k keys (8 rows, 64 chunks of
// D = 512) gives 8 workgroups with eight loads a lane in flight.
template <int D, bool IS_BF16, int ROWS, bool LARGE, int TPB>
__global__ __launch_bounds__(TPB) void kv4_join_kernel(const Kv4AttnParams p) {
  constexpr int LPR = D / 4;
  constexpr int GR = TPB / LPR;
  __shared__ f32x4 o_lds[TPB];
  const int lane = threadIdx.x & 63;
  int id = (int)blockIdx.x;
  const int head = id % p.cache.Hkv;
  id /= p.cache.Hkv;
  const int first_row = id % p.join_rows;
  const RowBlock blk = find_row_block<ROWS, LARGE>(p, id / p.join_rows, lane);
  if (blk.b < 0 || blk.nch == 1) return;
  if ((int64_t)(blk.item + blk.nch) * p.cache.Hkv > p.nblocks) return;  // cu that is no prefix sum: no such chunks
  const int rb = LARGE ? blk.rq.row_blocks - 1 - blk.rb : blk.rb;       // the chunk kernel takes the last rows first
  const int rows = min(ROWS, blk.rq.fresh * p.G - rb * ROWS);
  const int part = threadIdx.x / LPR, d = threadIdx.x % LPR * 4;
  for (int rr = first_row; rr < rows; rr += p.join_rows) {
    const int row = rb * ROWS + rr;
    const int t = blk.rq.t0 + row / p.G, qh = head * p.G + row % p.G;
    if (t < 0 || t >= p.T) continue;
    auto slot = [&](int c) { return ((int64_t)(blk.item + c) * p.cache.Hkv + head) * ROWS + rr; };
    float m = -INFINITY;
    for (int c = lane; c < blk.nch; c += 64) m = fmaxf(m, p.part_ml[slot(c) * 2]);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int c = lane; c < blk.nch; c += 64)
      l += p.part_ml[slot(c) * 2 + 1] * (m == -INFINITY ? 1.f : fast_exp2(p.part_ml[slot(c) * 2] - m_use));
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x);
    f32x4 o{};
#pragma unroll 8
    for (int c = part; c < blk.nch; c += GR) {
      const float mc = p.part_ml[slot(c) * 2];
      const f32x4 v = *reinterpret_cast<const f32x4*>(p.part + slot(c) * D + d);
      // no weight: of a chunk without tiles there are no sums either
      o += mc == -INFINITY ? f32x4{} : v * fast_exp2(mc - m_use);
    }
    o_lds[threadIdx.x] = o;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int k = 1; k < GR; ++k) o += o_lds[k * LPR + threadIdx.x];
      const bool none = m == -INFINITY && l == 0.f;
      const float inv = row_inv(m, l);
      uint16_t* op = p.o + (t / p.N) * p.osb + (int64_t)qh * p.osh + (t % p.N) * p.osn + d;
      i16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to16<IS_BF16>(none ? 0.f : o[e] * inv);
      *reinterpret_cast<i16x4*>(op) = v;
    }
    __syncthreads();
  }
}

hipError_t launch_kv4_join(const Kv4AttnParams& p, int D, bool bf16, bool large, hipStream_t stream) {
  auto go = [&](auto d, auto b) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value;
    const dim3 grid((unsigned)((int64_t)p.row_blocks * p.join_rows * p.cache.Hkv));
    if (large) {
      hipLaunchKernelGGL((kv4_join_kernel<DD, BB, kv4_chunk_rows(DD), true, 256>), grid, dim3(256), 0, stream, p);
    } else {
      hipLaunchKernelGGL((kv4_join_kernel<DD, BB, kSplitRows, false, 1024>), grid, dim3(1024), 0, stream, p);
    }
  };
  auto by_type = [&](auto d) {
    if (bf16) {
      go(d, std::true_type{});
    } else {
      go(d, std::false_type{});
    }
  };
  switch (D) {
    case 64: by_type(std::integral_constant<int, 64>{}); break;
    case 128: by_type(std::integral_constant<int, 128>{}); break;
    case 256: by_type(std::integral_constant<int, 256>{}); break;
    default: by_type(std::integral_constant<int, 512>{}); break;
  }
  return hipGetLastError();
}

}  // namespace gfa
