// The chunks' results of attention over the key/value cache, joined row by row, gfx950.
#include "gfa_kv4_sched.h"
#include "gfa_launch.h"

namespace gfa {

// Joins the chunks of a row: one workgroup per token and query head.
template <int D, bool IS_BF16, int ROWS, bool LARGE>
__global__ __launch_bounds__(256) void kv4_join_kernel(const Kv4AttnParams p) {
  constexpr int LPR = D / 4;         // lanes per row, four channels each
  constexpr int GR = 256 / LPR;      // chunks at a time
  __shared__ f32x4 o_lds[256];
  const int lane = threadIdx.x & 63;
  const int t = (int)(blockIdx.x / p.Hq), qh = (int)(blockIdx.x % p.Hq);
  const int head = qh / p.G;
  // the token's request
  const int per = chunk_tiles<ROWS, LARGE>(p, lane);
  int64_t items = 0, base = -1;
  Request rq{};
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const Request r = request_of<ROWS, LARGE>(p, b0 + lane);
    const int64_t mine = (int64_t)r.row_blocks * chunks_of(r, per);
    const int64_t s = wave_prefix64(mine, lane);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(t >= r.t0 && t < r.t0 + r.fresh);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      base = items + __shfl(s - mine, src);
      rq = request_of<ROWS, LARGE>(p, __builtin_amdgcn_readfirstlane(b0 + src));
      break;
    }
    items += __shfl(s, 63);
  }
  if (base < 0 || rq.row_blocks == 0) return;
  const int nch = chunks_of(rq, per);
  if (nch == 1) return;
  const int i = t - rq.t0;
  const int row = i * p.G + qh % p.G;
  const int rb = LARGE ? rq.row_blocks - 1 - row / ROWS : row / ROWS;  // the chunk kernel takes the last rows first
  const int64_t first = base + (int64_t)rb * nch;  // item of chunk 0
  if ((first + nch) * p.cache.Hkv > p.nblocks) return;       // lengths that do not fit the grid: see gfa.h
  const int rr = row % ROWS;
  auto slot = [&](int c) { return ((first + c) * p.cache.Hkv + head) * ROWS + rr; };
  float m = -INFINITY;
  for (int c = lane; c < nch; c += 64) m = fmaxf(m, p.part_ml[slot(c) * 2]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int c = lane; c < nch; c += 64)
    l += p.part_ml[slot(c) * 2 + 1] * (m == -INFINITY ? 1.f : fast_exp2(p.part_ml[slot(c) * 2] - m_use));
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x);
  f32x4 o{};
  const int part = threadIdx.x / LPR, d = threadIdx.x % LPR * 4;
  for (int c = part; c < nch; c += GR) {
    const float mc = p.part_ml[slot(c) * 2];
    if (mc == -INFINITY) continue;  // no weight (and, of a chunk without tiles, no sums)
    const float w = fast_exp2(mc - m_use);
    o += *reinterpret_cast<const f32x4*>(p.part + slot(c) * D + d) * w;
  }
  o_lds[threadIdx.x] = o;
  __syncthreads();
  if (part != 0) return;
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

hipError_t launch_kv4_join(const Kv4AttnParams& p, int D, bool bf16, bool large, hipStream_t stream) {
  auto go = [&](auto d, auto b) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value;
    constexpr int kLarge = kv4_chunk_rows(DD);
    const dim3 grid((unsigned)(p.T * p.Hq)), wg(256);
    if (large) {
      hipLaunchKernelGGL((kv4_join_kernel<DD, BB, kLarge, true>), grid, wg, 0, stream, p);
    } else {
      hipLaunchKernelGGL((kv4_join_kernel<DD, BB, 16, false>), grid, wg, 0, stream, p);
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
