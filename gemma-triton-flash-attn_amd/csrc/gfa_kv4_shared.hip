// Attention over the key/value cache in 4 bits for requests that share prefixes (gfa_kv4_share), gfx950.
//
// A group of requests whose tables begin with the same blocks is one request as far as those go: its rows, all of the group's
// new tokens and heads, see all of the prefix. So the prefix is read and decoded once per row block of the group instead of
// once per request, and many rows go to the matrix cores at once: 64 answers to a 16k prompt, 32:8 D = 128, are 256 rows a KV
// head, for which the chunk kernel's products replace 64 passes of the split kernel over the same codes. Behind the prefix
// every request is on its own. Softmax over both: sums with their maxima, joined as chunks of one row are.
//
// One launch computes the sums: the groups' prefixes by the chunk kernel's work (many rows) and the split kernel's (few), and the
// requests' rests by the split kernel's, as three runs of workgroups. A second launch joins a row's chunks of both.
#include "gfa_kv4_chunk.h"
#include "gfa_kv4_split.h"
#include "gfa_launch.h"

namespace gfa {

namespace {

constexpr int kTpb = 256;

template <int D, bool IS_BF16, bool CAP>
__device__ __forceinline__ void many_rows(const Kv4AttnParams& p, const int block) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr Kv4Part PART = kPart;
#include "gfa_kv4_chunk.inc"
#endif
}
template <int D, bool IS_BF16, bool CAP>
__device__ __forceinline__ void few_rows(const Kv4AttnParams& p, const int block) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr Kv4Part PART = kPart;
  constexpr bool ONCE = D < 512;  // as a call without prefixes
#include "gfa_kv4_split.inc"
#endif
}

// The call's parameters as one of the three parts has them.
__device__ __forceinline__ Kv4AttnParams part_of(const Kv4SharedParams& s, const Kv4Sums& sums, bool groups) {
  Kv4AttnParams p = s.p;
  if (groups) {
    p.cu = s.group_cu;
    p.lens = s.group_lens;
    p.skip = nullptr;
    p.causal = 0;
    p.row_limit = s.row_limit;
  }
  p.min_tiles = sums.min_tiles;
  p.share = sums.share;
  p.nblocks = sums.nblocks;
  p.slots = sums.slots;
  p.part = sums.part;
  p.part_ml = sums.part_ml;
  return p;
}

// The group of request b: where its first token is, and its sums.
struct Group {
  int t0, rows, row_blocks, nch, slot;
  bool large;
};
template <int BIG>
__device__ __forceinline__ Group find_group(const Kv4AttnParams& few, const Kv4AttnParams& many, int b, int lane) {
  Group out{};
  Request f = request_of<kSplitRows, false, kPart>(few, lane), m = request_of<BIG, true, kPart>(many, lane);
  const int per_f = chunk_tiles<kSplitRows, false, kPart>(few, f, lane), per_m = chunk_tiles<BIG, true, kPart>(many, m, lane);
  int slot_f = 0, slot_m = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    if (b0 > 0) {
      f = request_of<kSplitRows, false, kPart>(few, b0 + lane);
      m = request_of<BIG, true, kPart>(many, b0 + lane);
    }
    const int nf = chunks_of(f, per_f), nm = chunks_of(m, per_m);
    const int zf = wave_prefix_sum(f.row_blocks * nf), zm = wave_prefix_sum(m.row_blocks * nm);
    // a group's first request stands ahead of its others
    const uint64_t firsts = __builtin_amdgcn_ballot_w64(f.row_blocks + m.row_blocks > 0 && b0 + lane <= b);
    if (firsts != 0) {
      const int src = 63 - __builtin_clzll(firsts);
      auto at = [&](int x) { return __builtin_amdgcn_readlane(x, src); };
      out.large = at(m.row_blocks) > 0;
      out.t0 = at(f.t0);
      out.rows = at(f.fresh) * few.G;
      out.row_blocks = out.large ? at(m.row_blocks) : at(f.row_blocks);
      out.nch = __builtin_amdgcn_readfirstlane(out.large ? at(nm) : at(nf));
      out.slot = out.large ? slot_m + at(zm - m.row_blocks * nm) : slot_f + at(zf - f.row_blocks * nf);
    }
    slot_f += __builtin_amdgcn_readlane(zf, 63);
    slot_m += __builtin_amdgcn_readlane(zm, 63);
  }
  return out;
}

}  // namespace

template <int D, bool IS_BF16, bool CAP>
__global__ __launch_bounds__(kTpb, kv4_shared_wgs(D)) void kv4_shared_kernel(const Kv4SharedParams s) {
  int block = (int)blockIdx.x;
  if (block < s.many.nblocks) {
    many_rows<D, IS_BF16, CAP>(part_of(s, s.many, true), block);
    return;
  }
  block -= s.many.nblocks;
  const bool groups = block < s.few.nblocks;
  few_rows<D, IS_BF16, CAP>(part_of(s, groups ? s.few : s.rest, groups), groups ? block : block - s.few.nblocks);
}

// As kv4_join_kernel, of a row's chunks behind the prefix and of its row's in the group's sums. Bound: latency, two scans of
// the requests and one pass of loads.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_shared_join_kernel(const Kv4SharedParams s) {
  constexpr int ROWS = kSplitRows, BIG = kv4_chunk_rows(D);
  const Kv4AttnParams p = part_of(s, s.rest, false);
  const int LPR = p.join_slice / 4;  // a power of two
  const int GR = kTpb / LPR;
  __shared__ f32x4 o_lds[kTpb];
  __shared__ float ml_lds[kTpb / 16][2];
  const int lane = threadIdx.x & 63;
  int id = (int)blockIdx.x;
  const int head = p.hkv.rem(id);
  id = p.hkv.quot(id);
  const int slice = id % (D / p.join_slice);
  id /= D / p.join_slice;
  const RowBlock blk = find_row_block<ROWS, false, kPart>(p, id / p.join_rows, lane);
  if (blk.b < 0) return;
  if (blk.slot < 0 || (int64_t)blk.slot + blk.nch > p.slots) return;  // cu that is no prefix sum: no such chunks
  Group grp{};
  if (blk.rq.skip > 0) {
    grp = find_group<BIG>(part_of(s, s.few, true), part_of(s, s.many, true), blk.b, lane);
    if (grp.slot < 0 || (int64_t)grp.slot + (int64_t)grp.row_blocks * grp.nch > (grp.large ? s.many.slots : s.few.slots)) grp.nch = 0;
  }
  const float* const gp = grp.large ? s.many.part : s.few.part;
  const float* const gml = grp.large ? s.many.part_ml : s.few.part_ml;
  const int rb = blk.rb;
  const int rows = min(ROWS, blk.rq.fresh * p.G - rb * ROWS);
  const int all = blk.nch + grp.nch;
  const int parts = min(p.join_parts, all > 1 ? 1 << (32 - __builtin_clz(all - 1)) : 1);
  const int at_once = GR / parts;
  const int group = threadIdx.x / LPR, part = group % parts, d = slice * p.join_slice + threadIdx.x % LPR * 4;
  for (int r0 = id % p.join_rows * at_once; r0 < rows; r0 += p.join_rows * at_once) {
    const int rr = r0 + group / parts;
    const int row = rb * ROWS + rr;
    const int t = blk.rq.t0 + p.g.quot(row), hg = p.g.rem(row), qh = head * p.G + hg;
    const bool live = rr < rows && t >= 0 && t < p.T;
    float m = -INFINITY, l = 0.f;  // without a maximum l counts the rows' marks, see row_inv
    f32x4 o{};
    if (live) {
      // the row in its group: row block, and row of it
      const int row_g = (t - grp.t0) * p.G + hg, in = grp.large ? row_g % BIG : row_g % ROWS;
      const int blk_g = grp.large ? grp.row_blocks - 1 - row_g / BIG : row_g / ROWS;  // the chunk kernel takes the last rows first
      const int64_t item0 = (int64_t)grp.slot + (int64_t)blk_g * grp.nch;
      const int count = row_g >= 0 && row_g < grp.rows ? all : blk.nch;
      // one address or the other, then the load: behind a branch the loads would wait for each other
#pragma unroll 8
      for (int c = part; c < count; c += parts) {
        const int cg = c - blk.nch;
        const int64_t own = (((int64_t)blk.slot + c) * p.cache.Hkv + head) * ROWS + rr;
        const int64_t its = ((item0 + cg) * p.cache.Hkv + head) * (grp.large ? BIG : ROWS) + in;
        const int64_t at = cg < 0 ? own : its;
        const float2 ml = *reinterpret_cast<const float2*>((cg < 0 ? p.part_ml : gml) + at * 2);
        const f32x4 v = *reinterpret_cast<const f32x4*>((cg < 0 ? p.part : gp) + at * D + d);
        join_rows(m, l, o, ml.x, ml.y, v);
      }
    }
    if (parts > 1) {
      o_lds[threadIdx.x] = o;
      if (threadIdx.x % LPR == 0) {
        ml_lds[group][0] = m;
        ml_lds[group][1] = l;
      }
      __syncthreads();
      if (part == 0) {
        for (int k = 1; k < parts; ++k) join_rows(m, l, o, ml_lds[group + k][0], ml_lds[group + k][1], o_lds[threadIdx.x + k * LPR]);
      }
      __syncthreads();
    }
    if (part == 0 && live) {
      const bool none = m == -INFINITY && l == 0.f;
      const float inv = row_inv(m, l);
      uint16_t* op = p.o + p.n.quot(t) * p.osb + (int64_t)qh * p.osh + p.n.rem(t) * p.osn + d;
      i16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to16<IS_BF16>(none ? 0.f : o[e] * inv);
      *reinterpret_cast<i16x4*>(op) = v;
    }
  }
}

hipError_t launch_kv4_shared(const Kv4SharedParams& s, int D, bool bf16, bool cap, hipStream_t stream) {
  const dim3 wg(kTpb);
  const dim3 grid((unsigned)((int64_t)s.many.nblocks + s.few.nblocks + s.rest.nblocks));
  auto go = [&](auto d, auto b, auto c) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value, CC = decltype(c)::value;
    hipLaunchKernelGGL((kv4_shared_kernel<DD, BB, CC>), grid, wg, 0, stream, s);
    const dim3 join((unsigned)((int64_t)s.p.row_blocks * s.p.join_rows * (DD / s.p.join_slice) * s.p.cache.Hkv));
    hipLaunchKernelGGL((kv4_shared_join_kernel<DD, BB>), join, wg, 0, stream, s);
  };
  auto by_type = [&](auto d) {
    if (bf16 && cap) go(d, std::true_type{}, std::true_type{});
    if (bf16 && !cap) go(d, std::true_type{}, std::false_type{});
    if (!bf16 && cap) go(d, std::false_type{}, std::true_type{});
    if (!bf16 && !cap) go(d, std::false_type{}, std::false_type{});
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
