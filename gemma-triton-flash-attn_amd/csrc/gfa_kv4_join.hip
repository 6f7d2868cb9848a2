// The chunks' results of attention over the key/value cache, joined row by row, gfx950.
#include "gfa_kv4_sched.h"
#include "gfa_launch.h"

namespace gfa {

namespace {
constexpr int kTpb = 256;
}  // namespace

// A workgroup takes a slice of rows of one row block and head. LPR lanes of four channels are a group; `parts` of
// the GR groups share a row (as many as it has chunks, up to a power of two), take its chunks in turn with
// running maxima and are joined through LDS: fp32 sums in a fixed order. Bound: latency, one pass of
// loads behind the requests' lengths; every load of a lane's chunks is in flight at once. One
// request of 16k at D = 512 6.7 us, 32 ragged ones 6.3.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_join_kernel(const Kv4AttnParams p) {
  constexpr int ROWS = kSplitRows;
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
  const RowBlock blk = find_row_block<ROWS, false>(p, id / p.join_rows, lane);
  if (blk.b < 0 || blk.nch == 1) return;
  if (blk.slot < 0 || (int64_t)blk.slot + blk.nch > p.slots) return;  // cu that is no prefix sum: no such chunks
  const int rb = blk.rb;
  const int rows = min(ROWS, blk.rq.fresh * p.G - rb * ROWS);
  const int parts = min(p.join_parts, 1 << (32 - __builtin_clz(blk.nch - 1)));
  const int at_once = GR / parts;
  const int group = threadIdx.x / LPR, part = group % parts, d = slice * p.join_slice + threadIdx.x % LPR * 4;
  for (int r0 = id % p.join_rows * at_once; r0 < rows; r0 += p.join_rows * at_once) {
    const int rr = r0 + group / parts;
    const int row = rb * ROWS + rr;
    const int t = blk.rq.t0 + p.g.quot(row), qh = head * p.G + p.g.rem(row);
    const bool live = rr < rows && t >= 0 && t < p.T;
    float m = -INFINITY, l = 0.f;  // without a maximum l counts the rows' marks, see row_inv
    f32x4 o{};
    if (live) {
#pragma unroll 8
      for (int c = part; c < blk.nch; c += parts) {
        const int64_t at = (((int64_t)blk.slot + c) * p.cache.Hkv + head) * ROWS + rr;
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
        const f32x4 v = *reinterpret_cast<const f32x4*>(p.part + at * D + d);
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

// The chunk kernel's: its sums lie in the order its lanes held them (1 KB runs; per 32 rows, product row r and W
// channels: lane (h, row) W channels), and are read the same way: a wave takes runs, a lane one row's W channels
// of every chunk.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_join_large_kernel(const Kv4AttnParams p) {
  constexpr int ROWS = kv4_chunk_rows(D), CPL = D / 32, PP = D / 16, W = CPL < 4 ? CPL : 4;
  constexpr int RUNS = ROWS / 32 * 16 * (CPL / W);
  const int lane = threadIdx.x & 63;
  int id = (int)blockIdx.x;
  const int head = p.hkv.rem(id);
  id = p.hkv.quot(id);
  const RowBlock blk = find_row_block<ROWS, true>(p, id / p.join_rows, lane);
  if (blk.b < 0 || blk.nch == 1) return;
  if (blk.slot < 0 || (int64_t)blk.slot + blk.nch > p.slots) return;  // cu that is no prefix sum: no such chunks
  const int rb = blk.rq.row_blocks - 1 - blk.rb;                        // the chunk kernel takes the last rows first
  const int rows = min(ROWS, blk.rq.fresh * p.G - rb * ROWS);
  typedef float vec __attribute__((ext_vector_type(W)));
  for (int run = id % p.join_rows * (kTpb / 64) + (threadIdx.x >> 6); run < RUNS; run += p.join_rows * (kTpb / 64)) {
    const int rr = run / (16 * (CPL / W)) * 32 + (lane & 31);
    const int row = rb * ROWS + rr;
    const int t = blk.rq.t0 + p.g.quot(row), qh = head * p.G + p.g.rem(row);
    if (rr >= rows || t < 0 || t >= p.T) continue;
    float m = -INFINITY, l = 0.f;  // without a maximum l counts the rows' marks, see row_inv
    f32x4 o{};
#pragma unroll 8
    for (int c = 0; c < blk.nch; ++c) {
      const int64_t item = ((int64_t)blk.slot + c) * p.cache.Hkv + head;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (item * ROWS + rr) * 2);
      const vec v = *reinterpret_cast<const vec*>(p.part + item * (ROWS * D) + run * (64 * W) + lane * W);
      f32x4 v4{};
#pragma unroll
      for (int e = 0; e < W; ++e) v4[e] = v[e];
      join_rows(m, l, o, ml.x, ml.y, v4);
    }
    const int r = run / (CPL / W) % 16, x = run % (CPL / W) * W;
    const int idx = 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
    const bool none = m == -INFINITY && l == 0.f;
    const float inv = row_inv(m, l);
    typedef short out __attribute__((ext_vector_type(W)));
    out v;
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = to16<IS_BF16>(none ? 0.f : o[e] * inv);
    uint16_t* op = p.o + p.n.quot(t) * p.osb + (int64_t)qh * p.osh + p.n.rem(t) * p.osn;
    *reinterpret_cast<out*>(op + (idx & 15) * PP + CPL * (idx >> 4) + x) = v;
  }
}

hipError_t launch_kv4_join(const Kv4AttnParams& p, int D, bool bf16, bool large, hipStream_t stream) {
  auto go = [&](auto d, auto b) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value;
    const int slices = large ? 1 : DD / p.join_slice;
    const dim3 grid((unsigned)((int64_t)p.row_blocks * p.join_rows * slices * p.cache.Hkv));
    if (large) {
      hipLaunchKernelGGL((kv4_join_large_kernel<DD, BB>), grid, dim3(kTpb), 0, stream, p);
    } else {
      hipLaunchKernelGGL((kv4_join_kernel<DD, BB>), grid, dim3(kTpb), 0, stream, p);
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
