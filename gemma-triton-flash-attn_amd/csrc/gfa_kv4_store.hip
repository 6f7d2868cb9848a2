// The key/value cache in 4 bits (gfa_kv4.h): a step's plan, storing rows and reading them back, gfx950.
#include "gfa_kv4.h"
#include "gfa_launch.h"

namespace gfa {

namespace {

constexpr int kTpb = 256;

// Rows and the cache. A lane takes 8 channels of four tokens in a row: its 16-byte pieces of K and V are loaded and
// stored in whole 1 KB runs, the four lanes of a scale block sit side by side, and where the four tokens are a quarter of
// an operand row of V (consecutive slots from a multiple of four, as a prompt's are) their codes go in one
// piece. Bound: memory. 16384 tokens of 8 heads at D = 256, 172 MB each way: stored in 31.5 us (5.4 TB/s), read in
// 26 us (6.6 TB/s); with a scale block a lane, 64-byte strides between lanes, 41 and 47 us.
template <int D>
struct Rows {
  static constexpr int LPT = D / 8;     // lanes per token
  static constexpr int GPW = 64 / LPT;  // groups of four tokens per wave
};

__device__ __forceinline__ bool slot_ok(int64_t slot, const Kv4Cache& c) {
  return slot >= 0 && slot < (int64_t)c.num_blocks << c.bs_log2;
}

// Where a lane is: head, first of its four tokens, its 8 channels; the tokens' slots (-1: none).
template <int D>
struct Place {
  int head, lane_t;  // lane within the token's lanes
  int64_t t0;
  int64_t slot[4];
  bool quad;  // the four slots are one piece of V's order
  __device__ __forceinline__ Place(const Kv4RowsParams& p) {
    const int lane = threadIdx.x & 63;
    const int w = (int)blockIdx.x * (kTpb / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    head = p.hkv.rem(w);
    t0 = ((int64_t)p.hkv.quot(w) * Rows<D>::GPW + lane / Rows<D>::LPT) * 4;
    lane_t = lane % Rows<D>::LPT;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t s = t0 + i < p.T ? p.slots[t0 + i] : -1;
      slot[i] = slot_ok(s, p.cache) ? s : -1;
    }
    quad = slot[0] >= 0 && (slot[0] & 3) == 0 && slot[1] == slot[0] + 1 && slot[2] == slot[0] + 2 && slot[3] == slot[0] + 3;
  }
};

// A slot's bytes of one head: codes and scales of K and V, from the start of its tile.
template <int D>
struct SlotBytes {
  uint8_t *k, *v, *ks, *vs;
  int t;
  __device__ __forceinline__ SlotBytes(const Kv4Cache& c, int64_t slot, int head) {
    using L = Kv4Layout<D>;
    const int block = (int)(slot >> c.bs_log2), off = (int)(slot & ((1 << c.bs_log2) - 1)), tile = off >> 5;
    t = off & 31;
    k = c.codes + kv4_codes_at<D>(c, block, head, 0) + tile * L::TILE_CODES;
    v = c.codes + kv4_codes_at<D>(c, block, head, 1) + tile * L::TILE_CODES;
    ks = c.scales + kv4_scales_at<D>(c, block, head, 0) + tile * L::TILE_SCALES;
    vs = c.scales + kv4_scales_at<D>(c, block, head, 1) + tile * L::TILE_SCALES;
  }
};

// The scale byte of the block whose four lanes each hold 8 values, and this lane's codes. amax = the largest
// magnitude's float bits; its exponent field less 2 puts amax in [4, 8) of the scale; one more where it is
// above 7, the midpoint of 6 and the next scale's 8 (rms error of normal values 11.19% of theirs, 11.50%
// without). The conversion rounds to the nearest code, ties to the even one, and saturates at 6.
template <bool IS_BF16>
__device__ __forceinline__ int kv4_encode(const i16x8& x, unsigned& codes) {
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(from16<IS_BF16>(x[e])) & 0x7fffffffu);
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));  // quad_perm [1, 0, 3, 2]
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));  // quad_perm [2, 3, 0, 1]
  const bool bad = top >= 0x7f800000u;
  const int byte = min(max((int)((top + 0x1fffffu) >> 23) - 2, Kv4Range<IS_BF16>::lo), Kv4Range<IS_BF16>::hi);
  const float scale = __uint_as_float((unsigned)byte << 23);
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[0]), from16<IS_BF16>(x[1]), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[2]), from16<IS_BF16>(x[3]), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[4]), from16<IS_BF16>(x[5]), scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[6]), from16<IS_BF16>(x[7]), scale, 3);
  codes = bad ? 0u : c;
  return bad ? kKv4Nan : byte;
}

template <bool IS_BF16>
__device__ __forceinline__ i16x8 kv4_decode8(unsigned codes, int byte) {
  const float s = __uint_as_float((unsigned)min(byte, Kv4Range<IS_BF16>::hi) << 23);
  unsigned r[4] = {kv4_pair<IS_BF16, 0>(codes, s), kv4_pair<IS_BF16, 1>(codes, s), kv4_pair<IS_BF16, 2>(codes, s),
                   kv4_pair<IS_BF16, 3>(codes, s)};
  const unsigned nan2 = IS_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = byte == kKv4Nan ? nan2 : r[i];
  return __builtin_bit_cast(i16x8, r);
}

}  // namespace

// Rows to the cache; a slot outside it (padding: -1) stores nothing.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_write_kernel(const Kv4RowsParams p) {
  using L = Kv4Layout<D>;
  constexpr int LPT = Rows<D>::LPT;
  const Place<D> at(p);
  const int lane = threadIdx.x & 63, d = 8 * at.lane_t, c = d / 32;
  i16x8 kx[4], vx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    kx[i] = vx[i] = i16x8{};
    if (at.slot[i] >= 0) {
      const int t = (int)at.t0 + i, row = p.n.quot(t), n = t - row * (int)p.n.d;
      kx[i] = *reinterpret_cast<const i16x8*>(p.k + row * p.ksb + at.head * p.ksh + n * p.ksn + d);
      vx[i] = *reinterpret_cast<const i16x8*>(p.v + row * p.vsb + at.head * p.vsh + n * p.vsn + d);
    }
  }
  unsigned kc[4], vc[4];
  int ks[4], vs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ks[i] = kv4_encode<IS_BF16>(kx[i], kc[i]);
    vs[i] = kv4_encode<IS_BF16>(vx[i], vc[i]);
    // A value that is no number marks the token's first key block too: the attention kernels answer NaN to whoever
    // attends to the token, through its score, and keep the value out of every other row.
    const uint64_t bad = __builtin_amdgcn_ballot_w64(vs[i] == kKv4Nan);
    const uint64_t mine = (LPT == 64 ? ~0ull : (1ull << LPT) - 1) << (lane / LPT * LPT);
    if (c == 0 && (bad & mine) != 0) ks[i] = kKv4Nan;
  }
  const bool first = (at.lane_t & 3) == 0;  // of its block's four lanes
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (at.slot[i] < 0) continue;
    const SlotBytes<D> b(p.cache, at.slot[i], at.head);
    *reinterpret_cast<unsigned*>(b.k + L::k_code(b.t, c) + (d & 31) / 2) = kc[i];
    if (first) b.ks[L::k_scale(b.t, c)] = (uint8_t)ks[i];
    if (at.quad) continue;
    if constexpr (D == 64) {
      *reinterpret_cast<uint16_t*>(b.v + L::v_code(b.t, d / 4, 0)) = (uint16_t)vc[i];
      *reinterpret_cast<uint16_t*>(b.v + L::v_code(b.t, d / 4 + 1, 0)) = (uint16_t)(vc[i] >> 16);
    } else {
      *reinterpret_cast<unsigned*>(b.v + L::v_code(b.t, d / L::PP, d % L::PP / 8)) = vc[i];
    }
    if (first) b.vs[L::v_scale(b.t, c)] = (uint8_t)vs[i];
  }
  if (at.quad) {
    const SlotBytes<D> b(p.cache, at.slot[0], at.head);
    if constexpr (D == 64) {
      // two operand rows of 4 channels: tokens' 2 bytes side by side
      *reinterpret_cast<uint2*>(b.v + L::v_code(b.t, d / 4, 0)) =
          make_uint2(__builtin_amdgcn_perm(vc[1], vc[0], 0x05040100u), __builtin_amdgcn_perm(vc[3], vc[2], 0x05040100u));
      *reinterpret_cast<uint2*>(b.v + L::v_code(b.t, d / 4 + 1, 0)) =
          make_uint2(__builtin_amdgcn_perm(vc[1], vc[0], 0x07060302u), __builtin_amdgcn_perm(vc[3], vc[2], 0x07060302u));
    } else {
      *reinterpret_cast<uint4*>(b.v + L::v_code(b.t, d / L::PP, d % L::PP / 8)) = make_uint4(vc[0], vc[1], vc[2], vc[3]);
    }
    if (first)
      *reinterpret_cast<unsigned*>(b.vs + L::v_scale(b.t, c)) = (unsigned)vs[0] | (unsigned)vs[1] << 8 | (unsigned)vs[2] << 16 | (unsigned)vs[3] << 24;
  }
}

// Rows from the cache; a slot outside it reads as zeros.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_read_kernel(const Kv4RowsParams p) {
  using L = Kv4Layout<D>;
  const Place<D> at(p);
  const int d = 8 * at.lane_t, c = d / 32;
  unsigned kc[4] = {}, vc[4] = {}, vs4 = 0;
  int ks[4] = {};
  if (at.quad) {
    const SlotBytes<D> b(p.cache, at.slot[0], at.head);
    if constexpr (D == 64) {
      const uint2 x = *reinterpret_cast<const uint2*>(b.v + L::v_code(b.t, d / 4, 0));
      const uint2 y = *reinterpret_cast<const uint2*>(b.v + L::v_code(b.t, d / 4 + 1, 0));
      vc[0] = __builtin_amdgcn_perm(y.x, x.x, 0x05040100u);
      vc[1] = __builtin_amdgcn_perm(y.x, x.x, 0x07060302u);
      vc[2] = __builtin_amdgcn_perm(y.y, x.y, 0x05040100u);
      vc[3] = __builtin_amdgcn_perm(y.y, x.y, 0x07060302u);
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(b.v + L::v_code(b.t, d / L::PP, d % L::PP / 8));
      vc[0] = x.x;
      vc[1] = x.y;
      vc[2] = x.z;
      vc[3] = x.w;
    }
    vs4 = *reinterpret_cast<const unsigned*>(b.vs + L::v_scale(b.t, c));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (at.slot[i] < 0) continue;
    const SlotBytes<D> b(p.cache, at.slot[i], at.head);
    kc[i] = *reinterpret_cast<const unsigned*>(b.k + L::k_code(b.t, c) + (d & 31) / 2);
    ks[i] = b.ks[L::k_scale(b.t, c)];
    if (at.quad) continue;
    if constexpr (D == 64) {
      vc[i] = *reinterpret_cast<const uint16_t*>(b.v + L::v_code(b.t, d / 4, 0)) |
              (unsigned)*reinterpret_cast<const uint16_t*>(b.v + L::v_code(b.t, d / 4 + 1, 0)) << 16;
    } else {
      vc[i] = *reinterpret_cast<const unsigned*>(b.v + L::v_code(b.t, d / L::PP, d % L::PP / 8));
    }
    vs4 |= (unsigned)b.vs[L::v_scale(b.t, c)] << (8 * i);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (at.t0 + i >= p.T) continue;
    const int t = (int)at.t0 + i, row = p.n.quot(t), n = t - row * (int)p.n.d;
    // read once by whoever asked: past the caches
    __builtin_nontemporal_store(kv4_decode8<IS_BF16>(kc[i], ks[i]), reinterpret_cast<i16x8*>(p.ko + row * p.ksb + at.head * p.ksh + n * p.ksn + d));
    __builtin_nontemporal_store(kv4_decode8<IS_BF16>(vc[i], (int)(vs4 >> (8 * i) & 255)), reinterpret_cast<i16x8*>(p.vo + row * p.vsb + at.head * p.vsh + n * p.vsn + d));
  }
}

template <bool WRITE>
hipError_t launch_rows(const Kv4RowsParams& p, int D, bool bf16, hipStream_t stream) {
  const int64_t tpw = 2048 / D;  // four tokens a group
  const int64_t waves = (p.T + tpw - 1) / tpw * p.cache.Hkv;
  const dim3 grid((unsigned)((waves + kTpb / 64 - 1) / (kTpb / 64)));
  auto go = [&](auto d, auto b) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value;
    if constexpr (WRITE) {
      hipLaunchKernelGGL((kv4_write_kernel<DD, BB>), grid, dim3(kTpb), 0, stream, p);
    } else {
      hipLaunchKernelGGL((kv4_read_kernel<DD, BB>), grid, dim3(kTpb), 0, stream, p);
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

hipError_t launch_kv4_write(const Kv4RowsParams& p, int D, bool bf16, hipStream_t s) { return launch_rows<true>(p, D, bf16, s); }
hipError_t launch_kv4_read(const Kv4RowsParams& p, int D, bool bf16, hipStream_t s) { return launch_rows<false>(p, D, bf16, s); }

// A step's plan. Every workgroup scans the requests (prefix sums of their new tokens and of the blocks
// they grow by) and keeps the sums of its own tokens' requests; workgroup 0 writes what there is
// one of per request. Integer sums: the same in every run. Bound: latency of the loads and scans behind one another
// (8 requests 3.1 to 3.5 us, 256 with about 18000 new tokens 4.8); the host takes 6 us to issue it.
namespace {
constexpr int kPlanTpb = 256;

struct Pair {
  int64_t tokens, blocks;
};
__device__ __forceinline__ int64_t blocks_of(int64_t n, int bs_log2) { return (n + (1 << bs_log2) - 1) >> bs_log2; }

// Exclusive prefix over the workgroup's threads and the total; two barriers.
__device__ __forceinline__ Pair block_scan(Pair x, Pair* sums, Pair& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Pair s = x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t a = __shfl_up(s.tokens, m), b = __shfl_up(s.blocks, m);
    if (lane >= m) {
      s.tokens += a;
      s.blocks += b;
    }
  }
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  Pair before{0, 0};
  total = Pair{0, 0};
#pragma unroll
  for (int w = 0; w < kPlanTpb / 64; ++w) {
    if (w < wave) {
      before.tokens += sums[w].tokens;
      before.blocks += sums[w].blocks;
    }
    total.tokens += sums[w].tokens;
    total.blocks += sums[w].blocks;
  }
  __syncthreads();
  return Pair{before.tokens + s.tokens - x.tokens, before.blocks + s.blocks - x.blocks};
}
}  // namespace

__global__ __launch_bounds__(kPlanTpb) void kv4_plan_kernel(const Kv4PlanParams p) {
  __shared__ Pair sums[kPlanTpb / 64];
  __shared__ int64_t r_tok[kPlanTpb], r_blk[kPlanTpb], r_len[kPlanTpb];
  const int tid = threadIdx.x;
  const int bs = 1 << p.bs_log2;
  const int64_t used = max(p.used[0], 0);
  const int64_t first = (int64_t)blockIdx.x * kPlanTpb;  // this workgroup's tokens
  const int64_t t = first + tid;
  Pair run{0, 0};
  int64_t slot = -1;
  int position = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanTpb) {
    const int b = b0 + tid;
    const int64_t len = b < p.B ? max(p.lens[b], 0) : 0;
    const int64_t add = b < p.B ? max(p.fresh[b], 0) : 0;
    const int64_t have = blocks_of(len, p.bs_log2), want = blocks_of(len + add, p.bs_log2);
    Pair total;
    const Pair pre = block_scan(Pair{add, want - have}, sums, total);
    const int64_t tok0 = run.tokens + pre.tokens, blk0 = used + run.blocks + pre.blocks;
    r_tok[tid] = tok0;
    r_blk[tid] = blk0;
    r_len[tid] = len;
    __syncthreads();
    const int nb = min(kPlanTpb, p.B - b0);
    // The request of this thread's token: the last one of the batch that starts at or before it.
    if (t >= run.tokens && t < run.tokens + total.tokens && t < p.T) {
      int lo = 0, hi = nb - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (r_tok[mid] <= t) lo = mid; else hi = mid - 1;
      }
      const int64_t pos = r_len[lo] + (t - r_tok[lo]);
      const int64_t col = pos >> p.bs_log2, held = blocks_of(r_len[lo], p.bs_log2);
      position = (int)pos;
      if (col < p.M) {
        int64_t block = -1;
        if (col < held) {
          block = p.table[(int64_t)(b0 + lo) * p.table_stride + col];
        } else if (r_blk[lo] + (col - held) < p.F) {
          block = p.free_ids[r_blk[lo] + (col - held)];
        }
        if (block >= 0) slot = (block << p.bs_log2) + (pos & (bs - 1));
      }
    }
    if (blockIdx.x == 0 && b < p.B) {
      p.cu[b] = (int)min(tok0, (int64_t)p.T);
      p.lens_out[b] = (int)min(len + add, (int64_t)0x7fffffff);
    }
    // New entries of the block tables, the workgroups taking requests in turn, a wave a request.
    for (int i = (int)blockIdx.x * (kPlanTpb / 64) + (tid >> 6); i < nb; i += (int)gridDim.x * (kPlanTpb / 64)) {
      const int64_t end = i + 1 < nb ? r_blk[i + 1] : used + run.blocks + total.blocks;
      const int64_t n = end - r_blk[i], at = blocks_of(r_len[i], p.bs_log2);
      for (int64_t j = tid & 63; j < n && at + j < p.M; j += 64) {
        const int64_t f = r_blk[i] + j;
        p.table[(int64_t)(b0 + i) * p.table_stride + at + j] = f < p.F ? p.free_ids[f] : -1;
      }
    }
    run.tokens += total.tokens;
    run.blocks += total.blocks;
    __syncthreads();
  }
  if (t < p.T) {
    p.slots[t] = slot;
    p.positions[t] = position;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.cu[p.B] = (int)min(run.tokens, (int64_t)p.T);
    p.used_out[0] = (int)min(used + run.blocks, (int64_t)0x7fffffff);
  }
}

hipError_t launch_kv4_plan(const Kv4PlanParams& p, hipStream_t stream) {
  const unsigned wgs = (unsigned)((p.T + kPlanTpb - 1) / kPlanTpb);
  hipLaunchKernelGGL(kv4_plan_kernel, dim3(wgs > 0 ? wgs : 1u), dim3(kPlanTpb), 0, stream, p);
  return hipGetLastError();
}

}  // namespace gfa
