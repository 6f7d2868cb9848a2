// The key/value cache in 4 bits (gfa_kv4.h): a step's plan, storing rows and reading them back, gfx950.
#include "gfa_kv4.h"
#include "gfa_launch.h"

namespace gfa {

namespace {

constexpr int kTpb = 256;
// One lane owns one scale block: 32 channels of a token, K and V.

__device__ __forceinline__ bool slot_ok(int64_t slot, const Kv4Cache& c) {
  return slot >= 0 && slot < (int64_t)c.num_blocks << c.bs_log2;
}

// The block's scale byte and 16 bytes of codes. amax = the largest magnitude's float bits; its exponent
// field less 2 puts amax in [4, 8) of the scale; one more where it is above 7, the midpoint of 6 and the
// next scale's 8 (rms error of normal values 11.19% of theirs, 11.50% without). The conversion
// rounds to the nearest code, ties to the even one, and saturates at 6.
template <bool IS_BF16>
__device__ __forceinline__ int kv4_encode(const i16x8 (&x)[4], unsigned (&codes)[4]) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(from16<IS_BF16>(x[i][e])) & 0x7fffffffu);
  }
  const bool bad = top >= 0x7f800000u;
  const int byte = min(max((int)((top + 0x1fffffu) >> 23) - 2, Kv4Range<IS_BF16>::lo), Kv4Range<IS_BF16>::hi);
  const float scale = __uint_as_float((unsigned)byte << 23);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[i][0]), from16<IS_BF16>(x[i][1]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[i][2]), from16<IS_BF16>(x[i][3]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[i][4]), from16<IS_BF16>(x[i][5]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, from16<IS_BF16>(x[i][6]), from16<IS_BF16>(x[i][7]), scale, 3);
    codes[i] = bad ? 0u : c;
  }
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

// Rows to the cache. A wave takes 2048 / D tokens of one head, a lane one scale block of K and of V. A
// token's slot is read by its lanes; a slot outside the cache (padding: -1) stores nothing.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_write_kernel(const Kv4RowsParams p) {
  using L = Kv4Layout<D>;
  constexpr int SC = L::SC, TPW = 64 / SC;
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * (kTpb / 64) + (threadIdx.x >> 6);
  const int head = (int)(w % p.cache.Hkv);
  const int64_t t64 = w / p.cache.Hkv * TPW + lane / SC;
  const int c = lane % SC;
  const int64_t slot = t64 < p.T ? p.slots[t64] : -1;
  const bool live = slot_ok(slot, p.cache);
  i16x8 kx[4] = {}, vx[4] = {};
  if (live) {
    const int row = (int)t64 / p.N, n = (int)t64 % p.N;
    const uint16_t* kp = p.k + row * p.ksb + head * p.ksh + n * p.ksn + 32 * c;
    const uint16_t* vp = p.v + row * p.vsb + head * p.vsh + n * p.vsn + 32 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = *reinterpret_cast<const i16x8*>(kp + 8 * i);
      vx[i] = *reinterpret_cast<const i16x8*>(vp + 8 * i);
    }
  }
  unsigned kc[4], vc[4];
  int ks = kv4_encode<IS_BF16>(kx, kc);
  const int vs = kv4_encode<IS_BF16>(vx, vc);
  // A value that is no number marks the token's first key block too: the attention kernel answers NaN to
  // whoever attends to the token, through its score, and keeps the value out of every other row.
  const uint64_t bad = __builtin_amdgcn_ballot_w64(vs == kKv4Nan);
  const uint64_t mine = (SC == 64 ? ~0ull : (1ull << SC) - 1) << (lane / SC * SC);
  if (c == 0 && (bad & mine) != 0) ks = kKv4Nan;
  if (!live) return;
  const int block = (int)(slot >> p.cache.bs_log2);
  const int off = (int)(slot & ((1 << p.cache.bs_log2) - 1));
  const int t = off & 31;
  uint8_t* kb = p.cache.codes + kv4_codes_at<D>(p.cache, block, head, 0) + (off >> 5) * L::TILE_CODES;
  uint8_t* vb = p.cache.codes + kv4_codes_at<D>(p.cache, block, head, 1) + (off >> 5) * L::TILE_CODES;
  *reinterpret_cast<uint4*>(kb + L::k_code(t, c)) = make_uint4(kc[0], kc[1], kc[2], kc[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // channels 32 c + 8 i ..
    const int d = 32 * c + 8 * i;
    if constexpr (D == 64) {
      *reinterpret_cast<uint16_t*>(vb + L::v_code(t, d / 4, 0)) = (uint16_t)vc[i];
      *reinterpret_cast<uint16_t*>(vb + L::v_code(t, d / 4 + 1, 0)) = (uint16_t)(vc[i] >> 16);
    } else {
      *reinterpret_cast<unsigned*>(vb + L::v_code(t, d / L::PP, d % L::PP / 8)) = vc[i];
    }
  }
  uint8_t* kse = p.cache.scales + kv4_scales_at<D>(p.cache, block, head, 0) + (off >> 5) * L::TILE_SCALES;
  uint8_t* vse = p.cache.scales + kv4_scales_at<D>(p.cache, block, head, 1) + (off >> 5) * L::TILE_SCALES;
  kse[L::k_scale(t, c)] = (uint8_t)ks;
  vse[L::v_scale(t, c)] = (uint8_t)vs;
}

// Rows from the cache, the same split; a slot outside the cache reads as zeros.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_read_kernel(const Kv4RowsParams p) {
  using L = Kv4Layout<D>;
  constexpr int SC = L::SC, TPW = 64 / SC;
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * (kTpb / 64) + (threadIdx.x >> 6);
  const int head = (int)(w % p.cache.Hkv);
  const int64_t t64 = w / p.cache.Hkv * TPW + lane / SC;
  const int c = lane % SC;
  if (t64 >= p.T) return;
  const int64_t slot = p.slots[t64];
  unsigned kc[4] = {}, vc[4] = {};
  int ks = 0, vs = 0;
  if (slot_ok(slot, p.cache)) {
    const int block = (int)(slot >> p.cache.bs_log2);
    const int off = (int)(slot & ((1 << p.cache.bs_log2) - 1));
    const int t = off & 31;
    const uint8_t* kb = p.cache.codes + kv4_codes_at<D>(p.cache, block, head, 0) + (off >> 5) * L::TILE_CODES;
    const uint8_t* vb = p.cache.codes + kv4_codes_at<D>(p.cache, block, head, 1) + (off >> 5) * L::TILE_CODES;
    const uint4 k4 = *reinterpret_cast<const uint4*>(kb + L::k_code(t, c));
    kc[0] = k4.x;
    kc[1] = k4.y;
    kc[2] = k4.z;
    kc[3] = k4.w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * c + 8 * i;
      if constexpr (D == 64) {
        vc[i] = *reinterpret_cast<const uint16_t*>(vb + L::v_code(t, d / 4, 0)) |
                (unsigned)*reinterpret_cast<const uint16_t*>(vb + L::v_code(t, d / 4 + 1, 0)) << 16;
      } else {
        vc[i] = *reinterpret_cast<const unsigned*>(vb + L::v_code(t, d / L::PP, d % L::PP / 8));
      }
    }
    ks = (p.cache.scales + kv4_scales_at<D>(p.cache, block, head, 0) + (off >> 5) * L::TILE_SCALES)[L::k_scale(t, c)];
    vs = (p.cache.scales + kv4_scales_at<D>(p.cache, block, head, 1) + (off >> 5) * L::TILE_SCALES)[L::v_scale(t, c)];
  }
  const int row = (int)t64 / p.N, n = (int)t64 % p.N;
  uint16_t* kp = p.ko + row * p.ksb + head * p.ksh + n * p.ksn + 32 * c;
  uint16_t* vp = p.vo + row * p.vsb + head * p.vsh + n * p.vsn + 32 * c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *reinterpret_cast<i16x8*>(kp + 8 * i) = kv4_decode8<IS_BF16>(kc[i], ks);
    *reinterpret_cast<i16x8*>(vp + 8 * i) = kv4_decode8<IS_BF16>(vc[i], vs);
  }
}

template <bool WRITE>
hipError_t launch_rows(const Kv4RowsParams& p, int D, bool bf16, hipStream_t stream) {
  const int64_t tpw = 2048 / D;
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
// one of per request. Integer sums: the same in every run.
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
