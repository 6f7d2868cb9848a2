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
#include "gfa_kv4_sched.h"
#include "gfa_launch.h"

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

// 16 bytes of codes; ONCE: non-temporal, for tiles that no other workgroup reads.
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

}  // namespace

template <int D, bool IS_BF16, bool CAP, bool ONCE>
__global__ __launch_bounds__(kWaves * 64, D == 512 ? 1 : 2) void kv4_split_kernel(const Kv4AttnParams p) {
  using L = Kv4Layout<D>;
  constexpr int KT = D / 32;   // products of a score block
  constexpr int XB = D / 16;   // 16-row blocks of O^T, one per channel of an operand row
  constexpr int NJ = TileRegs<D>::NJ;
  __shared__ __attribute__((aligned(16))) f32x4 o_lds[kWaves][XB * 64];
  __shared__ float ml_lds[kWaves][kRows][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int head = p.hkv.rem((int)blockIdx.x);

  const Item it = find_item<kRows, false>(p, p.hkv.quot((int)blockIdx.x), lane);
  const Request& rq = it.rq;
  if (it.b < 0) {
    // No item: tokens ahead of the first request's and behind the last one's are zeros, the workgroups without an item take
    // them in turn.
    if (p.cu == nullptr) return;
    const int lead = min(max(p.cu[0], 0), p.T), n0 = min(max(p.cu[p.B], 0), p.T);
    const int64_t taken = (int64_t)it.items * p.cache.Hkv;
    const int64_t extra = (int)blockIdx.x - taken, n_extra = p.nblocks - taken;
    const int64_t pieces = ((int64_t)lead + p.T - n0) * p.Hq * (D / 8);
    for (int64_t i = extra * blockDim.x + threadIdx.x; i < pieces; i += n_extra * blockDim.x) {
      const int64_t hd = i / (D / 8), n = hd / p.Hq;
      const int t = (int)(n < lead ? n : n0 + (n - lead));
      uint16_t* at = p.o + p.n.quot(t) * p.osb + hd % p.Hq * p.osh + p.n.rem(t) * p.osn + i % (D / 8) * 8;
      *reinterpret_cast<i16x8*>(at) = i16x8{};
    }
    return;
  }

  // ---- the chunk's tiles ----
  const int per = chunk_len(rq, it.nch);
  const int2 tiles = tiles_of_rows(p, rq, it.rb * kRows, kRows);
  const int t_first = __builtin_amdgcn_readfirstlane(tiles.x + it.ch * per);
  const int t_end = __builtin_amdgcn_readfirstlane(min(tiles.y, t_first + per));
  const int tpb_log2 = p.cache.bs_log2 - 5;
  const int* table = p.table + (int64_t)it.b * p.table_stride;
  auto block_of = [&](int tile) __attribute__((always_inline)) { return table_entry(table, min(tile, t_end - 1) >> tpb_log2); };

  const int t0 = t_first + wave;
  const int b0 = t_first < t_end ? block_of(t0) : 0;
  int b1 = t_first < t_end ? block_of(t0 + kWaves) : 0;

  // ---- this lane's row: token, head, visible keys ----
  const int row = it.rb * kRows + c16;
  const int i = p.g.quot(row);
  const int qh = head * p.G + p.g.rem(row);
  const int t = rq.t0 + i;
  const bool live = i < rq.fresh && t >= 0 && t < p.T;
  const int pos = rq.len - rq.fresh + i;
  const int hi = live ? min(p.causal ? pos : rq.len - 1, (p.M << p.cache.bs_log2) - 1) : -1;
  const int lo = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
  const VisRange vis = make_range(lo, hi);

  i16x8 qf[KT];
  {
    const int tc = live ? t : 0;  // rows past the last read another's query; nothing of theirs goes out
    const uint16_t* qp = p.q + p.n.quot(tc) * p.qsb + (int64_t)qh * p.qsh + p.n.rem(tc) * p.qsn;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int k = 0; k < KT / NJ; ++k) {
        // product (j, k): lane group g holds channels 128 j + 32 g + 8 k .. (D = 64: 16 g + 8 k ..)
        const int d = D == 64 ? 16 * g + 8 * k : 128 * j + 32 * g + 8 * k;
        qf[j * (KT / NJ) + k] = *reinterpret_cast<const i16x8*>(qp + d);
      }
    }
  }

  f32x4 acc[XB];
#pragma unroll
  for (int x = 0; x < XB; ++x) acc[x] = f32x4{};
  float m_run = -INFINITY, l_run = 0.f;
  bool seen = false;  // the row sees a token of a tile this wave took
  const unsigned nan2 = IS_BF16 ? 0x7fc07fc0u : 0x7e007e00u;

  auto load = [&](int tile, int block, TileRegs<D>& r) __attribute__((always_inline)) {
    const int sub = min(tile, t_end - 1) & ((1 << tpb_log2) - 1);
    r.held = (unsigned)block < (unsigned)p.cache.num_blocks && tile < t_end;
    block = r.held ? block : 0;
    const uint8_t* kc = p.cache.codes + kv4_codes_at<D>(p.cache, block, head, 0) + sub * L::TILE_CODES;
    const uint8_t* vc = p.cache.codes + kv4_codes_at<D>(p.cache, block, head, 1) + sub * L::TILE_CODES;
    const uint8_t* ks = p.cache.scales + kv4_scales_at<D>(p.cache, block, head, 0) + sub * L::TILE_SCALES;
    const uint8_t* vs = p.cache.scales + kv4_scales_at<D>(p.cache, block, head, 1) + sub * L::TILE_SCALES;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int tok = hh * 16 + c16;
      if constexpr (D == 64) {
        const uint2 w = *reinterpret_cast<const uint2*>(kc + tok * 32 + g * 8);
        if (hh == 0) {
          r.k[0].x = w.x;
          r.k[0].y = w.y;
        } else {
          r.k[0].z = w.x;
          r.k[0].w = w.y;
        }
        r.ks[hh] = ks[tok * 2 + (g >> 1)];
      } else {
#pragma unroll
        for (int j = 0; j < NJ; ++j) r.k[hh * NJ + j] = load16<ONCE>(kc + j * 2048 + tok * 64 + g * 16);
        const uint8_t* sp = ks + tok * L::SC + g * NJ;
        if constexpr (NJ == 4) {
          r.ks[hh] = *reinterpret_cast<const unsigned*>(sp);
        } else if constexpr (NJ == 2) {
          r.ks[hh] = *reinterpret_cast<const uint16_t*>(sp);
        } else {
          r.ks[hh] = *sp;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < (D == 64 ? 1 : 2 * NJ); ++j) r.v[j] = load16<ONCE>(vc + j * 1024 + lane * 16);
    r.vs = *reinterpret_cast<const uint2*>(vs + (g * L::SC + c16 * L::PP / 32) * 8);
  };

  auto compute = [&](int tile, const TileRegs<D>& r) __attribute__((always_inline)) {
    // Two tiles' codes fill half the VGPRs at D = 512: Q and O^T live in AGPRs (left to the allocator some spill, and
    // a reload waits for every load in flight).
    if constexpr (D == 512) {
#pragma unroll
      for (int k = 0; k < KT; ++k) pin_agpr(qf[k]);
#pragma unroll
      for (int x = 0; x < XB; ++x) asm volatile("" : "+a"(acc[x]));
    }
    // ---- S^T, 16 tokens at a time ----
    f32x4 s[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      s[hh] = f32x4{};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        unsigned bits, cw[4];
        if constexpr (D == 64) {
          bits = r.ks[hh] << 23;
          cw[0] = hh == 0 ? r.k[0].x : r.k[0].z;
          cw[1] = hh == 0 ? r.k[0].y : r.k[0].w;
        } else {
          const unsigned sb = r.ks[hh];
          bits = j == 0 ? kv4_scale_bits<0>(sb) : j == 1 ? kv4_scale_bits<1>(sb) : j == 2 ? kv4_scale_bits<2>(sb) : kv4_scale_bits<3>(sb);
          const uint4 w = r.k[hh * NJ + j];
          cw[0] = w.x;
          cw[1] = w.y;
          cw[2] = w.z;
          cw[3] = w.w;
        }
        const float sc = __uint_as_float(bits);
#pragma unroll
        for (int k = 0; k < KT / NJ; ++k) {
          unsigned a[4] = {kv4_pair<IS_BF16, 0>(cw[k], sc), kv4_pair<IS_BF16, 1>(cw[k], sc),
                           kv4_pair<IS_BF16, 2>(cw[k], sc), kv4_pair<IS_BF16, 3>(cw[k], sc)};
          if (k == 0) a[0] = bits == 0x7f800000u ? nan2 : a[0];
          s[hh] = mma16<IS_BF16>(__builtin_bit_cast(i16x8, a), qf[j * (KT / NJ) + k], s[hh]);
        }
      }
    }

    // ---- softmax: this lane's row, tokens 4 g + r and 16 + 4 g + r ----
    // a tile without a block: nothing there to see
    const VisRange see = r.held ? vis : make_range(0, -1);
    seen = seen || (r.held && lo < (tile + 1) * kTile && hi >= tile * kTile);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = s[e >> 2][e & 3];
      if constexpr (CAP) v = cap_tanh(v * p.cap_a);
      x[e] = see.has(tile * kTile + (e >> 2) * 16 + 4 * g + (e & 3)) ? v * p.xs : -INFINITY;
    }
    float mt = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mt = fmaxf(mt, x[e]);
    // The maximum moves when a score passes it by more than kMargin (or is the row's first). With none it is exact, the
    // largest weight is 1 and unrounded, and nothing is slower for it; at D = 512 O^T comes out of the AGPRs to be
    // rescaled, and P may reach 2^8 instead (32 ragged requests: 95 us, exact 108; rms error 0.0019 and
    // 0.0017 of the result, 0.0016 of which its rounding gives).
    constexpr float kMargin = D == 512 ? 8.0f : 0.0f;  // log2
    mt = quad_max(mt);
    if (__builtin_amdgcn_ballot_w64(mt > m_run + (m_run == -INFINITY ? 0.f : kMargin)) != 0) {
      const float m_new = fmaxf(m_run, mt);
      const float a = m_new == -INFINITY ? 0.f : fast_exp2(m_run - m_new);
      l_run *= a;
#pragma unroll
      for (int xb = 0; xb < XB; ++xb) acc[xb] *= a;
      m_run = m_new;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    i16x8 pb;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pb[e] = to16<IS_BF16>(fast_exp2(x[e] - m_use));
    }
    l_run = kv4_add_weights<IS_BF16>(pb, l_run);

    // ---- O^T += V^T P^T ----
    float sc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned w = e < 4 ? r.vs.x : r.vs.y;
      const unsigned bits = (e & 3) == 0 ? kv4_scale_bits<0>(w) : (e & 3) == 1 ? kv4_scale_bits<1>(w) : (e & 3) == 2 ? kv4_scale_bits<2>(w) : kv4_scale_bits<3>(w);
      // finite whatever the byte: P is 0 where a row does not see the token, and 0 times that stays 0
      sc[e] = __uint_as_float(min(bits, (unsigned)Kv4Range<IS_BF16>::hi << 23));
    }
    auto products = [&](auto sel, int x0, const unsigned (&cw)[8]) __attribute__((always_inline)) {
      constexpr int SEL = decltype(sel)::value;
      unsigned q[8], even[4], odd[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = kv4_pair<IS_BF16, SEL>(cw[e], sc[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        even[e] = __builtin_amdgcn_perm(q[2 * e + 1], q[2 * e], 0x05040100u);
        odd[e] = __builtin_amdgcn_perm(q[2 * e + 1], q[2 * e], 0x07060302u);
      }
      acc[x0] = mma16<IS_BF16>(__builtin_bit_cast(i16x8, even), pb, acc[x0]);
      acc[x0 + 1] = mma16<IS_BF16>(__builtin_bit_cast(i16x8, odd), pb, acc[x0 + 1]);
    };
    if constexpr (D == 64) {
      const uint4 w = r.v[0];
      const unsigned cw[8] = {w.x, w.x >> 16, w.y, w.y >> 16, w.z, w.z >> 16, w.w, w.w >> 16};
      products(std::integral_constant<int, 0>{}, 0, cw);
      products(std::integral_constant<int, 1>{}, 2, cw);
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint4 a = r.v[2 * j], c = r.v[2 * j + 1];
        const unsigned cw[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
        products(std::integral_constant<int, 0>{}, 8 * j, cw);
        products(std::integral_constant<int, 1>{}, 8 * j + 2, cw);
        products(std::integral_constant<int, 2>{}, 8 * j + 4, cw);
        products(std::integral_constant<int, 3>{}, 8 * j + 6, cw);
      }
    }
  };

  // The wave's tiles, one loaded ahead. One copy of the body, the registers moved: few tiles a wave run it, and a
  // second copy would have to come into the instruction cache.
  if (t0 < t_end) {
    TileRegs<D> now, next;
    load(t0, b0, now);
    for (int tile = t0;;) {
      load(tile + kWaves, b1, next);
      b1 = block_of(tile + 2 * kWaves);
      compute(tile, now);
      if ((tile += kWaves) >= t_end) break;
      now = next;
    }
  }

  // ---- join the waves: each leaves its sums, each takes a quarter of the channels ----
  // A row without weight (m = -inf) keeps in l whether it saw a key: none is a zero row, keys whose scores
  // are all -inf are 0 / 0 as in the formula. Against a finite maximum either weighs nothing.
  float l_row = quad_sum(l_run);
  if (m_run == -INFINITY && l_row == 0.f && seen) l_row = 1.f;
  if (g == 0) {
    ml_lds[wave][c16][0] = m_run;
    ml_lds[wave][c16][1] = l_row;
  }
#pragma unroll
  for (int x = 0; x < XB; ++x) o_lds[wave][x * 64 + lane] = acc[x];
  __syncthreads();
  float m_all = -INFINITY, m_w[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    m_w[w] = ml_lds[w][c16][0];
    m_all = fmaxf(m_all, m_w[w]);
  }
  const float m_use = m_all == -INFINITY ? 0.f : m_all;
  float l_all = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    m_w[w] = fast_exp2(m_w[w] - m_use);
    l_all += ml_lds[w][c16][1] * (m_all == -INFINITY ? 1.f : m_w[w]);
  }
  constexpr int XW = XB / kWaves;  // this wave's: channels (4 g + r) PP + wave XW ..
  f32x4 o[XW];
#pragma unroll
  for (int x = 0; x < XW; ++x) {
    o[x] = f32x4{};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) o[x] += o_lds[w][(wave * XW + x) * 64 + lane] * m_w[w];
  }

  const int d0 = 4 * g * L::PP + wave * XW;
  if (it.nch > 1) {
    if ((unsigned)it.slot >= (unsigned)p.slots) return;
    const int64_t at = ((int64_t)it.slot * p.cache.Hkv + head) * kRows + c16;
    if (live) {
      typedef float vec __attribute__((ext_vector_type(XW)));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        vec v;
#pragma unroll
        for (int x = 0; x < XW; ++x) v[x] = o[x][r];
        *reinterpret_cast<vec*>(p.part + at * D + d0 + r * L::PP) = v;
      }
    }
    if (wave == 0 && g == 0) {
      p.part_ml[at * 2] = m_all;
      p.part_ml[at * 2 + 1] = l_all;
    }
    return;
  }
  if (!live) return;
  const bool none = m_all == -INFINITY && l_all == 0.f;
  const float inv = row_inv(m_all, l_all);
  uint16_t* op = p.o + p.n.quot(t) * p.osb + (int64_t)qh * p.osh + p.n.rem(t) * p.osn + d0;
  typedef short vec __attribute__((ext_vector_type(XW)));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    vec v;
#pragma unroll
    for (int x = 0; x < XW; ++x) v[x] = to16<IS_BF16>(none ? 0.f : o[x][r] * inv);
    *reinterpret_cast<vec*>(op + r * L::PP) = v;
  }
}

// Codes are loaded non-temporally: 64 requests at 16k, 32:8 D = 128, 170 -> 153 us, 16:8 D = 256 112 -> 98. At D = 512 only
// where a request's rows are one row block (99 -> 95 us; two, which share tiles in L2, 96 -> 107).
hipError_t launch_kv4_split(const Kv4AttnParams& p, int D, bool bf16, bool cap, bool once, hipStream_t stream) {
  auto go = [&](auto d, auto b, auto c) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value, CC = decltype(c)::value;
    const dim3 grid((unsigned)p.nblocks), wg(kWaves * 64);
    if (DD < 512 || once) {
      hipLaunchKernelGGL((kv4_split_kernel<DD, BB, CC, true>), grid, wg, 0, stream, p);
    } else {
      hipLaunchKernelGGL((kv4_split_kernel<512, BB, CC, false>), grid, wg, 0, stream, p);
    }
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
