// Attention of a step's new tokens over the key/value cache in 4 bits (gfa_kv4.h), gfx950: many query rows per
// request (chunks of a prompt).
//
// A workgroup takes ROWS query rows of one request and KV head (all query heads of neighbouring tokens, so
// that causal row blocks end close together) and one chunk of the key tiles they see (gfa_kv4_sched.h; one
// chunk where the row blocks fill the GPU). Its four waves hold MT x 32 rows each:
//  * A tile's codes and scales (34 D bytes for 32 tokens; K swizzled) are copied global -> LDS once per
//    workgroup, one tile ahead, and every wave decodes what it multiplies in registers: S^T = K Q^T
//    and O^T += V^T P^T with v_mfma_f32_32x32x16, rows on lanes, P in registers in the B layout of the
//    second product. At D = 512 a tile kept decoded in LDS would cost four times the LDS reads (64 D bytes per
//    wave and product), which then take as long as the products; the codes cost a quarter, and the
//    decoding (one instruction per two elements, two for V) issues in the products' shadow. At D = 64 and 128
//    no 16-bit tiles were tried.
//  * Softmax: a running reference per row, moved when a score passes it by more than 2^kMargin, so that O^T is
//    rescaled once or twice per row and P stays within 2^kMargin. Row sums are held in 32 bits.
// Bound: issue of one wave per SIMD at D = 512, products and decoding together. 4096 tokens over 16384: 32:4 D = 512 3.6 ms
// (3.58 to 3.70 from card to card), 1.06 PFLOP/s (matrix cores 41-42% busy by their counter), 16:8 D = 256 960, 32:8 D = 128 811,
// 16:16 D = 64 558 TFLOP/s. Bound at D = 128 and 64: the vector unit, 81 and 70% busy. It issues 10, 12, 17.5 and 18 instructions a product (D = 512 to 64, the product among
// them), 7 of them for decoding (D = 64: 3.5), most of the others per score whatever D.
#include "gfa_kv4_sched.h"
#include "gfa_launch.h"

namespace gfa {

namespace {

// Tile copies of one wave: 1 KB runs of codes (K, then V) and the scales, dealt to the four waves in turn. K pieces land
// swizzled: a lane's 16-byte reads of a column of pieces then touch every bank once.
template <int D>
__device__ __forceinline__ void copy_tile(const Kv4Cache& c, int block, int head, int sub, int wave, int lane, char GFA_LDS* kt,
                                          char GFA_LDS* vt, char GFA_LDS* st) {
  using L = Kv4Layout<D>;
  constexpr int RUNS = L::TILE_CODES / 1024;  // per side
  // 16 tokens of 4 pieces a run; D = 64: 32 of 2
  const int t = D == 64 ? lane >> 1 : lane >> 2;
  const unsigned k_off = D == 64 ? t * 32 + (((lane & 1) ^ ((t >> 3) & 1)) << 4) : t * 64 + (((lane & 3) ^ ((t >> 2) & 3)) << 4);
  // one (block, head): K side, then V side
  const int side = (D / 2) << c.bs_log2, sside = (D / 32) << c.bs_log2;
  const auto rc = __builtin_amdgcn_make_buffer_rsrc(c.codes + kv4_codes_at<D>(c, block, head, 0), 0, 2 * side, 0x00020000);
#pragma unroll
  for (int i = 0; i < 2 * RUNS; i += 4) {
    const int run = i + wave;
    if (2 * RUNS >= 4 || run < 2 * RUNS) {
      const bool v = run >= RUNS;
      const int r = v ? run - RUNS : run;
      const unsigned soff = (unsigned)((v ? side : 0) + sub * L::TILE_CODES + r * 1024);
      char GFA_LDS* dst = (v ? vt : kt) + r * 1024;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rc, (void GFA_LDS*)dst, 16, v ? (unsigned)lane * 16 : k_off, soff, 0, 0);
    }
  }
  if (wave == (2 * RUNS) % 4) {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(c.scales + kv4_scales_at<D>(c, block, head, 0), 0, 2 * sside, 0x00020000);
    constexpr int LS = D / 16;  // lanes per side
    const unsigned off = (unsigned)(lane < LS ? lane * 16 : sside + (lane - LS) * 16);
    if (lane < 2 * LS) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (void GFA_LDS*)st, 16, off, sub * L::TILE_SCALES, 0, 0);
  }
}

// The lane's number, computed where it is needed (two instructions) rather than held with what derives from it: at D >=
// 256 a register more in the loop is a reload, whose wait is one for the tile copies too.
__device__ __forceinline__ int fresh_lane() { return opaque((int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u))); }

// A product of the S^T chain kept in VGPRs (O^T fills the AGPRs, and built from the builtin the chain would
// run there too), whose operand the vector unit has just decoded: two wait states until a product may
// read it. The chain's result is read behind mfma_result_fence.
template <bool IS_BF16, bool FIRST>
__device__ __forceinline__ void mma32_decoded(f32x16& c, const i16x8& a, const i16x8& b) {
  if constexpr (FIRST) {
    if constexpr (IS_BF16) {
      asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
    } else {
      asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
    }
  } else {
    if constexpr (IS_BF16) {
      asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    } else {
      asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    }
  }
}

}  // namespace

template <int D, bool IS_BF16, bool CAP, Kv4Part PART>
__global__ __launch_bounds__(256, kv4_chunk_wgs(D)) void kv4_chunk_kernel(const Kv4AttnParams p) {
  using L = Kv4Layout<D>;
  constexpr int ROWS = kv4_chunk_rows(D);
  constexpr int MT = ROWS / 128;                 // 32-row blocks per wave
  constexpr int KT = D / 16;                     // products of a score block
  constexpr int CPL = D / 32;                    // channels of an O^T operand row: 32-row blocks of O^T
  constexpr int NJ = D == 64 ? 1 : D / 128;
  constexpr bool PIN = D == 512;                 // O^T fills the AGPRs
  constexpr float kMargin = 8.0f;                // log2
  __shared__ __attribute__((aligned(1024))) char k_lds0[L::TILE_CODES], k_lds1[L::TILE_CODES];
  __shared__ __attribute__((aligned(1024))) char v_lds0[L::TILE_CODES], v_lds1[L::TILE_CODES];
  __shared__ __attribute__((aligned(1024))) char s_lds0[1024], s_lds1[1024];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  const int head = p.hkv.rem((int)blockIdx.x);

  const Item it = find_item<ROWS, true, PART>(p, p.hkv.quot((int)blockIdx.x), lane);
  if (it.b < 0) return;
  const Request& rq = it.rq;
  const int rb = rq.row_blocks - 1 - it.rb;  // the rows that see most keys first
  const int row0 = rb * ROWS;

  // ---- key tiles of this row block's chunk ----
  const int held = min(rq.len, p.M << p.cache.bs_log2);
  const int pos0 = rq.len - rq.fresh;  // position of new token 0
  const int2 tiles = tiles_of_rows(p, rq, row0, ROWS);
  const int per = chunk_len(rq, it.nch);
  const int t_first = __builtin_amdgcn_readfirstlane(tiles.x + it.ch * per);
  const int t_end = __builtin_amdgcn_readfirstlane(max(t_first, min(tiles.y, t_first + per)));

  // ---- this lane's rows ----
  // A row's token and query head; taken again for the stores rather than held through the loop.
  struct Row {
    int i, t, qh;
    bool live;
  };
  auto row_of = [&](int m, int ln) __attribute__((always_inline)) {
    const int row = row0 + (wave * MT + m) * 32 + (ln & 31);
    Row r;
    r.i = p.g.quot(row);
    r.t = rq.t0 + r.i;
    r.qh = head * p.G + p.g.rem(row);
    r.live = r.i < rq.fresh && r.t >= 0 && r.t < p.T;
    return r;
  };
  VisRange vis[MT];
  int all_lo = 0, all_hi = held;  // keys that every row of the wave sees
  i16x8 qf[MT][KT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const Row r = row_of(m, lane);
    const int pos = pos0 + r.i;
    const int last = r.live ? min(p.causal ? pos : rq.len - 1, held - 1) : -1;
    vis[m] = make_range(p.causal && p.window > 0 ? max(pos - p.window + 1, 0) : 0, last);
    const int tc = r.live ? r.t : 0;  // rows past the last read another's query; nothing of theirs goes out
    const uint16_t* qp = p.q + p.n.quot(tc) * p.qsb + (int64_t)r.qh * p.qsh + p.n.rem(tc) * p.qsn;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int u = 0; u < (D == 64 ? 1 : 2); ++u) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          qf[m][(j * 2 + u) * 4 + k] = *reinterpret_cast<const i16x8*>(qp + 128 * j + 32 * (2 * u + h) + 8 * k);
      }
    }
  }
  if (p.causal) {
    const int first = row0 + wave * MT * 32;
    all_hi = min(all_hi, pos0 + p.g.quot(first) + 1);
    if (p.window > 0) all_lo = pos0 + p.g.quot(first + MT * 32 - 1) - p.window + 1;
  }

  // the wave's, in scalar registers: what the compiler divides it keeps in vector ones
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  f32x16 acc[MT][CPL];
  float m_ref[MT], l_run[MT];
  bool seen[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int x = 0; x < CPL; ++x) acc[m][x] = f32x16{};
    m_ref[m] = -INFINITY;
    l_run[m] = 0.f;
    seen[m] = false;
  }

  const int tpb_log2 = p.cache.bs_log2 - 5;
  const int* table = p.table + (int64_t)it.b * p.table_stride;
  auto block_of = [&](int tile) __attribute__((always_inline)) { return table_entry(table, min(tile, t_end - 1) >> tpb_log2); };
  int block_next = 0;
  const unsigned n_blocks = (unsigned)p.cache.num_blocks;
  bool held_next = false;
  auto fetch = [&](int tile, int ln, char GFA_LDS* kt, char GFA_LDS* vt, char GFA_LDS* st) __attribute__((always_inline)) {
    const int block = block_next;
    block_next = block_of(tile + 1);
    const bool there = (unsigned)block < n_blocks;
    held_next = there && tile < t_end;
    copy_tile<D>(p.cache, there ? block : 0, head, tile & ((1 << tpb_log2) - 1), wave, ln, kt, vt, st);
  };

  const unsigned nan2 = IS_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
  auto step = [&](int tile, const char GFA_LDS* kt, const char GFA_LDS* vt, const char GFA_LDS* st, char GFA_LDS* kn,
                  char GFA_LDS* vn, char GFA_LDS* sn) __attribute__((always_inline)) {
    barrier_tile();
    const bool is_held = held_next;
    const int ln = fresh_lane();
    const int h = ln >> 5, l32 = ln & 31, p16 = ln & 15, hi = (ln >> 4) & 1;
    fetch(tile + 1, ln, kn, vn, sn);

    // LDS bytes of this lane: its K pieces (pair u of a chunk), its V pieces and the scale block of their channels
    const int k_row = D == 64 ? l32 * 32 : l32 * 64;
    const int k_swz = D == 64 ? (l32 >> 3) & 1 : (l32 >> 2) & 3;
    const int v_piece = p16 * 16;
    const int v_blk = p16 * L::PP / 32;

    // ---- S^T ----
    f32x16 s[MT];
    if constexpr (!PIN) {
#pragma unroll
      for (int m = 0; m < MT; ++m) s[m] = f32x16{};
    }
    // piece i = (u, j): 32 channels of a token a lane, four products; read one piece ahead
    constexpr int NU = D == 64 ? 1 : 2, NP = NU * NJ;
    auto k_piece = [&](int i) __attribute__((always_inline)) {
      const int u = i / NJ, j = i % NJ;
      return __builtin_bit_cast(uint4, lds_read16(kt, j * 2048 + k_row + (((D == 64 ? h : 2 * u + h) ^ k_swz) << 4)));
    };
    auto k_scales = [&](int u) __attribute__((always_inline)) -> unsigned {
      if constexpr (D == 64) return *reinterpret_cast<const uint8_t GFA_LDS*>(st + l32 * 2 + h);
      const char GFA_LDS* sp = st + l32 * L::SC + (2 * u + h) * NJ;
      if constexpr (NJ == 4) return *reinterpret_cast<const unsigned GFA_LDS*>(sp);
      if constexpr (NJ == 2) return *reinterpret_cast<const uint16_t GFA_LDS*>(sp);
      return *reinterpret_cast<const uint8_t GFA_LDS*>(sp);
    };
    uint4 next = k_piece(0);
    unsigned sbs[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) sbs[u] = k_scales(u);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int j = i % NJ;
      const uint4 w = next;
      if (i + 1 < NP) next = k_piece(i + 1);
      const unsigned sb = sbs[i / NJ];
      const unsigned bits = j == 0 ? kv4_scale_bits<0>(sb) : j == 1 ? kv4_scale_bits<1>(sb) : j == 2 ? kv4_scale_bits<2>(sb) : kv4_scale_bits<3>(sb);
      const float sc = __uint_as_float(bits);
      const unsigned cw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned a[4] = {kv4_pair<IS_BF16, 0>(cw[k], sc), kv4_pair<IS_BF16, 1>(cw[k], sc),
                         kv4_pair<IS_BF16, 2>(cw[k], sc), kv4_pair<IS_BF16, 3>(cw[k], sc)};
        if (k == 0) a[0] = bits == 0x7f800000u ? nan2 : a[0];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const i16x8& q = qf[m][(j * 2 + i / NJ) * 4 + k];
          if constexpr (!PIN) {
            s[m] = mma32<IS_BF16>(__builtin_bit_cast(i16x8, a), q, s[m]);
          } else if (i == 0 && k == 0) {
            mma32_decoded<IS_BF16, true>(s[m], __builtin_bit_cast(i16x8, a), q);
          } else {
            mma32_decoded<IS_BF16, false>(s[m], __builtin_bit_cast(i16x8, a), q);
          }
        }
        // few operands ahead: at two waves a SIMD and D = 256 the registers are full
        if (D == 256 && (k & 1)) __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (PIN) {
#pragma unroll
      for (int m = 0; m < MT; ++m) mfma_result_fence(s[m]);
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- softmax ----
    const int k0 = tile * kTile;
    const bool whole = is_held && k0 + kTile <= all_hi && k0 >= all_lo;
    i16x8 pb[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (CAP) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[m][r] = cap_tanh(s[m][r] * p.cap_a);
      }
      if (!whole) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[m][r] = is_held && vis[m].has(k0 + 8 * (r >> 2) + 4 * h + (r & 3)) ? s[m][r] : -INFINITY;
      }
      const int from = max(vis[m].base, k0);
      seen[m] = seen[m] || (is_held && from < k0 + kTile && vis[m].has(from));
      auto row_max = [&]() __attribute__((always_inline)) {
        float mt = s[m][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[m][r]);
        return halves_max(mt) * p.xs;
      };
      const float mt = row_max();
      if (__builtin_amdgcn_ballot_w64(mt > m_ref[m] + (m_ref[m] == -INFINITY ? 0.f : kMargin)) != 0) {
        const float m_new = fmaxf(m_ref[m], mt);
        const float a = m_new == -INFINITY ? 0.f : fast_exp2(m_ref[m] - m_new);
        l_run[m] *= a;
        m_ref[m] = m_new;
#pragma unroll
        for (int x = 0; x < CPL; ++x) {
          // by way of a whole VGPR block: scaled element by element the block would live in two AGPR blocks at once
          f32x16 c = acc[m][x];
          if constexpr (PIN) pin_vgpr(c);
          c *= a;
          if constexpr (PIN) pin_vgpr(c);
          acc[m][x] = c;
          if constexpr (PIN) {
            pin_agpr(acc[m][x]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      const float m_use = m_ref[m] == -INFINITY ? 0.f : m_ref[m];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pb[m][r >> 3][r & 7] = to16<IS_BF16>(fast_exp2(s[m][r] * p.xs - m_use));
      }
      l_run[m] = kv4_add_weights<IS_BF16>(pb[m][1], kv4_add_weights<IS_BF16>(pb[m][0], l_run[m]));
    }

    __builtin_amdgcn_sched_barrier(0);
    // ---- O^T += V^T P^T; step s2 over tokens 16 s2 .. 16 s2 + 15 ----
    unsigned vsb[2][2];  // [token group h, 2 + h][half]
#pragma unroll
    for (int g2 = 0; g2 < 2; ++g2) {
      const char GFA_LDS* sp = st + L::TILE_SCALES + ((2 * g2 + h) * L::SC + v_blk) * 8;
      vsb[g2][0] = *reinterpret_cast<const unsigned GFA_LDS*>(sp);
      vsb[g2][1] = *reinterpret_cast<const unsigned GFA_LDS*>(sp + 4);
    }
    // piece i = (s2, xx): 8 tokens of up to 8 channels a lane; read one piece ahead. Operand row (hi, p):
    // channels p PP + CPL hi + x
    constexpr int NX = D == 512 ? 2 : 1;
    auto v_read = [&](int i, unsigned (&cw)[8]) __attribute__((always_inline)) {
      const int s2 = i / NX, xx = i % NX;
#pragma unroll
      for (int g2 = 0; g2 < 2; ++g2) {
        if constexpr (D == 64) {
          const char GFA_LDS* vp = vt + (2 * g2 + h) * 256 + v_piece + s2 * 8;
          const unsigned a = *reinterpret_cast<const unsigned GFA_LDS*>(vp), b = *reinterpret_cast<const unsigned GFA_LDS*>(vp + 4);
          cw[4 * g2] = a >> (8 * hi);
          cw[4 * g2 + 1] = a >> (16 + 8 * hi);
          cw[4 * g2 + 2] = b >> (8 * hi);
          cw[4 * g2 + 3] = b >> (16 + 8 * hi);
        } else {
          const int x8 = D == 512 ? 2 * hi + xx : D == 256 ? hi : 0;
          const uint4 w = __builtin_bit_cast(uint4, lds_read16(vt, x8 * 2048 + s2 * 1024 + (2 * g2 + h) * 256 + v_piece));
          cw[4 * g2] = w.x;
          cw[4 * g2 + 1] = w.y;
          cw[4 * g2 + 2] = w.z;
          cw[4 * g2 + 3] = w.w;
        }
      }
    };
    float sc[8];
    unsigned ahead[8];
    v_read(0, ahead);
#pragma unroll
    for (int i = 0; i < 2 * NX; ++i) {
      const int s2 = i / NX, xx = i % NX;
      unsigned cw[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) cw[e] = D == 128 ? ahead[e] >> (16 * hi) : ahead[e];
      if (i + 1 < 2 * NX) v_read(i + 1, ahead);
      if (xx == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned w = vsb[e >> 2][s2];
          const unsigned bits = (e & 3) == 0 ? kv4_scale_bits<0>(w) : (e & 3) == 1 ? kv4_scale_bits<1>(w) : (e & 3) == 2 ? kv4_scale_bits<2>(w) : kv4_scale_bits<3>(w);
          // finite whatever the byte: P is 0 where a row does not see the token, and 0 times that stays 0
          sc[e] = __uint_as_float(min(bits, (unsigned)Kv4Range<IS_BF16>::hi << 23));
        }
      }
      auto products = [&](auto sel, int x0) __attribute__((always_inline)) {
        constexpr int SEL = decltype(sel)::value;
        unsigned q[8], even[4], odd[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = kv4_pair<IS_BF16, SEL>(cw[e], sc[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          even[e] = __builtin_amdgcn_perm(q[2 * e + 1], q[2 * e], 0x05040100u);
          odd[e] = __builtin_amdgcn_perm(q[2 * e + 1], q[2 * e], 0x07060302u);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          acc[m][x0] = mma32<IS_BF16>(__builtin_bit_cast(i16x8, even), pb[m][s2], acc[m][x0]);
          acc[m][x0 + 1] = mma32<IS_BF16>(__builtin_bit_cast(i16x8, odd), pb[m][s2], acc[m][x0 + 1]);
        }
      };
      products(std::integral_constant<int, 0>{}, 8 * xx);
      if constexpr (D >= 128) products(std::integral_constant<int, 1>{}, 8 * xx + 2);
      if constexpr (D >= 256) {
        products(std::integral_constant<int, 2>{}, 8 * xx + 4);
        products(std::integral_constant<int, 3>{}, 8 * xx + 6);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (PIN) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int x = 0; x < CPL; ++x) pin_agpr(acc[m][x]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  char GFA_LDS* const K0 = (char GFA_LDS*)k_lds0;
  char GFA_LDS* const K1 = (char GFA_LDS*)k_lds1;
  char GFA_LDS* const V0 = (char GFA_LDS*)v_lds0;
  char GFA_LDS* const V1 = (char GFA_LDS*)v_lds1;
  char GFA_LDS* const S0 = (char GFA_LDS*)s_lds0;
  char GFA_LDS* const S1 = (char GFA_LDS*)s_lds1;
  // Two tiles a turn, straight-line: an odd number of tiles gets one that nothing sees, and the last step a copy that
  // nothing reads.
  if (t_first < t_end) {
    block_next = block_of(t_first);
    fetch(t_first, lane, K0, V0, S0);
  }
  for (int t = t_first; t < t_end; t += 2) {
    step(t, K0, V0, S0, K1, V1, S1);
    step(t + 1, K1, V1, S1, K0, V0, S0);
  }
  drain_tile_copies();

  // ---- rows out ----
  const int ln = fresh_lane();
  const int ho = ln >> 5;
  const int64_t part_at = (int64_t)it.slot * p.cache.Hkv + head;
  constexpr int W = CPL < 4 ? CPL : 4;  // neighbouring channels stored at once
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const Row r0 = row_of(m, ln);
    float l = halves_sum(l_run[m]);
    if (m_ref[m] == -INFINITY && l == 0.f && seen[m]) l = 1.f;  // a mark, see row_inv
    if (PART != kWhole || it.nch > 1) {
      if ((unsigned)it.slot >= (unsigned)p.slots) return;
      const int64_t at = part_at * ROWS + (wave * MT + m) * 32 + (ln & 31);
      if (ho == 0) {
        p.part_ml[at * 2] = m_ref[m];
        p.part_ml[at * 2 + 1] = l;
      }
      if (t_first < t_end) {
        // in the order the lanes hold them, whole 1 KB runs (kv4_join_large_kernel): by rows a store would touch 64 of them
        float* part = p.part + (part_at * ROWS + (wave * MT + m) * 32) * D + ln * W;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
#pragma unroll
          for (int x = 0; x < CPL; x += W) {
            typedef float vec __attribute__((ext_vector_type(W)));
            vec v;
#pragma unroll
            for (int e = 0; e < W; ++e) v[e] = acc[m][x + e][r];
            *reinterpret_cast<vec*>(part + (r * (CPL / W) + x / W) * (64 * W)) = v;
          }
        }
      }
      continue;
    }
    if (!r0.live) continue;
    const bool none = m_ref[m] == -INFINITY && l == 0.f;
    const float inv = row_inv(m_ref[m], l);
    uint16_t* op = p.o + p.n.quot(r0.t) * p.osb + (int64_t)r0.qh * p.osh + p.n.rem(r0.t) * p.osn;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int idx = 8 * (r >> 2) + 4 * ho + (r & 3);
      uint16_t* d = op + (idx & 15) * L::PP + CPL * (idx >> 4);
      constexpr int WO = CPL < 8 ? CPL : 8;
#pragma unroll
      for (int x = 0; x < CPL; x += WO) {
        typedef short vec __attribute__((ext_vector_type(WO)));
        vec v;
#pragma unroll
        for (int e = 0; e < WO; ++e) v[e] = to16<IS_BF16>(none ? 0.f : acc[m][x + e][r] * inv);
        *reinterpret_cast<vec*>(d + x) = v;
      }
    }
  }
}

// Explicit instantiations: the host launch stubs must exist for each variant.
#define GFA_KV4_CHUNK_INST1(DD, PART)                                                     \
  template __global__ void kv4_chunk_kernel<DD, true, true, PART>(const Kv4AttnParams);   \
  template __global__ void kv4_chunk_kernel<DD, true, false, PART>(const Kv4AttnParams);  \
  template __global__ void kv4_chunk_kernel<DD, false, true, PART>(const Kv4AttnParams);  \
  template __global__ void kv4_chunk_kernel<DD, false, false, PART>(const Kv4AttnParams);
#define GFA_KV4_CHUNK_INST(DD)      \
  GFA_KV4_CHUNK_INST1(DD, kWhole)   \
  GFA_KV4_CHUNK_INST1(DD, kPrefix)
GFA_KV4_CHUNK_INST(64)
GFA_KV4_CHUNK_INST(128)
GFA_KV4_CHUNK_INST(256)
GFA_KV4_CHUNK_INST(512)
#undef GFA_KV4_CHUNK_INST
#undef GFA_KV4_CHUNK_INST1

hipError_t launch_kv4_chunk(const Kv4AttnParams& p, int D, bool bf16, bool cap, Kv4Part part, hipStream_t stream) {
  auto go = [&](auto d, auto b, auto c) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value, CC = decltype(c)::value;
    if (part == kPrefix) {
      hipLaunchKernelGGL((kv4_chunk_kernel<DD, BB, CC, kPrefix>), dim3((unsigned)p.nblocks), dim3(256), 0, stream, p);
    } else {
      hipLaunchKernelGGL((kv4_chunk_kernel<DD, BB, CC, kWhole>), dim3((unsigned)p.nblocks), dim3(256), 0, stream, p);
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
