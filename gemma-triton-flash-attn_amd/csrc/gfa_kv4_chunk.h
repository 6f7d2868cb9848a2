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
#pragma once
#include "gfa_kv4_sched.h"

namespace gfa {

namespace {

// Tiles a step of the chunk kernel can take at once, see gfa_kv4_chunk.inc (at D = 64 no group of so few rows comes to it).
__host__ __device__ constexpr int kv4_chunk_steps(Kv4Part part, int D) { return part == kPart && D > 64 ? 2 : 1; }

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

}  // namespace gfa
