// The key/value cache in 4 bits: format, byte order and the device helpers its kernels share.
//
// Format (OCP Microscaling, MXFP4): 32 neighbouring channels of one token and KV head share a power
// of two 2^e, held as the byte e + 127; an element is a sign and one of {0, .5, 1, 1.5, 2, 3, 4, 6},
// channel 2i in the low half of a byte, 2i + 1 in the high half. gfx950 decodes two elements,
// scale included, in one instruction (v_cvt_scalef32_pk_{bf16,f16}_fp4).
//
// Byte order. A block holds `block_size` tokens of every KV head, its bytes as (head, K | V, tiles of
// 32 tokens). Inside a tile the order is the one in which the lanes of a wave take 16-byte pieces
// as operands of v_mfma_f32_16x16x32, so that the attention kernel reads whole 1 KB runs and
// decodes in registers. With token t of the tile, channel d, PP = D / 16:
//   K (operand row = token, lane 16 g + t % 16 holds 32 channels of token t): 128 channels a chunk,
//     byte (d / 128) * 2048 + t * 64 + (d % 128) / 2; D = 64: t * 32 + d / 2
//   V (operand row p = channels p PP .. p PP + PP - 1, lane 16 g + p holds tokens 4 g + r and
//     16 + 4 g + r): byte (d % PP / 8) * 2048 + (t / 16) * 1024 + (16 g + p) * 16 + r * 4 + (d % 8) / 2 with
//     p = d / PP, g = t % 16 / 4, r = t % 4; D = 64: (16 g + p) * 16 + (t / 16) * 8 + r * 2 + (d % 4) / 2
//   scales, D bytes a tile, block c = d / 32: K t * (D / 32) + (c % 4) * (D / 128) + c / 4 (D = 64: t * 2 + c);
//     V (g * (D / 32) + c) * 8 + (t / 16) * 4 + r
// A token's bytes are its own: tokens of one tile are stored by different waves without a race.
#pragma once
#include "gfa_common.h"

namespace gfa {

// 2^e a written block can have, as the byte: 0.5 * 2^e and 6 * 2^e are finite in the 16-bit type, and
// the smallest is no subnormal of bf16.
template <bool IS_BF16>
struct Kv4Range {
  static constexpr int lo = IS_BF16 ? 127 - 125 : 127 - 23;
  static constexpr int hi = IS_BF16 ? 127 + 125 : 127 + 13;
};
constexpr int kKv4Nan = 255;  // scale byte of a block that holds an infinity or a NaN

// Division by a number that the host knows: x / d = x m >> s for x below 2^31 (m = ceil(2^s / d), s = 31 + ceil(log2 d),
// after Granlund and Montgomery). A division by a kernel argument takes some twenty instructions, and the short calls
// are made of little else.
struct Div {
  unsigned m, s, d;
  __host__ void set(unsigned divisor) {
    unsigned log2 = 0;
    while ((1ull << log2) < divisor) ++log2;
    d = divisor;
    s = 31 + log2;
    m = (unsigned)(((1ull << s) + divisor - 1) / divisor);
  }
  __device__ __forceinline__ int quot(int x) const { return (int)(((uint64_t)(unsigned)x * m) >> s); }
  __device__ __forceinline__ int rem(int x) const { return x - quot(x) * (int)d; }
};

// x / d for 0 <= x < 2^31 and d > 0 known on the device alone, rcp = 1 / d within a unit in the last place: a float's
// quotient, off by 2^-22 of itself (512) and one more at most, and by the remainder's, which is off by less than one.
__host__ __device__ __forceinline__ int quotient_by(int x, int d, float rcp) {
  // unsigned: q d may pass 2^31, the remainder does not
  unsigned q = (unsigned)((float)x * rcp);
  int r = (int)((unsigned)x - q * (unsigned)d);
  const int more = (int)((float)r * rcp);
  q += (unsigned)more;
  r -= more * d;
  q += r >= d;
  q -= r < 0;
  return (int)q;
}
__device__ __forceinline__ int quotient(int x, int d) { return quotient_by(x, d, __builtin_amdgcn_rcpf((float)d)); }

struct Kv4Cache {
  uint8_t* codes;   // (num_blocks, Hkv, 2, block_size, D / 2)
  uint8_t* scales;  // (num_blocks, Hkv, 2, block_size, D / 32)
  int num_blocks, Hkv, bs_log2;  // block_size = 1 << bs_log2 >= 32
};

template <int D>
struct Kv4Layout {
  static constexpr int PP = D / 16;              // channels of a V operand row
  static constexpr int KW = D < 128 ? D : 128;   // channels of a K chunk
  static constexpr int SC = D / 32;              // scale blocks of a token
  static constexpr int TILE_CODES = 16 * D, TILE_SCALES = D;
  // Byte of the 16-byte piece that holds channels 32 c .. 32 c + 31 of token t.
  static __device__ __forceinline__ int k_code(int t, int c) {
    return c / (KW / 32) * (16 * KW) + t * (KW / 2) + c % (KW / 32) * 16;
  }
  // Byte of the piece (4 bytes, 8 channels; D = 64: 2 bytes, 4 channels) of operand row p, piece x8.
  static __device__ __forceinline__ int v_code(int t, int p, int x8) {
    const int lane = (t & 12) * 4 + p;
    if constexpr (D == 64) return lane * 16 + (t >> 4) * 8 + (t & 3) * 2;
    return x8 * 2048 + (t >> 4) * 1024 + lane * 16 + (t & 3) * 4;
  }
  static __device__ __forceinline__ int k_scale(int t, int c) {
    if constexpr (D == 64) return t * 2 + c;
    return t * SC + (c & 3) * (D / 128) + (c >> 2);
  }
  static __device__ __forceinline__ int v_scale(int t, int c) {
    return (((t >> 2) & 3) * SC + c) * 8 + (t >> 4) * 4 + (t & 3);
  }
};

// First byte of the codes (scales) of side 0 (K) or 1 (V) of a block and head; 64-bit, a cache may pass 4 GiB.
template <int D>
__device__ __forceinline__ int64_t kv4_codes_at(const Kv4Cache& c, int block, int head, int side) {
  return ((((int64_t)block * c.Hkv + head) * 2 + side) << c.bs_log2) * (D / 2);
}
template <int D>
__device__ __forceinline__ int64_t kv4_scales_at(const Kv4Cache& c, int block, int head, int side) {
  return ((((int64_t)block * c.Hkv + head) * 2 + side) << c.bs_log2) * (D / 32);
}

// Elements 2 SEL and 2 SEL + 1 of the 8 in a dword, times the power of two in `scale`, as a pair of
// 16-bit values. Exact: a 2-bit significand.
template <bool IS_BF16, int SEL>
__device__ __forceinline__ unsigned kv4_pair(unsigned codes, float scale) {
  if constexpr (IS_BF16) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  } else {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
  }
}

// c + the sum of a row's rounded weights in p (32 bits). The weights that multiply V then add up to the sum that divides them:
// what rounding does to a row's largest weight drops out (rms error of one token over 333 keys 0.0024 of the
// result with the unrounded sum, 0.0017 with this one, which rounding the result alone gives).
template <bool IS_BF16>
__device__ __forceinline__ float kv4_add_weights(const i16x8& p, float c) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 w = __builtin_bit_cast(u32x4, p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned two = w[i];  // a copy: the compiler's bit cast of a vector's element takes element 0
    if constexpr (IS_BF16) {
      typedef __bf16 pair __attribute__((ext_vector_type(2)));
      c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, two), pair{(__bf16)1.0f, (__bf16)1.0f}, c, false);
    } else {
      typedef _Float16 pair __attribute__((ext_vector_type(2)));
      c = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, two), pair{(_Float16)1.0f, (_Float16)1.0f}, c, false);
    }
  }
  return c;
}

// Power of two of byte I of a dword of scale bytes, as a float's bits.
template <int I>
__device__ __forceinline__ unsigned kv4_scale_bits(unsigned bytes) {
  if constexpr (I == 3) return (bytes >> 1) & 0x7f800000u;
  return (bytes << (23 - 8 * I)) & 0x7f800000u;
}

struct Kv4RowsParams {
  Kv4Cache cache;
  const uint16_t *k, *v;  // write: (rows, Hkv, N, D)
  uint16_t *ko, *vo;      // read
  int64_t ksb, ksh, ksn, vsb, vsh, vsn;
  const int64_t* slots;   // (T,), T = rows * N
  int T;
  Div n, hkv;  // N, Hkv
};

struct Kv4PlanParams {
  const int *lens, *fresh, *free_ids, *used;
  int* table;
  int64_t table_stride;
  int B, M, F, bs_log2, T;
  int64_t* slots;
  int *positions, *cu, *lens_out, *used_out;
};

// Pages (gfa_kv4_pages.hip): bit maps of blocks in LDS, counted in groups of 8 words, one per thread of a workgroup.
constexpr int kKv4PagesBlocks = 1 << 18, kKv4PagesRows = 4096;  // most blocks of a pool, rows of a table
constexpr int kKv4CopyPiece = 16384;                             // bytes
constexpr int kKv4CopyArrays = 64;                               // of one launch: codes and scales of 32 layers
constexpr int kKv4ShareMost = 4096;                              // requests
inline int kv4_pages_words(int num_blocks) { return (num_blocks + 255) / 256 * 8; }
inline size_t kv4_fork_lds_words(int words, int requests, int rows) {
  return (size_t)3 * words + 2 * (words / 8) + requests + 2 * (size_t)rows;
}

struct Kv4PagesParams {
  const int *table, *lens, *parents, *keep, *used;
  int64_t table_stride;
  int B, M, rows, F, num_blocks, words, bs_log2;
  Div m;  // M
  int* free_ids;
  int *table_out, *lens_out, *used_out;
  int *src, *dst, *count;  // blocks to copy
};

struct Kv4CopyParams {
  uint8_t* base[kKv4CopyArrays];
  int64_t bytes[kKv4CopyArrays];    // of a block
  int first[kKv4CopyArrays];        // an array's first piece of a pair's
  int arrays, num_blocks, pairs;
  Div pieces;                       // of a pair
  const int *src, *dst, *count;     // count NULL: all pairs
};

struct Kv4ShareParams {
  const int *table, *lens, *cu;
  int64_t table_stride;
  int R, M, bs_log2, least;
  int *skip, *cu_out, *lens_out;
};

// Query rows of a workgroup of the split and of the chunk kernel.
constexpr int kSplitRows = 16;
constexpr int kv4_chunk_rows(int D) { return D >= 128 ? 128 : 256; }

// Workgroups of the chunk kernel that a CU holds (by their registers).
constexpr int kv4_chunk_wgs(int D) { return D == 512 ? 1 : D == 128 ? 3 : 2; }
// Of the shared prefixes' kernel (gfa_kv4_shared.hip) rows of a workgroup and workgroups of a CU that the compiler leaves registers for. With the
// chunk kernel's 256 rows at D = 64 those are two (forty drawn calls, geometric mean 16.7 us; three, with spills, 15.8; 128 rows, at least three 15.5; the
// kernel takes 108 registers, with which a CU holds four), and groups seldom have as many.
constexpr int kSharedRows = 128;
constexpr int kv4_shared_wgs(int D) { return D == 64 ? 3 : kv4_chunk_wgs(D); }

// What the attention kernels' device functions work on: a whole call; or, where requests share prefixes (gfa_kv4_share), the groups'
// prefixes as requests of their own or the requests' keys behind them.
enum Kv4Part : int { kWhole, kPart };

struct Kv4AttnParams {
  Kv4Cache cache;
  const uint16_t* q;
  uint16_t* o;
  int64_t qsb, qsh, qsn, osb, osh, osn;
  int T;       // tokens of q
  Div n, g, hkv;  // tokens per batch row of q and o, query heads per KV head, KV heads
  int each;    // without cu: new tokens of a request
  const int *table, *lens, *cu;
  int64_t table_stride;
  int B, M, Hq, G;
  int causal, window;  // window 0: none
  int window_tiles;    // most key tiles a row block of this kernel sees through the window
  float xs;     // multiplier of a score ahead of exp2: scale log2(e), or with soft-capping cap log2(e)
  float cap_a;  // scale / cap, 0: no soft-capping
  int min_tiles;  // work split, see chunk_tiles in gfa_kv4_sched.h
  float share;
  int nblocks;    // workgroups of the split or chunk grid
  int slots;      // of a split row block's chunk, per KV head (more only for a cu that is no prefix sum: left out)
  int row_limit;  // requests with more query rows than this belong to the chunk kernel
  // the join grid: most row blocks, workgroups for the rows of one, channels of each, groups of lanes that share a row
  int row_blocks, join_rows, join_slice, join_parts;
  float* part;    // (slots, Hkv, rows, D) sums and (slots, Hkv, rows, 2) row maxima and sums
  float* part_ml;
  const int* skip;  // kPart: (B) tokens of the request's prefix
};

// A call over shared prefixes (gfa_kv4_shared.hip): the sums of one part of the work, see Kv4AttnParams.
struct Kv4Sums {
  int min_tiles;
  float share;
  int nblocks, slots;
  float *part, *part_ml;
};
// A row block of a request: its chunks' sums (slot -1: it is out already), its first token and new ones, and its group's sums.
struct Kv4Join {
  int slot, nch, rb, t0, fresh;
  int group_nch, group_slot, group_blocks, group_t0, group_rows, large, unused;
};
struct Kv4SharedParams {
  Kv4AttnParams p;
  const int *group_cu, *group_lens;
  int row_limit;          // of the groups
  Kv4Sums many, few, rest;  // prefixes of groups of many rows and of few, the requests behind their prefixes
  float many_cost, apart_cost, worth, group_blocks;  // see plan_of in gfa_kv4_shared.hip
  int grid;                 // workgroups, that take items in turn
  int* joined;              // row blocks of the requests, and where their sums are
  Kv4Join* joins;
};

}  // namespace gfa
