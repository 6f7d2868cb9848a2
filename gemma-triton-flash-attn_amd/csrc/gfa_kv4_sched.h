// The split of one attention call over the cache (gfa_kv4_attn.hip, gfa_kv4_chunk.hip) into work items, derived
// on the device from the requests' lengths, the same in every wave of every kernel of the call.
//
// The rows of a request and KV head are the G query heads of each of its new tokens, row r = token r / G, head r % G.
// An item is a row block of ROWS of them and a chunk of the key tiles they see. A row block of several chunks leaves
// their sums in slots of the workspace: a request is split where it has more than `per` tiles, so into fewer than
// 2 tiles / per chunks, and with per at least the call's tiles / target there are fewer than 2 target slots. Requests of up to
// row_limit rows are the split kernel's, the others the chunk kernel's (LARGE).
#pragma once
#include <type_traits>

#include "gfa_kv4.h"

namespace gfa {

constexpr int kTile = 32;  // tokens

// What a request asks for.
struct Request {
  int t0, fresh, len;  // first new token, new tokens, tokens with the new ones
  int row_blocks;      // 0: not this kernel's
  int tiles;           // most key tiles that a row block sees
};
// Its three loads go out together (one wait: their latency is a good part of a short call).
template <int ROWS, bool LARGE>
__device__ __forceinline__ Request request_of(const Kv4AttnParams& p, int b) {
  Request r{};
  const int bc = min(b, p.B - 1);
  const int* cu = p.cu != nullptr ? p.cu : p.lens;  // without cu read for nothing
  const int t0 = cu[bc], t1 = cu[p.cu != nullptr ? bc + 1 : bc], len = p.lens[bc];
  if (b >= p.B) return r;
  r.t0 = p.cu != nullptr ? t0 : b * p.each;
  r.fresh = p.cu != nullptr ? min(max((int)((unsigned)t1 - (unsigned)t0), 0), p.T) : p.each;
  r.len = max(len, 0);
  const int rows = r.fresh * p.G;
  r.row_blocks = (rows > p.row_limit) != LARGE ? 0 : (int)(((unsigned)rows + ROWS - 1) / ROWS);
  const int held = min(r.len, p.M << p.cache.bs_log2);
  const int lo = p.window > 0 ? (int)max((int64_t)r.len - r.fresh - p.window + 1, (int64_t)0) : 0;
  r.tiles = held > lo ? (held + kTile - 1) / kTile - lo / kTile : 0;
  if (p.window > 0) r.tiles = min(r.tiles, p.window_tiles);
  return r;
}
// Key tiles [x, y) that some row of the request's row block of `rows` rows from row0 on sees.
__device__ __forceinline__ int2 tiles_of_rows(const Kv4AttnParams& p, const Request& r, int row0, int rows) {
  const int i_lo = p.g.quot(row0), i_hi = min(p.g.quot(row0 + rows - 1), r.fresh - 1);
  const int pos0 = r.len - r.fresh;  // position of new token 0
  const int held = min(r.len, p.M << p.cache.bs_log2);
  const int k_hi = p.causal ? min(held, pos0 + i_hi + 1) : held;
  const int k_lo = p.window > 0 ? max(0, pos0 + i_lo - p.window + 1) : 0;
  return k_hi > k_lo ? make_int2(k_lo / kTile, (k_hi + kTile - 1) / kTile) : make_int2(0, 0);
}
// Lane src's request in every lane.
__device__ __forceinline__ Request request_from(const Request& r, int src) {
  auto at = [&](int x) { return __builtin_amdgcn_readlane(x, src); };
  return Request{at(r.t0), at(r.fresh), at(r.len), at(r.row_blocks), at(r.tiles)};
}

// Sum over the wave's lanes (the steps of wave_prefix_sum).
__device__ __forceinline__ float wave_sum(float x) {
  auto step = [&](auto ctrl, auto rows, auto bound) __attribute__((always_inline)) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, decltype(bound)::value));
  };
  constexpr std::integral_constant<int, 0xf> all{};
  constexpr std::true_type zero{};
  constexpr std::false_type keep{};
  step(std::integral_constant<int, 0x111>{}, all, zero);
  step(std::integral_constant<int, 0x112>{}, all, zero);
  step(std::integral_constant<int, 0x114>{}, all, zero);
  step(std::integral_constant<int, 0x118>{}, all, zero);
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}, keep);
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}, keep);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Key tiles per chunk: the whole call's tiles spread over about `target` workgroups, at least min_tiles each. The
// sum is a float's (a product of two counts can pass 32 bits); `share` = Hkv / target is rounded up by more than the
// sum can be off, so that the grid the host sized holds every item. The same operations in the same order wherever
// it is taken: contraction is off.
template <int ROWS, bool LARGE>
__device__ __forceinline__ int chunk_tiles(const Kv4AttnParams& p, const Request& r0, int lane) {
#pragma clang fp contract(off)
  float total = (float)r0.row_blocks * (float)r0.tiles;
  for (int b0 = 64; b0 < p.B; b0 += 64) {
    const Request r = request_of<ROWS, LARGE>(p, b0 + lane);
    const float x = (float)r.row_blocks * (float)r.tiles;
    total += x;
  }
  const float each = ceilf(wave_sum(total) * p.share);
  return __builtin_amdgcn_readfirstlane(max((int)fminf(each, 1.0e9f), p.min_tiles));
}
__device__ __forceinline__ int chunks_of(const Request& r, int per) { return max(quotient(r.tiles + per - 1, per), 1); }
// (Of a request that is the wave's.) Chunks of one length each, not full ones and a rest: the grid's last workgroups end closer together.
__device__ __forceinline__ int chunk_len(const Request& r, int nch) { return __builtin_amdgcn_readfirstlane(quotient(r.tiles + nch - 1, nch)); }

struct Item {
  Request rq;
  int b;            // -1: there is no such item
  int rb, ch, nch;  // row block, chunk of nch
  int items;        // of the whole call, where b < 0
  int slot;         // of nch > 1: its place among the items of split row blocks
};
template <int ROWS, bool LARGE>
__device__ __forceinline__ Item find_item(const Kv4AttnParams& p, int item, int lane) {
  Item it{};
  it.b = -1;
  Request r = request_of<ROWS, LARGE>(p, lane);
  const int per = chunk_tiles<ROWS, LARGE>(p, r, lane);
  for (int b0 = 0;;) {
    const int nch = chunks_of(r, per);
    const int mine = r.row_blocks * nch, split = nch > 1 ? mine : 0;
    const int s = wave_prefix_sum(mine), z = wave_prefix_sum(split);
    const int before = it.items + s - mine;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item >= before && item < before + mine);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      it.b = b0 + src;
      it.rq = request_from(r, src);
      it.nch = __builtin_amdgcn_readfirstlane(chunks_of(it.rq, per));
      const int i = item - __builtin_amdgcn_readlane(before, src);
      it.rb = __builtin_amdgcn_readfirstlane(quotient(i, it.nch));
      it.ch = i - it.rb * it.nch;
      it.slot += __builtin_amdgcn_readlane(z - split, src) + i;
      break;
    }
    it.items += __builtin_amdgcn_readlane(s, 63);
    it.slot += __builtin_amdgcn_readlane(z, 63);
    if ((b0 += 64) >= p.B) break;
    r = request_of<ROWS, LARGE>(p, b0 + lane);
  }
  return it;
}

// Row block `block` of the call, counted through the requests: rq, b, rb, nch, and the first chunk's slot.
struct RowBlock {
  Request rq;
  int b;           // -1: there is no such row block
  int rb, nch;
  int slot;
};
template <int ROWS, bool LARGE>
__device__ __forceinline__ RowBlock find_row_block(const Kv4AttnParams& p, int block, int lane) {
  RowBlock out{};
  out.b = -1;
  Request r = request_of<ROWS, LARGE>(p, lane);
  const int per = chunk_tiles<ROWS, LARGE>(p, r, lane);
  int blocks = 0;
  for (int b0 = 0;;) {
    const int s = wave_prefix_sum(r.row_blocks);
    const int nch = chunks_of(r, per), split = nch > 1 ? r.row_blocks * nch : 0;
    const int z = wave_prefix_sum(split);
    const int before = blocks + s - r.row_blocks;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(block >= before && block < before + r.row_blocks);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      out.b = b0 + src;
      out.rq = request_from(r, src);
      out.nch = __builtin_amdgcn_readfirstlane(chunks_of(out.rq, per));
      out.rb = block - __builtin_amdgcn_readlane(before, src);
      out.slot += __builtin_amdgcn_readlane(z - split, src) + out.rb * out.nch;
      break;
    }
    blocks += __builtin_amdgcn_readlane(s, 63);
    out.slot += __builtin_amdgcn_readlane(z, 63);
    if ((b0 += 64) >= p.B) break;
    r = request_of<ROWS, LARGE>(p, b0 + lane);
  }
  return out;
}

// Entry `col` of a block table row, through the scalar cache: the address is the wave's, and a scalar load's wait leaves
// the tile loads in flight alone.
__device__ __forceinline__ int table_entry(const int* row, int col) {
  typedef const int __attribute__((address_space(4))) * Scalar;
  return ((Scalar)(uintptr_t)row)[col];
}

// Adds a part's row (maximum mc, sum lc, O^T values v) to the row (m, l, o). Without a maximum on either side the
// sums are marks and add up; a part without one has no values (they may never have been written).
__device__ __forceinline__ void join_rows(float& m, float& l, f32x4& o, float mc, float lc, const f32x4& v) {
  const float mn = fmaxf(m, mc);
  const bool none = mn == -INFINITY;
  const float a = none ? 1.f : fast_exp2(m - mn), b = none ? 1.f : fast_exp2(mc - mn);
  l = l * a + lc * b;
  o = mc == -INFINITY ? o * a : o * a + v * b;
  m = mn;
}

// 1 / l of a finished row. Without weight l is a mark, not a sum: the row is 0 / 0 where it saw keys.
__device__ __forceinline__ float row_inv(float m, float l) { return m == -INFINITY ? 1.0f / (0.f * l) : 1.0f / l; }

}  // namespace gfa
