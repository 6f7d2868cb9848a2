// The split of one attention call over the cache (gfa_kv4_attn.hip, gfa_kv4_chunk.hip) into work items, derived
// on the device from the requests' lengths, the same in every wave of every kernel of the call.
//
// The rows of a request and KV head are the G query heads of each of its new tokens, row r = token r / G, head r % G.
// An item is a row block of ROWS of them and a chunk of the key tiles they see. Requests of up to
// row_limit rows are the split kernel's, the others the chunk kernel's (LARGE).
#pragma once
#include "gfa_kv4.h"

namespace gfa {

constexpr int kTile = 32;  // tokens

// What a request asks for.
struct Request {
  int t0, fresh, len;  // first new token, new tokens, tokens with the new ones
  int row_blocks;      // 0: not this kernel's
  int first, tiles;    // key tiles that some row sees
};
template <int ROWS, bool LARGE>
__device__ __forceinline__ Request request_of(const Kv4AttnParams& p, int b) {
  Request r{};
  if (b >= p.B) return r;
  if (p.cu != nullptr) {
    r.t0 = p.cu[b];
    r.fresh = max(p.cu[b + 1] - r.t0, 0);
  } else {
    r.fresh = p.T / p.B;
    r.t0 = b * r.fresh;
  }
  r.len = max(p.lens[b], 0);
  const int64_t rows = (int64_t)r.fresh * p.G;
  r.row_blocks = (rows > p.row_limit) != LARGE ? 0 : (int)((rows + ROWS - 1) / ROWS);
  const int held = (int)min((int64_t)r.len, (int64_t)p.M << p.cache.bs_log2);
  const int lo = p.causal && p.window > 0 ? (int)max((int64_t)r.len - r.fresh - p.window + 1, (int64_t)0) : 0;
  r.first = lo / kTile;
  r.tiles = held > lo ? (held + kTile - 1) / kTile - r.first : 0;
  return r;
}

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m);
  return x;
}
__device__ __forceinline__ int64_t wave_prefix64(int64_t x, int lane) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  return x;
}

// Key tiles per chunk: the whole grid's tiles spread over about `target` workgroups, at least min_tiles each.
template <int ROWS, bool LARGE>
__device__ __forceinline__ int chunk_tiles(const Kv4AttnParams& p, int lane) {
  int64_t total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const Request r = request_of<ROWS, LARGE>(p, b0 + lane);
    total += (int64_t)r.row_blocks * r.tiles;
  }
  total = wave_sum64(total) * p.cache.Hkv;
  const int64_t each = (total + p.target - 1) / p.target;
  return (int)min(max(each, (int64_t)p.min_tiles), (int64_t)0x3fffffff);
}
__device__ __forceinline__ int chunks_of(const Request& r, int per) { return max((r.tiles + per - 1) / per, 1); }

struct Item {
  Request rq;
  int b;             // -1: there is no such item
  int rb, ch, nch;   // row block, chunk of nch
  int per;           // tiles a chunk
  int64_t items;     // of the whole call, where b < 0
};
template <int ROWS, bool LARGE>
__device__ __forceinline__ Item find_item(const Kv4AttnParams& p, int64_t item, int lane) {
  Item it{};
  it.b = -1;
  it.per = chunk_tiles<ROWS, LARGE>(p, lane);
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const Request r = request_of<ROWS, LARGE>(p, b0 + lane);
    const int64_t mine = (int64_t)r.row_blocks * chunks_of(r, it.per);
    const int64_t s = wave_prefix64(mine, lane);
    const int64_t before = it.items + s - mine;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item >= before && item < before + mine);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      it.b = __builtin_amdgcn_readfirstlane(b0 + src);
      it.rq = request_of<ROWS, LARGE>(p, it.b);
      it.nch = chunks_of(it.rq, it.per);
      const int i = (int)(item - __shfl(before, src));
      it.rb = __builtin_amdgcn_readfirstlane(i / it.nch);
      it.ch = __builtin_amdgcn_readfirstlane(i % it.nch);
      break;
    }
    it.items += __shfl(s, 63);
  }
  return it;
}

// 1 / l of a finished row. Without weight l is a mark, not a sum: the row is 0 / 0 where it saw keys.
__device__ __forceinline__ float row_inv(float m, float l) { return m == -INFINITY ? 1.0f / (0.f * l) : 1.0f / l; }

}  // namespace gfa
