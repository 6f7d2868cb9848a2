// Attention over the key/value cache in 4 bits for requests that share prefixes (gfa_kv4_share), gfx950.
//
// A group of requests whose tables begin with the same blocks is one request as far as those go: its rows, all of the group's
// new tokens and heads, see all of the prefix. So the prefix is read and decoded once per row block of the group instead of
// once per request, and many rows go to the matrix cores at once: 64 answers to a 16k prompt, 32:8 D = 128, are 256 rows a KV
// head, for which the chunk kernel's products replace 64 passes of the split kernel over the same codes. Behind the prefix
// every request is on its own. Softmax over both: sums with their maxima, joined as chunks of one row are.
//
// One launch computes the sums: the groups' prefixes by the chunk kernel's work (many rows) and the split kernel's (few), and the
// requests' rests by the split kernel's, as three runs of workgroups. A second launch joins a row's chunks of both. Whether that
// pays depends on the lengths: where it does not, the first launch takes the requests whole.
//
// Bound: issue of the chunk kernel's products and decoding (64 answers to a 16k prompt, 32:8 D = 128: 47.8 us against 215 without
// sharing; the tiles' loop 31, 1.1 us a tile and CU), around it latency: 2.5 us until a workgroup has its work, 8 until its first
// products, 2 (D = 128) to 7 us (D = 512) for sums out, 6 for the join. Eight answers to each of four prompts of 8k, 32:4 D = 512, 54 us
// (90), 16 of 4 drafted tokens, 3k, 8:4 D = 256, 25 (21, to which tables so narrow leave it).
#include <algorithm>

#include "gfa_kv4_chunk.h"
#include "gfa_kv4_split.h"
#include "gfa_launch.h"

namespace gfa {

namespace {

constexpr int kTpb = 256;
constexpr int kSpare = 64;  // workgroups for rows of no request

template <int D, bool IS_BF16, bool CAP>
__device__ __forceinline__ void many_rows(const Kv4AttnParams& p, const int lane, const int wave, const int head, const Item& it, char GFA_LDS* const K0,
                                          char GFA_LDS* const K1, char GFA_LDS* const V0, char GFA_LDS* const V1, char GFA_LDS* const S0,
                                          char GFA_LDS* const S1) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr Kv4Part PART = kPart;
  constexpr int ROWS = kSharedRows;
#include "gfa_kv4_chunk.inc"
#endif
}
template <int D, bool IS_BF16, bool CAP>
__device__ __forceinline__ void few_rows(const Kv4AttnParams& p, const int lane, const int wave, const int head, const Item& it, char GFA_LDS* const K0,
                                         char GFA_LDS* const K1, char GFA_LDS* const V0, char GFA_LDS* const V1) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr Kv4Part PART = kPart;
  __shared__ __attribute__((aligned(16))) f32x4 sums_lds[kWaves][D == 512 ? D / 32 * 64 : 1];  // (its own place: no lane registers to choose one of four)
  auto o_lds = [&](int w) __attribute__((always_inline)) {
    return D == 512 ? (f32x4 GFA_LDS*)sums_lds[w] : (f32x4 GFA_LDS*)(w == 0 ? K0 : w == 1 ? K1 : w == 2 ? V0 : V1);
  };
  // Past the caches below D = 512, also where up to four row blocks of a group read the same tiles: through the caches 44 calls with groups of 17 to
  // 64 rows took 1.0% (D = 64) to 1.7% (D = 256) longer, single row blocks 4.7%. At D = 512 either way within 0.5%.
  constexpr bool ONCE = D < 512;
#include "gfa_kv4_split.inc"
#endif
}

// The call's parameters as a group's prefix or a request's rest has them.
__device__ __forceinline__ Kv4AttnParams part_of(const Kv4SharedParams& s, const Kv4Sums& sums, bool group) {
  Kv4AttnParams p = s.p;
  if (group) p.causal = 0;
  p.slots = sums.slots;
  p.part = sums.part;
  p.part_ml = sums.part_ml;
  return p;
}

// ---- the split of the call ----
// As in gfa_kv4_sched.h, of three kinds of items in this order: row blocks of groups of many rows, of groups of few, of the
// requests behind their prefixes. A grid for any lengths would be several times the items there are, and one that finds nothing takes
// 2 to 4 us to find that out: three times kv4_shared_wgs for every CU are launched at most, and take the items in turn (308 requests without
// prefixes, 16:8 D = 256, 87 -> 74 us, 93 in three groups, 32:8 D = 128, 28 -> 24; as many as the CUs hold 10 to 20% slower where there
// is more to do, ten times the same as a grid for any lengths).
// Up to 64 requests every wave looks through all of them; more are dealt to the four waves, which trade what they found in LDS.
enum Which : int { kMany, kFew, kRests, kBlocks };
struct Both {
  Request own, group;  // of the request; of the group that begins with it (no rows: none does). own.tiles: of all its keys
  int behind;          // own tiles behind the prefix
  bool large;
};
template <int BIG>
__device__ __forceinline__ Both both_of(const Kv4SharedParams& s, int b) {
  const Kv4AttnParams& p = s.p;
  Both x{};
  const int bc = min(b, p.B - 1);
  const int c0 = p.cu[bc], c1 = p.cu[bc + 1], len = p.lens[bc], skip = p.skip[bc];
  const int g0 = s.group_cu[bc], g1 = s.group_cu[bc + 1], glen = s.group_lens[bc];
  if (b >= p.B) return x;
  const int most = p.M << p.cache.bs_log2;
  auto tokens = [&](int from, int to) { return min(max((int)((unsigned)to - (unsigned)from), 0), p.T); };
  auto blocks = [&](int rows, int log2) { return (int)(((unsigned)rows + (1u << log2) - 1) >> log2); };
  static_assert(kSplitRows == 16 && BIG == 128);
  x.own.t0 = c0;
  x.own.fresh = tokens(c0, c1);
  x.own.len = max(len, 0);
  x.own.skip = max(skip, 0);
  // tokens past q's have no rows; those of a request of many rows are the chunk kernel's
  x.own.row_blocks = x.own.fresh * p.G > p.row_limit ? 0 : blocks(min(x.own.fresh, max(p.T - max(c0, 0), 0)) * p.G, 4);
  const int held = min(x.own.len, most);
  x.own.tiles = (held + kTile - 1) / kTile;
  x.behind = held > x.own.skip ? x.own.tiles - x.own.skip / kTile : 0;
  x.group.t0 = g0;
  x.group.len = max(glen, 0);
  x.group.fresh = x.group.len > 0 ? tokens(g0, g1) : 0;
  x.large = x.group.fresh * p.G > s.row_limit;
  x.group.row_blocks = blocks(x.group.fresh * p.G, x.large ? 7 : 4);
  x.group.tiles = (min(x.group.len, most) + kTile - 1) / kTile;
  return x;
}

struct Plan {
  int first, end;  // this wave's requests
  bool alone;      // all of them
  bool apart;      // prefixes are taken apart
  bool fits;       // the host's arrays hold the requests' row blocks (not only for a cu that is no prefix sum)
  int per_many, per_few, per_rest;  // key tiles per chunk
};
// A group's rows and sums.
struct Group {
  int t0, rows, row_blocks, nch, slot;
  bool large;
};
struct PlanLds {
  float total[4][6];
  int count[4][4], found[16], group[4][8];
};

// Key tiles per chunk of each kind, see chunk_tiles, and whether prefixes are taken apart at all: where that leaves more than
// `worth` fewer passes of the split kernel over tiles (a KV head's; one of the chunk kernel counts as many_cost).
template <int BIG>
__device__ __forceinline__ Plan plan_of(const Kv4SharedParams& s, const Both& x0, int first, int end, bool alone, PlanLds& lds, int lane, int wave) {
#pragma clang fp contract(off)
  Plan out{};
  out.first = first;
  out.end = end;
  out.alone = alone;
  // the call's parameters all at once: a line of them on its own waits for memory
  asm volatile("" ::"s"(s.many_cost), "s"(s.worth), "s"(s.apart_cost), "s"(s.group_blocks), "s"(s.many.share), "s"(s.few.share), "s"(s.rest.share),
               "s"(s.many.min_tiles), "s"(s.few.min_tiles), "s"(s.rest.min_tiles));
  float t[6] = {};  // kMany, kFew, kRests, whole requests; their row blocks, the groups'
  Both x = x0;
  for (int b0 = first;;) {
    const float own = (float)x.own.row_blocks, group = (float)x.group.row_blocks * (float)x.group.tiles;
    t[kMany] += x.large ? group : 0.f;
    t[kFew] += x.large ? 0.f : group;
    t[kRests] += own * (float)x.behind;
    t[3] += own * (float)x.own.tiles;
    t[4] += own;
    t[5] += (float)x.group.row_blocks;
    if ((b0 += 64) >= end) break;
    x = both_of<BIG>(s, b0 + lane);
  }
#pragma unroll
  for (int k = 0; k < 6; ++k) t[k] = wave_sum(t[k]);
  if (!alone) {
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < 6; ++k) lds.total[wave][k] = t[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 6; ++k) t[k] = ((lds.total[0][k] + lds.total[1][k]) + lds.total[2][k]) + lds.total[3][k];
  }
  out.apart = __builtin_amdgcn_readfirstlane(t[3] - t[kRests] - t[kFew] - t[kMany] * s.many_cost - t[4] * s.apart_cost > s.worth) && t[5] <= s.group_blocks;
  out.fits = t[4] <= (float)s.p.row_blocks;
  auto per = [&](float total, int min_tiles, float share) {
    return __builtin_amdgcn_readfirstlane(max((int)fminf(ceilf(total * share), 1.0e9f), min_tiles));
  };
  out.per_many = per(t[kMany], s.many.min_tiles, s.many.share);
  out.per_few = per(t[kFew], s.few.min_tiles, s.few.share);
  out.per_rest = per(out.apart ? t[kRests] : t[3], s.rest.min_tiles, s.rest.share);
  return out;
}

// A request's items, and at kBlocks its own row blocks.
struct Counts {
  int n[4];
};
__device__ __forceinline__ Counts counts_of(const Both& x, const Plan& plan) {
  Counts c;
  const int group = plan.apart ? x.group.row_blocks * chunks_of(x.group, x.large ? plan.per_many : plan.per_few) : 0;
  Request rest = x.own;
  rest.tiles = plan.apart ? x.behind : x.own.tiles;
  c.n[kMany] = x.large ? group : 0;
  c.n[kFew] = x.large ? 0 : group;
  c.n[kRests] = rest.row_blocks * chunks_of(rest, plan.per_rest);
  c.n[kBlocks] = rest.row_blocks;
  return c;
}

// A wave's requests 64 at a time: their counts and the sums of the counts up to each.
template <int BIG>
struct Round {
  Both x;
  Counts c;
  int upto[4];
  __device__ __forceinline__ void take(const Both& of, const Plan& plan) {
    x = of;
    c = counts_of(x, plan);
#pragma unroll
    for (int k = 0; k < 4; ++k) upto[k] = wave_prefix_sum(c.n[k]);
  }
};
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

// What is ahead of this wave's requests, and the call's counts.
struct Ahead {
  int before[4], all[4];
};
template <int BIG>
__device__ __forceinline__ Ahead ahead_of(const Kv4SharedParams& s, const Plan& plan, Round<BIG>& r, PlanLds& lds, int lane, int wave) {
  Ahead out{};
  for (int b0 = plan.first;;) {
#pragma unroll
    for (int k = 0; k < 4; ++k) out.all[k] += last_lane(r.upto[k]);
    if ((b0 += 64) >= plan.end) break;
    r.take(both_of<BIG>(s, b0 + lane), plan);
  }
  if (plan.alone) return out;
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) lds.count[wave][k] = out.all[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    out.all[k] = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = __builtin_amdgcn_readfirstlane(lds.count[w][k]);
      out.before[k] += w < wave ? n : 0;
      out.all[k] += n;
    }
  }
  if (plan.end - plan.first > 64) r.take(both_of<BIG>(s, plan.first + lane), plan);
  return out;
}

__device__ __forceinline__ void wave_range(int B, int wave, int& first, int& end, bool& alone) {
  alone = B <= 64;
  const int each = alone ? 64 : (B + 255) / 256 * 64;
  first = alone ? 0 : wave * each;
  end = first + each;
}

}  // namespace

template <int D, bool IS_BF16, bool CAP>
__global__ __launch_bounds__(kTpb, kv4_shared_wgs(D)) void kv4_shared_kernel(const Kv4SharedParams) {
  constexpr int BIG = kSharedRows;
  __shared__ PlanLds lds;
  // The chunk kernel's tiles, or what the waves of the split kernel join: D * 32 bytes each (D = 64: 4 KB).
  constexpr int TILE = std::max(kv4_chunk_steps(kPart, D) * Kv4Layout<D>::TILE_CODES, D == 64 ? 4096 : D * 32), SCALES = kv4_chunk_steps(kPart, D) * 1024;
  __shared__ __attribute__((aligned(1024))) char k_lds0[TILE], k_lds1[TILE], v_lds0[TILE], v_lds1[TILE], s_lds0[SCALES], s_lds1[SCALES];
  char GFA_LDS* const K0 = (char GFA_LDS*)k_lds0;
  char GFA_LDS* const K1 = (char GFA_LDS*)k_lds1;
  char GFA_LDS* const V0 = (char GFA_LDS*)v_lds0;
  char GFA_LDS* const V1 = (char GFA_LDS*)v_lds1;
  char GFA_LDS* const S0 = (char GFA_LDS*)s_lds0;
  char GFA_LDS* const S1 = (char GFA_LDS*)s_lds1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  typedef const Kv4SharedParams __attribute__((address_space(4)))* Args;
  for (int at = (int)blockIdx.x;;) {
    // read anew each turn: held through the loop they spill
    Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    const Kv4SharedParams& s = *(const Kv4SharedParams*)args;
    const int lane = fresh_lane();
    const int head = s.p.hkv.rem(at);
    int item = s.p.hkv.quot(at);
    int first, end;
    bool alone;
    wave_range(s.p.B, wave, first, end, alone);
    const Both x0 = both_of<BIG>(s, first + lane);
    const Plan plan = plan_of<BIG>(s, x0, first, end, alone, lds, lane, wave);
    if (!plan.fits) {
      if (at == 0 && wave == 0 && lane == 0) *s.joined = 0;
      return;
    }
    Round<BIG> r;
    r.take(x0, plan);
    if (wave == 0 && lane == 0) lds.found[0] = -1;
    const Ahead a = ahead_of<BIG>(s, plan, r, lds, lane, wave);
    const int taken = (a.all[kMany] + a.all[kFew] + a.all[kRests]) * s.p.cache.Hkv;
    if (at == 0 && wave == 0 && lane == 0) *s.joined = a.all[kBlocks];
    const int which = item < a.all[kMany] ? kMany : item < a.all[kMany] + a.all[kFew] ? kFew : kRests;
    item -= which == kMany ? 0 : which == kFew ? a.all[kMany] : a.all[kMany] + a.all[kFew];
    if (which == kRests && item >= a.all[kRests]) {
      if (at < taken + kSpare) zero_rows<D>(s.p, wave * 64 + lane, at - taken, kSpare);
      return;
    }
    Item it{};
    it.b = -1;
    Group grp{};
    int block = 0, before[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) before[k] = a.before[k];
    for (int b0 = plan.first;;) {
      const int n = which == kMany ? r.c.n[kMany] : which == kFew ? r.c.n[kFew] : r.c.n[kRests];
      const int upto = which == kMany ? r.upto[kMany] : which == kFew ? r.upto[kFew] : r.upto[kRests];
      const int from = (which == kMany ? before[kMany] : which == kFew ? before[kFew] : before[kRests]) + upto - n;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(item >= from && item < from + n);
      const int src = hit != 0 ? __builtin_ctzll(hit) : 63;
      if (which == kRests && plan.apart) {
        // the last group that begins with the request or ahead of it
        const uint64_t groups = __builtin_amdgcn_ballot_w64(r.x.group.row_blocks > 0 && lane <= src);
        if (groups != 0) {
          const int g = 63 - __builtin_clzll(groups);
          auto at = [&](int x) { return __builtin_amdgcn_readlane(x, g); };
          const bool large = at(r.x.large) != 0;
          const int row_blocks = at(r.x.group.row_blocks), items = at(large ? r.c.n[kMany] : r.c.n[kFew]);
          const int slot = (large ? before[kMany] : before[kFew]) + at(large ? r.upto[kMany] : r.upto[kFew]) - items;
          grp = Group{at(r.x.group.t0), at(r.x.group.fresh) * s.p.G, row_blocks, __builtin_amdgcn_readfirstlane(quotient(items, row_blocks)), slot, large};
        }
      }
      if (hit != 0) {
        it.b = b0 + src;
        it.rq = request_from(which == kRests ? r.x.own : r.x.group, src);
        if (which == kRests) {
          it.rq.tiles = plan.apart ? __builtin_amdgcn_readlane(r.x.behind, src) : it.rq.tiles;
          it.rq.skip = plan.apart ? it.rq.skip : 0;
        }
        it.nch = __builtin_amdgcn_readfirstlane(quotient(__builtin_amdgcn_readlane(n, src), it.rq.row_blocks));
        const int i = item - __builtin_amdgcn_readlane(from, src);
        it.rb = __builtin_amdgcn_readfirstlane(quotient(i, it.nch));
        it.ch = i - it.rb * it.nch;
        it.slot = which == kRests && it.nch == 1 && it.rq.skip == 0 ? -1 : item;
        block = before[kBlocks] + __builtin_amdgcn_readlane(r.upto[kBlocks], src) - it.rq.row_blocks + it.rb;
        break;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) before[k] += last_lane(r.upto[k]);
      if ((b0 += 64) >= plan.end) break;
      r.take(both_of<BIG>(s, b0 + lane), plan);
    }
    if (!alone) {
      if (lane == 0) {
        const int group[] = {grp.t0, grp.rows, grp.row_blocks, grp.nch, grp.slot, grp.large};
#pragma unroll
        for (int k = 0; k < 6; ++k) lds.group[wave][k] = group[k];
        if (it.b >= 0) {
          const int of[] = {it.b, it.rb, it.ch, it.nch, it.slot, it.rq.t0, it.rq.fresh, it.rq.len, it.rq.row_blocks, it.rq.tiles, it.rq.skip, block, wave};
#pragma unroll
          for (int k = 0; k < 13; ++k) lds.found[k] = of[k];
        }
      }
      __syncthreads();
      auto at = [&](int k) { return __builtin_amdgcn_readfirstlane(lds.found[k]); };
      it = Item{Request{at(5), at(6), at(7), at(8), at(9), at(10)}, at(0), at(1), at(2), at(3), 0, at(4)};
      if (it.b < 0) return;
      block = at(11);
      int w = at(12);  // the group: of that wave's requests, or of one ahead of it
      while (w > 0 && __builtin_amdgcn_readfirstlane(lds.group[w][2]) == 0) --w;
      auto of = [&](int k) { return __builtin_amdgcn_readfirstlane(lds.group[w][k]); };
      grp = Group{of(0), of(1), of(2), of(3), of(4), of(5) != 0};
    }
    if (it.b < 0) return;
    // for the join
    if (which == kRests && head == 0 && it.ch == 0 && (unsigned)block < (unsigned)s.p.row_blocks && wave == 0 && lane == 0) {
      const Kv4Sums& sums = grp.large ? s.many : s.few;
      const bool there = it.rq.skip > 0 && (int64_t)grp.slot + (int64_t)grp.row_blocks * grp.nch <= sums.slots;
      s.joins[block] = Kv4Join{it.slot, it.nch, it.rb, it.rq.t0, it.rq.fresh, there ? grp.nch : 0, grp.slot, grp.row_blocks, grp.t0, grp.rows, grp.large, 0};
    }
    if (which == kMany) {
      many_rows<D, IS_BF16, CAP>(part_of(s, s.many, true), lane, wave, head, it, K0, K1, V0, V1, S0, S1);
    } else {
      few_rows<D, IS_BF16, CAP>(part_of(s, which == kFew ? s.few : s.rest, which == kFew), lane, wave, head, it, K0, K1, V0, V1);
    }
    if ((at += s.grid) >= taken + kSpare) return;
    __syncthreads();
  }
}

// As kv4_join_kernel, of a row's chunks behind the prefix and of its row's in the group's sums; where they are the first kernel has
// written down. Bound: latency, of a row block's place and of one pass of loads.
template <int D, bool IS_BF16>
__global__ __launch_bounds__(kTpb) void kv4_shared_join_kernel(const Kv4SharedParams s) {
  constexpr int ROWS = kSplitRows, BIG = kSharedRows;
  const Kv4AttnParams p = part_of(s, s.rest, false);
  const int LPR = p.join_slice / 4;  // a power of two
  const int GR = kTpb / LPR;
  __shared__ f32x4 o_lds[kTpb];
  __shared__ float ml_lds[kTpb / 16][2];
  int id = (int)blockIdx.x;
  const int head = p.hkv.rem(id);
  id = p.hkv.quot(id);
  const int slice = id % (D / p.join_slice);
  id /= D / p.join_slice;
  const int block = __builtin_amdgcn_readfirstlane(id / p.join_rows);
  const int blocks = *s.joined;
  const Kv4Join j = s.joins[block];
  if (block >= blocks || j.slot < 0) return;  // none; out already
  if ((int64_t)j.slot + j.nch > p.slots) return;  // cu that is no prefix sum: no such chunks
  const float* const gp = j.large ? s.many.part : s.few.part;
  const float* const gml = j.large ? s.many.part_ml : s.few.part_ml;
  const int rb = j.rb;
  const int rows = min(ROWS, j.fresh * p.G - rb * ROWS);
  const int all = j.nch + j.group_nch;
  const int parts = min(p.join_parts, all > 1 ? 1 << (32 - __builtin_clz(all - 1)) : 1);
  const int at_once = GR / parts;
  const int group = threadIdx.x / LPR, part = group % parts, d = slice * p.join_slice + threadIdx.x % LPR * 4;
  for (int r0 = id % p.join_rows * at_once; r0 < rows; r0 += p.join_rows * at_once) {
    const int rr = r0 + group / parts;
    const int row = rb * ROWS + rr;
    const int t = j.t0 + p.g.quot(row), hg = p.g.rem(row), qh = head * p.G + hg;
    const bool live = rr < rows && t >= 0 && t < p.T;
    float m = -INFINITY, l = 0.f;  // without a maximum l counts the rows' marks, see row_inv
    f32x4 o{};
    if (live) {
      // the row in its group: row block, and row of it
      const int row_g = (t - j.group_t0) * p.G + hg, in = j.large ? row_g % BIG : row_g % ROWS;
      const int blk_g = j.large ? j.group_blocks - 1 - row_g / BIG : row_g / ROWS;  // the chunk kernel takes the last rows first
      const int64_t item0 = (int64_t)j.group_slot + (int64_t)blk_g * j.group_nch;
      const int count = row_g >= 0 && row_g < j.group_rows ? all : j.nch;
      // one address or the other, then the load: behind a branch the loads would wait for each other
#pragma unroll 8
      for (int c = part; c < count; c += parts) {
        const int cg = c - j.nch;
        const int64_t own = (((int64_t)j.slot + c) * p.cache.Hkv + head) * ROWS + rr;
        const int64_t its = ((item0 + cg) * p.cache.Hkv + head) * (j.large ? BIG : ROWS) + in;
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
  const dim3 grid((unsigned)s.grid);
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
