// Pages of the key/value cache in 4 bits that requests share: forked and given back, compacted, copied; and what
// neighbouring requests have in common. gfx950.
//
// Sets of blocks are bit maps in LDS, built by every workgroup for itself from the block tables; ranks and k-th members come
// from prefix counts over 256-block groups, so every list is in ascending order whatever the order of the atomics (all of
// them OR, MIN and MAX of integers). One launch decides, a second one moves the bytes.
#include <algorithm>

#include "gfa_kv4.h"
#include "gfa_launch.h"

namespace gfa {

namespace {

constexpr int kTpb = 1024, kWaves = kTpb / 64;
constexpr int kGroup = 8;  // words of a counted group

// Inclusive prefix over the workgroup's threads of two counts; two barriers.
struct Two {
  int a, b;
};
__device__ __forceinline__ Two block_prefix(Two x, Two* sums, Two& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Two s{wave_prefix_sum(x.a), wave_prefix_sum(x.b)};
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  total = Two{0, 0};
  Two before{0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Two y = sums[w];
    if (w < wave) {
      before.a += y.a;
      before.b += y.b;
    }
    total.a += y.a;
    total.b += y.b;
  }
  __syncthreads();
  return Two{s.a + before.a, s.b + before.b};
}

// Place of the k-th set bit of w (k below its count).
__device__ __forceinline__ int kth_bit(unsigned w, int k) {
  int at = 0;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const int c = __builtin_popcount(w & ((1u << s) - 1));
    if (k >= c) {
      k -= c;
      w >>= s;
      at += s;
    }
  }
  return at;
}

// Members of a set ahead of id, and its k-th member. `word(i)` are the set's 32-block words, before[g] its members ahead
// of group g.
template <typename Word>
__device__ __forceinline__ int rank_of(int id, const int* before, const Word& word) {
  const int w = id >> 5;
  int n = before[w / kGroup];
  for (int i = w / kGroup * kGroup; i < w; ++i) n += __builtin_popcount(word(i));
  return n + __builtin_popcount(word(w) & ((1u << (id & 31)) - 1));
}
template <typename Before, typename Word>
__device__ __forceinline__ int kth_member(int k, int groups, const Before& before, const Word& word) {
  int lo = 0, hi = groups - 1;  // the last group with at most k members ahead of it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (before(mid) <= k) lo = mid; else hi = mid - 1;
  }
  k -= before(lo);
  int w = lo * kGroup;
  for (int i = 0; i + 1 < kGroup; ++i) {
    const int c = __builtin_popcount(word(w));
    if (k < c) break;
    k -= c;
    ++w;
  }
  return w * 32 + kth_bit(word(w), k);
}

__device__ __forceinline__ bool bit_of(const unsigned* set, int id) { return set[id >> 5] >> (id & 31) & 1; }
__device__ __forceinline__ void mark(unsigned* set, int id) { atomicOr(&set[id >> 5], 1u << (id & 31)); }

__device__ __forceinline__ int columns_of(int tokens, int bs_log2, int M) {
  return (int)min(((int64_t)max(tokens, 0) + (1 << bs_log2) - 1) >> bs_log2, (int64_t)M);
}

// Calls visit(row, column, entry) for every entry that the old requests hold, kTpb requests at a time: the entries in
// use are counted through, so that a wide table with short requests costs what they hold. Eight entries of a
// thread are in flight at once. `ends`: kTpb ints of LDS.
template <typename Visit>
__device__ __forceinline__ void each_entry(const Kv4PagesParams& p, int* ends, Two* sums, const Visit& visit) {
  constexpr int U = 8;
  for (int b0 = 0; b0 < p.B; b0 += kTpb) {
    const int b = b0 + (int)threadIdx.x;
    const int cols = b < p.B ? columns_of(p.lens[b], p.bs_log2, p.M) : 0;
    Two total;
    ends[threadIdx.x] = block_prefix(Two{cols, 0}, sums, total).a;  // tables of up to 2^30 entries
    __syncthreads();
    const int rows = min(kTpb, p.B - b0);
    for (int i0 = 0; i0 < total.a; i0 += U * kTpb) {
      int row[U], col[U], entry[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kTpb + (int)threadIdx.x;
        row[u] = -1;
        entry[u] = -1;
        if (i < total.a) {
          int lo = 0, hi = rows - 1;  // the first row that ends behind i
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (ends[mid] > i) hi = mid; else lo = mid + 1;
          }
          row[u] = b0 + lo;
          col[u] = i - (lo > 0 ? ends[lo - 1] : 0);
          entry[u] = p.table[(int64_t)row[u] * p.table_stride + col[u]];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row[u] >= 0 && (unsigned)entry[u] < (unsigned)p.num_blocks) visit(row[u], col[u], entry[u]);
    }
    __syncthreads();
  }
}

// A new row: its parent (-1: none) and the tokens it keeps.
struct NewRow {
  int parent, tokens;
};
__device__ __forceinline__ NewRow new_row(const Kv4PagesParams& p, int r) {
  const int b = p.parents != nullptr ? p.parents[r] : r;
  if ((unsigned)b >= (unsigned)p.B) return NewRow{-1, 0};
  const int n = max(p.lens[b], 0);
  return NewRow{b, p.keep != nullptr ? min(n, max(p.keep[r], 0)) : n};
}

}  // namespace

// Block tables of the next step's requests. A block that new rows hold in part (n % block_size tokens) goes on in the first
// of them, if no row holds it whole; the others get copies, in the order of the rows, from the blocks given back and
// then from the free list. Bound: latency of dependent loads and LDS steps (8 rows 7.0 us, 24 prompts of 170 blocks forked into 192
// rows 9.7).
__global__ __launch_bounds__(kTpb) void kv4_fork_kernel(const Kv4PagesParams p) {
  extern __shared__ unsigned lds[];
  __shared__ Two sums[kWaves];
  __shared__ int ends[kTpb];
  const int tid = threadIdx.x, W = p.words, groups = W / kGroup;
  unsigned *old = lds, *whole = lds + W, *part = lds + 2 * W;
  int* freed_before = reinterpret_cast<int*>(lds + 3 * W);  // members of old less the new rows' ahead of a group
  int* part_before = freed_before + groups;
  int* most = part_before + groups;  // (B): whole blocks of a parent's that some new row keeps
  int* first = most + p.B;           // (rows): the first row that holds the partial block of a rank
  int* last = first + p.rows;        // (rows): a row's last block, if it is partial
  for (int i = tid; i < 3 * W; i += kTpb) lds[i] = 0;
  for (int i = tid; i < p.B; i += kTpb) most[i] = 0;
  __syncthreads();

  // ---- what the new rows ask for ----
  for (int r = tid; r < p.rows; r += kTpb) {
    const NewRow n = new_row(p, r);
    first[r] = 0x7fffffff;
    int x = -1;
    if (n.parent >= 0) {
      const int full = n.tokens >> p.bs_log2;
      atomicMax(&most[n.parent], full);
      if ((n.tokens & ((1 << p.bs_log2) - 1)) != 0 && full < p.M) {
        x = p.table[(int64_t)n.parent * p.table_stride + full];
        x = (unsigned)x < (unsigned)p.num_blocks ? x : -1;
      }
    }
    last[r] = x;
    if (x >= 0) mark(part, x);
  }
  __syncthreads();
  each_entry(p, ends, sums, [&](int row, int col, int id) {
    mark(old, id);
    if (col < most[row]) mark(whole, id);
  });

  // ---- counts ----
  const auto freed = [&](int w) { return old[w] & ~(whole[w] | part[w]); };
  const auto partial = [&](int w) { return part[w]; };
  Two total;
  {
    Two n{0, 0};
    if (tid < groups) {
      for (int i = 0; i < kGroup; ++i) {
        n.a += __builtin_popcount(freed(tid * kGroup + i));
        n.b += __builtin_popcount(part[tid * kGroup + i]);
      }
    }
    const Two s = block_prefix(n, sums, total);
    if (tid < groups) {
      freed_before[tid] = s.a - n.a;
      part_before[tid] = s.b - n.b;
    }
  }
  const int used = min(max(p.used[0], 0), p.F);
  const int given = min(total.a, used);
  __syncthreads();

  // ---- copies ----
  for (int r = tid; r < p.rows; r += kTpb)
    if (last[r] >= 0) atomicMin(&first[rank_of(last[r], part_before, partial)], r);
  __syncthreads();
  int copies = 0;
  for (int r0 = 0; r0 < p.rows; r0 += kTpb) {
    const int r = r0 + tid, x = r < p.rows ? last[r] : -1;
    const bool copy = x >= 0 && (bit_of(whole, x) || first[rank_of(x, part_before, partial)] != r);
    Two now;
    const int k = copies + block_prefix(Two{copy, 0}, sums, now).a - 1;
    if (copy) {
      int to = -1;
      if (k < given) {
        to = kth_member(k, groups, [&](int g) { return freed_before[g]; }, freed);
      } else if (used + (k - given) < p.F) {
        to = p.free_ids[used + (k - given)];
      }
      to = (unsigned)to < (unsigned)p.num_blocks ? to : -1;
      last[r] = to;
      if (blockIdx.x == 0) {
        p.src[k] = x;
        p.dst[k] = to;
      }
    }
    copies += now.a;
  }
  __syncthreads();

  // ---- results, the workgroups in turn ----
  const int at = (int)blockIdx.x * kTpb + tid, all = (int)gridDim.x * kTpb;
  // entries below `used` are only written, those from there on only read
  for (int k = at; k < given; k += all)
    p.free_ids[used - given + k] = kth_member(k, groups, [&](int g) { return freed_before[g]; }, freed);
  if (at == 0) {
    p.used_out[0] = (int)min((int64_t)used - given + copies, (int64_t)0x7fffffff);
    p.count[0] = copies;
  }
  for (int r = at; r < p.rows; r += all) p.lens_out[r] = new_row(p, r).tokens;
  const int64_t entries = (int64_t)p.rows * p.M;
  for (int64_t i = at; i < entries; i += all) {
    const int r = p.m.quot((int)i), c = p.m.rem((int)i);
    const NewRow n = new_row(p, r);
    int x = -1;
    if (c < columns_of(n.tokens, p.bs_log2, p.M)) {
      if (c == n.tokens >> p.bs_log2) {  // the column that is not full
        x = last[r];
      } else {
        x = p.table[(int64_t)n.parent * p.table_stride + c];
        x = (unsigned)x < (unsigned)p.num_blocks ? x : -1;
      }
    }
    p.table_out[i] = x;
  }
}

// The pool's live blocks moved to its lowest ids: of n live ones, the k-th that is at or past n goes to the k-th hole below n. Bound:
// as the fork's (small tables 5.2 us, a pool of thousands of blocks 11.4).
__global__ __launch_bounds__(kTpb) void kv4_compact_kernel(const Kv4PagesParams p) {
  extern __shared__ unsigned lds[];
  __shared__ Two sums[kWaves];
  __shared__ int ends[kTpb];
  const int tid = threadIdx.x, W = p.words, groups = W / kGroup;
  unsigned* live = lds;
  int* before = reinterpret_cast<int*>(lds + W);
  for (int i = tid; i < W; i += kTpb) live[i] = 0;
  __syncthreads();
  each_entry(p, ends, sums, [&](int, int, int id) { mark(live, id); });
  Two total;
  {
    int n = 0;
    if (tid < groups) {
      for (int i = 0; i < kGroup; ++i) n += __builtin_popcount(live[tid * kGroup + i]);
    }
    const Two s = block_prefix(Two{n, 0}, sums, total);
    if (tid < groups) before[tid] = s.a - n;
  }
  __syncthreads();
  const auto in = [&](int w) { return live[w]; };
  const auto out = [&](int w) { return ~live[w]; };
  const auto in_before = [&](int g) { return before[g]; };
  const auto out_before = [&](int g) { return g * (32 * kGroup) - before[g]; };
  const int n = total.a;
  const int low = n < p.num_blocks ? rank_of(n, before, in) : n;  // live blocks that stay
  const int at = (int)blockIdx.x * kTpb + tid, all = (int)gridDim.x * kTpb;
  for (int k = at; k < n - low; k += all) {
    p.src[k] = kth_member(low + k, groups, in_before, in);
    p.dst[k] = kth_member(k, groups, out_before, out);
  }
  if (at == 0) {
    p.used_out[0] = n;
    p.count[0] = n - low;
  }
  for (int i = at; i < p.num_blocks; i += all) p.free_ids[i] = i;
  const int64_t entries = (int64_t)p.B * p.M;
  for (int64_t i = at; i < entries; i += all) {
    const int b = p.m.quot((int)i), c = p.m.rem((int)i);
    int x = -1;
    if (c < columns_of(p.lens[b], p.bs_log2, p.M)) {
      x = p.table[(int64_t)b * p.table_stride + c];
      x = (unsigned)x < (unsigned)p.num_blocks ? x : -1;
      if (x >= n) x = kth_member(rank_of(x, before, in) - low, groups, out_before, out);
    }
    p.table_out[i] = x;
  }
}

// Whole blocks of every layer, bytes as they are: a piece of 16 KB of one layer's codes or scales a turn, the workgroups
// counting through (pair, piece). Stores go past the caches, where blocks are read again from other addresses; loads do not: a
// fork's copies are often of one block (24 prompts' last blocks seven times each, 8 layers: 20 us, with loads past the
// caches too 25-30). Bound: memory. 1140 blocks of 4 layers, 317 MB each way, 105-113 us, 5.6-6.0 TB/s (stores through the caches 128).
constexpr int kCopyTpb = 256, kCopyUnroll = 4;
static_assert(kCopyTpb * kCopyUnroll * 16 == kKv4CopyPiece, "a workgroup's turn is one piece");
__global__ __launch_bounds__(kCopyTpb) void kv4_copy_kernel(const Kv4CopyParams p) {
  const int pairs = p.count != nullptr ? min(max(p.count[0], 0), p.pairs) : p.pairs;
  const int64_t units = (int64_t)pairs * p.pieces.d;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int pair = p.pieces.quot((int)u), piece = p.pieces.rem((int)u);
    const int from = p.src[pair], to = p.dst[pair];
    if ((unsigned)from >= (unsigned)p.num_blocks || (unsigned)to >= (unsigned)p.num_blocks) continue;
    int a = 0;  // the array that the piece is of
    while (a + 1 < p.arrays && piece >= p.first[a + 1]) ++a;
    const int64_t size = p.bytes[a];
    const int64_t off = (int64_t)(piece - p.first[a]) * kKv4CopyPiece + threadIdx.x * 16;
    const uint8_t* s = p.base[a] + from * size;
    uint8_t* d = p.base[a] + to * size;
    typedef unsigned vec __attribute__((ext_vector_type(4)));
    vec x[kCopyUnroll];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)  // past the end the last 16 bytes again, for nothing
      x[i] = *reinterpret_cast<const vec*>(s + min(off + i * (kCopyTpb * 16), size - 16));
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
      if (off + i * (kCopyTpb * 16) < size) __builtin_nontemporal_store(x[i], reinterpret_cast<vec*>(d + off + i * (kCopyTpb * 16)));
  }
}

// What neighbouring requests have in common: their first blocks, as far as both hold them ahead of the step's new tokens.
// Neighbours with at least `least` tokens in common are a group; its prefix is what all of them have. One workgroup, 16
// lanes a pair of rows. Bound: latency (8 requests 4.2 us, 256 7.4).
__global__ __launch_bounds__(kTpb) void kv4_share_kernel(const Kv4ShareParams p) {
  __shared__ Two sums[kWaves];
  __shared__ int common[kKv4ShareMost], prefix[kKv4ShareMost], end[kKv4ShareMost];
  const int tid = threadIdx.x;
  // ---- whole blocks ahead of the new tokens ----
  for (int b = tid; b < p.R; b += kTpb) {
    const int64_t fresh = max((int64_t)p.cu[b + 1] - p.cu[b], (int64_t)0);
    end[b] = (int)min(max(((int64_t)p.lens[b] - fresh), (int64_t)0) >> p.bs_log2, (int64_t)p.M);
    prefix[b] = 0x7fffffff;
  }
  __syncthreads();
  // ---- blocks that a row and the one before it begin with ----
  constexpr int LPP = 16, U = 8;  // lanes of a pair, entries of a lane at once
  const int sub = tid % LPP;
  for (int b = tid / LPP; b < p.R; b += kTpb / LPP) {
    const int* y = p.table + (int64_t)b * p.table_stride;
    const int* x = y - p.table_stride;
    const int n = b > 0 ? min(end[b - 1], end[b]) : 0;
    int same = n;
    for (int c0 = 0; c0 < n && same == n; c0 += LPP * U) {
      int l[U], r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = min(c0 + u * LPP + sub, n - 1);
        l[u] = x[c];
        r[u] = y[c];
      }
#pragma unroll
      for (int u = U - 1; u >= 0; --u)
        if (l[u] != r[u]) same = min(same, c0 + u * LPP + sub);
#pragma unroll
      for (int m = 1; m < LPP; m <<= 1) same = min(same, __shfl_xor(same, m));
    }
    if (sub == 0) common[b] = min(same, n) << p.bs_log2;
  }
  __syncthreads();
  for (int b = tid; b < p.R; b += kTpb) end[b] = 0;
  __syncthreads();
  // ---- groups ----
  int seen = 0;
  for (int b0 = 0; b0 < p.R; b0 += kTpb) {
    const int b = b0 + tid;
    const bool first = b < p.R && (b == 0 || common[b] < p.least);
    Two now;
    const int g = seen + block_prefix(Two{first, 0}, sums, now).a - 1;
    if (b < p.R) {
      if (!first) atomicMin(&prefix[g], common[b]);
      atomicMax(&end[g], b + 1);
    }
    seen += now.a;
  }
  __syncthreads();
  seen = 0;
  for (int b0 = 0; b0 < p.R; b0 += kTpb) {
    const int b = b0 + tid;
    const bool first = b < p.R && (b == 0 || common[b] < p.least);
    Two now;
    const int g = seen + block_prefix(Two{first, 0}, sums, now).a - 1;
    if (b < p.R) {
      const int n = prefix[g] == 0x7fffffff ? 0 : prefix[g];
      p.skip[b] = n;
      p.lens_out[b] = first ? n : 0;
      p.cu_out[b] = p.cu[first ? b : end[g]];
    }
    seen += now.a;
  }
  if (tid == 0) p.cu_out[p.R] = p.cu[p.R];
}

namespace {
template <typename Kernel>
hipError_t launch_pages(Kernel kernel, const Kv4PagesParams& p, int64_t work, size_t lds, hipStream_t stream) {
  // A workgroup for every 2048 results, each marking the tables for itself.
  const unsigned wgs = (unsigned)std::min<int64_t>(32, (work + 2047) / 2048);
  if (lds > 65536) {
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (err != hipSuccess) return err;
  }
  hipLaunchKernelGGL(kernel, dim3(wgs), dim3(kTpb), lds, stream, p);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_kv4_fork(const Kv4PagesParams& p, hipStream_t stream) {
  return launch_pages(kv4_fork_kernel, p, (int64_t)p.rows * p.M, 4 * kv4_fork_lds_words(p.words, p.B, p.rows), stream);
}
hipError_t launch_kv4_compact(const Kv4PagesParams& p, hipStream_t stream) {
  return launch_pages(kv4_compact_kernel, p, (int64_t)p.B * p.M + p.num_blocks, 4 * (size_t)(p.words + p.words / kGroup), stream);
}
hipError_t launch_kv4_copy(const Kv4CopyParams& p, hipStream_t stream) {
  const int64_t units = (int64_t)p.pairs * p.pieces.d;
  const unsigned wgs = (unsigned)std::min<int64_t>(units, 4096);  // twice what the CUs hold
  if (wgs == 0) return hipSuccess;
  hipLaunchKernelGGL(kv4_copy_kernel, dim3(wgs), dim3(kCopyTpb), 0, stream, p);
  return hipGetLastError();
}
hipError_t launch_kv4_share(const Kv4ShareParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(kv4_share_kernel, dim3(1), dim3(kTpb), 0, stream, p);
  return hipGetLastError();
}

}  // namespace gfa
