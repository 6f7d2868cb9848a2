// Drafted tokens verified by the target's probabilities, and the token that follows the accepted ones, gfx950.
//
// Token t of a request was drawn from the draft's probabilities q_t, the target's after token t - 1 are p_{t-1}. With a
// uniform u_t it is accepted while u_t q_t(x) < p_{t-1}(x); the first one that is not is replaced by a draw from
// max(p - q, 0), behind the last accepted one a draw from p follows. The tokens then have the target's distribution
// whatever the draft's was. Both sides of the comparison are exact in 64 bits (products of two 24-bit numbers).
//
// A draw: the first entry whose running sum of weights passes r times their sum, in 64 bits, sums in a fixed order: segments
// of a wave each, then the segment's entries. Only two rows of the vocabulary are read per request, whatever was
// drafted: the first kernel finds the row (every wave for itself, one probability a lane) and sums its segments, the
// second picks the segment and the entry.
// Bound: memory for large batches (64 requests, 262144 entries in 32 bits, a drafted token not accepted in 40 of them, so 104 rows: 109 MB in
// 21.8 us, 5.0 TB/s, then 5.8 to pick), latency of dependent loads for small ones (8 requests, 32000 entries: 4.4 and 5.4 us).
#include "gfa_common.h"
#include "gfa_launch.h"
#include "gfa_verify.h"

namespace gfa {

namespace {

constexpr int kTpb = 256, kWaves = kTpb / 64, kLane = 8;  // entries of a lane at once
static_assert(64 * kLane == kVerifyStep, "a wave's step");

enum class Kind { f16, bf16, f32 };

template <Kind K>
__device__ __forceinline__ float value(const void* p, int64_t i) {
  if constexpr (K == Kind::f32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t x = reinterpret_cast<const uint16_t*>(p)[i];
  return from16<K == Kind::bf16>((short)x);
}
// A probability: what is no positive number counts as none.
__device__ __forceinline__ double weight(float x) { return x > 0.f && x < INFINITY ? (double)x : 0.0; }

// Entries i .. i + 7 of a row; those from `end` on are 0. Rows start anywhere, so the loads are of the type's alignment.
template <Kind K>
__device__ __forceinline__ void load8(const void* row, int64_t at, int i, int end, float (&x)[kLane]) {
  if (i + kLane <= end) {
    if constexpr (K == Kind::f32) {
      __builtin_memcpy(x, reinterpret_cast<const float*>(row) + at + i, sizeof(x));
    } else {
      uint16_t h[kLane];
      __builtin_memcpy(h, reinterpret_cast<const uint16_t*>(row) + at + i, sizeof(h));
#pragma unroll
      for (int e = 0; e < kLane; ++e) x[e] = from16<K == Kind::bf16>((short)h[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e) x[e] = i + e < end ? value<K>(row, at + i + e) : 0.f;
  }
}

// A request's tokens: the first, how many.
struct Tokens {
  int t0, n;
};
__device__ __forceinline__ Tokens tokens_of(const VerifyParams& p, int b) {
  if (p.cu == nullptr) return Tokens{b * p.each, p.each};
  const int64_t t0 = min(max((int64_t)p.cu[b], (int64_t)0), (int64_t)p.T);
  const int64_t t1 = min(max((int64_t)p.cu[b + 1], t0), (int64_t)p.T);
  return Tokens{(int)t0, (int)(t1 - t0)};
}

// Drafted tokens that are accepted; the same in every lane.
template <Kind K>
__device__ __forceinline__ int accepted_of(const VerifyParams& p, const Tokens& r, int lane) {
  for (int i0 = 0; i0 + 1 < r.n; i0 += 64) {
    const int i = i0 + lane;
    bool fails = false;
    if (i + 1 < r.n) {
      const int64_t t = r.t0 + i;
      const int64_t x = p.tokens[t + 1];
      fails = true;
      if (x >= 0 && x < p.V) {
        const double q = p.draft != nullptr ? weight(value<K>(p.draft, (t + 1) * p.ds + x)) : 1.0;
        fails = !((double)p.accept[t + 1] * q < weight(value<K>(p.target, t * p.ts + x)));
      }
    }
    const uint64_t any = __builtin_amdgcn_ballot_w64(fails);
    if (any != 0) return i0 + __builtin_ctzll(any);
  }
  return r.n - 1;
}

// The weights that the next token is drawn from: p, with a draft that was not accepted max(p - q, 0).
template <Kind K>
struct Row {
  const void *target, *draft;
  int64_t at, drawn_at;
  int64_t certain;  // without the draft's probabilities: the token
  bool residual;
  __device__ __forceinline__ Row(const VerifyParams& p, const Tokens& r, int taken) {
    const int64_t t = r.t0 + taken;
    residual = taken < r.n - 1;
    target = p.target;
    draft = residual ? p.draft : nullptr;
    at = t * p.ts;
    drawn_at = (t + 1) * p.ds;
    certain = residual && p.draft == nullptr ? p.tokens[t + 1] : -1;
  }
  // Residual weights and probabilities of entries i .. i + 7.
  __device__ __forceinline__ void weights(int i, int end, double (&w)[kLane], double (&whole)[kLane]) const {
    float x[kLane], y[kLane];
    load8<K>(target, at, i, end, x);
    if (draft != nullptr) load8<K>(draft, drawn_at, i, end, y);
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      whole[e] = weight(x[e]);
      const double q = draft != nullptr ? weight(y[e]) : i + e == certain ? 1.0 : 0.0;
      w[e] = fmax(whole[e] - q, 0.0);
    }
  }
};

__device__ __forceinline__ double wave_total(double x) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

// Inclusive prefix over the wave's lanes.
__device__ __forceinline__ double wave_prefix(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  return x;
}

// Inclusive prefix over the workgroup in the threads' order, and the total; two barriers.
__device__ __forceinline__ double block_prefix(double x, double* sums, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_prefix(x);
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? sums[w] : 0.0;
    total += sums[w];
  }
  __syncthreads();
  return before + x;
}

// The least of the threads' x and the largest of their y; two barriers.
__device__ __forceinline__ int2 block_ends(int x, int y, int2* ends) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    x = min(x, __shfl_xor(x, m));
    y = max(y, __shfl_xor(y, m));
  }
  if ((threadIdx.x & 63) == 0) ends[threadIdx.x >> 6] = make_int2(x, y);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    x = min(x, ends[w].x);
    y = max(y, ends[w].y);
  }
  __syncthreads();
  return make_int2(x, y);
}

}  // namespace

template <Kind K>
__global__ __launch_bounds__(kTpb) void verify_sums_kernel(const VerifyParams p) {
  const int lane = threadIdx.x & 63, b = (int)blockIdx.y;
  const int seg = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + (int)(threadIdx.x >> 6));
  if (seg >= p.segments) return;
  const Tokens r = tokens_of(p, b);
  if (r.n == 0) return;
  const int taken = accepted_of<K>(p, r, lane);
  if (seg == 0 && lane == 0) p.taken[b] = taken;
  const Row<K> row(p, r, taken);
  const int first = seg * p.segment, end = min(p.V, first + p.segment);
  double s = 0.0, z = 0.0;
#pragma unroll 2
  for (int i = first + lane * kLane; i < end; i += kVerifyStep) {
    double w[kLane], whole[kLane];
    row.weights(i, end, w, whole);
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      s += w[e];
      z += whole[e];
    }
  }
  s = wave_total(s);
  z = wave_total(z);
  if (lane == 0) {
    double* out = p.sums + ((int64_t)b * p.segments + seg) * 2;
    out[0] = s;
    out[1] = z;
  }
}

template <Kind K>
__global__ __launch_bounds__(kTpb) void verify_pick_kernel(const VerifyParams p) {
  __shared__ double sums[kWaves];
  __shared__ int2 ends[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, b = (int)blockIdx.x;
  const Tokens r = tokens_of(p, b);
  // tokens of no request
  if (b == 0) {
    for (int t = tid; t < r.t0; t += kTpb) p.follows[t] = -1;
  }
  if (b == p.R - 1) {
    for (int t = r.t0 + r.n + tid; t < p.T; t += kTpb) p.follows[t] = -1;
  }
  if (r.n == 0) {
    if (tid == 0) {
      p.accepted[b] = 0;
      p.lens_out[b] = p.lens[b];
    }
    return;
  }
  const int taken = p.taken[b];
  const Row<K> row(p, r, taken);
  // ---- the segment: the first at which the running sum passes the goal, else the last with weight ----
  // Every wave for itself, a lane neighbouring segments: no barrier.
  const double* seg = p.sums + (int64_t)b * p.segments * 2;
  const int per = (p.segments + 63) / 64, s0 = lane * per, s1 = min(s0 + per, p.segments);
  double mine[2] = {0.0, 0.0};
  for (int s = s0; s < s1; ++s) {
    mine[0] += seg[s * 2];
    mine[1] += seg[s * 2 + 1];
  }
  // a residual without weight (the draft's probabilities are the target's) leaves the target's
  const int use = wave_total(mine[0]) > 0.0 ? 0 : 1;
  const double x = use == 0 ? mine[0] : mine[1];
  const double upto = wave_prefix(x), total = __shfl(upto, 63);
  const float u = p.sample[b];
  const double goal = (u > 0.f ? fmin((double)u, 1.0) : 0.0) * total;
  double run = upto - x, before = 0.0;  // weight ahead of the lane's segments, of its pick
  int pick = -1, last = -1;
  for (int s = s0; s < s1; ++s) {
    const double w = seg[s * 2 + use];
    if (w > 0.0) {
      last = s;
      if (pick < 0 && run + w > goal) {
        pick = s;
        before = run;
      }
    }
    run += w;
  }
  const uint64_t hits = __builtin_amdgcn_ballot_w64(pick >= 0), heavy = __builtin_amdgcn_ballot_w64(last >= 0);
  int next = -1;
  if (heavy != 0) {
    const bool passed = hits != 0;
    const int src = passed ? __builtin_ctzll(hits) : 63 - __builtin_clzll(heavy);
    pick = __shfl(passed ? pick : last, src);
    double base = __shfl(before, src);
    // ---- its entry, by the whole workgroup ----
    const int first = pick * p.segment, end = min(p.V, first + p.segment);
    int hit = 0x7fffffff, most = -1;
    for (int i0 = first; i0 < end && hit == 0x7fffffff; i0 += kTpb * kLane) {
      const int i = min(i0 + tid * kLane, end);
      double w[kLane], whole[kLane], sum = 0.0;
      row.weights(i, end, w, whole);
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        if (use == 1) w[e] = whole[e];
        sum += w[e];
      }
      double all;
      double at = base + (block_prefix(sum, sums, all) - sum);
      int found = 0x7fffffff, heaviest = -1;
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        at += w[e];
        if (w[e] > 0.0 && at > goal && found == 0x7fffffff) found = i + e;
        if (w[e] > 0.0) heaviest = i + e;
      }
      // one pass for both: the least entry that passes the goal, the last with weight
      const int2 both = block_ends(passed ? found : 0x7fffffff, heaviest, ends);
      hit = both.x;
      most = max(most, both.y);
      base += all;
    }
    next = hit != 0x7fffffff ? hit : most;
  }
  for (int i = tid; i < r.n; i += kTpb) {
    const int64_t t = r.t0 + i;
    p.follows[t] = i < taken ? p.tokens[t + 1] : i == taken ? (int64_t)next : -1;
  }
  if (tid == 0) {
    p.accepted[b] = taken;
    p.lens_out[b] = p.lens[b] - (r.n - 1 - taken);
  }
}

hipError_t launch_verify(const VerifyParams& p, int kind, hipStream_t stream) {
  auto go = [&](auto k) {
    constexpr Kind K = decltype(k)::value;
    hipLaunchKernelGGL((verify_sums_kernel<K>), dim3((unsigned)((p.segments + kWaves - 1) / kWaves), (unsigned)p.R), dim3(kTpb), 0, stream, p);
    hipLaunchKernelGGL((verify_pick_kernel<K>), dim3((unsigned)p.R), dim3(kTpb), 0, stream, p);
  };
  switch (kind) {
    case 0: go(std::integral_constant<Kind, Kind::f16>{}); break;
    case 1: go(std::integral_constant<Kind, Kind::bf16>{}); break;
    default: go(std::integral_constant<Kind, Kind::f32>{}); break;
  }
  return hipGetLastError();
}

}  // namespace gfa
