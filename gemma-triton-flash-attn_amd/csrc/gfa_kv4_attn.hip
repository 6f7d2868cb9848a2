// Attention over the key/value cache in 4 bits, few query rows per request: the kernel's instances (gfa_kv4_split.h), gfx950.
#include "gfa_kv4_split.h"
#include "gfa_launch.h"

namespace gfa {

template <int D, bool IS_BF16, bool CAP, bool ONCE>
__global__ __launch_bounds__(kWaves * 64, D == 512 ? 1 : 2) void kv4_split_kernel(const Kv4AttnParams p) {
  constexpr Kv4Part PART = kWhole;
  __shared__ __attribute__((aligned(16))) f32x4 sums_lds[kWaves][D / 16 * 64];
  auto o_lds = [&](int w) __attribute__((always_inline)) { return sums_lds[w]; };
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = (int)blockIdx.x;
  const int head = p.hkv.rem(block);
  const Item it = find_item<kRows, false>(p, p.hkv.quot(block), lane);
  if (it.b < 0) {
    if (p.cu == nullptr) return;
    const int64_t taken = (int64_t)it.items * p.cache.Hkv;
    zero_rows<D>(p, threadIdx.x, block - taken, p.nblocks - taken);
    return;
  }
#include "gfa_kv4_split.inc"
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
