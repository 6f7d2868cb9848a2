// Attention over the key/value cache in 4 bits, many query rows per request: the kernel's instances (gfa_kv4_chunk.h), gfx950.
#include "gfa_kv4_chunk.h"
#include "gfa_launch.h"

namespace gfa {

template <int D, bool IS_BF16, bool CAP>
__global__ __launch_bounds__(256, kv4_chunk_wgs(D)) void kv4_chunk_kernel(const Kv4AttnParams p) {
  constexpr Kv4Part PART = kWhole;
  constexpr int TILE = Kv4Layout<D>::TILE_CODES;
  __shared__ __attribute__((aligned(1024))) char k_lds0[TILE], k_lds1[TILE], v_lds0[TILE], v_lds1[TILE], s_lds0[1024], s_lds1[1024];
  char GFA_LDS* const K0 = (char GFA_LDS*)k_lds0;
  char GFA_LDS* const K1 = (char GFA_LDS*)k_lds1;
  char GFA_LDS* const V0 = (char GFA_LDS*)v_lds0;
  char GFA_LDS* const V1 = (char GFA_LDS*)v_lds1;
  char GFA_LDS* const S0 = (char GFA_LDS*)s_lds0;
  char GFA_LDS* const S1 = (char GFA_LDS*)s_lds1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = (int)blockIdx.x;
  const int head = p.hkv.rem(block);
  constexpr int ROWS = kv4_chunk_rows(D);
  const Item it = find_item<ROWS, true>(p, p.hkv.quot(block), lane);
  if (it.b < 0) return;
#include "gfa_kv4_chunk.inc"
}

// Explicit instantiations: the host launch stubs must exist for each variant.
#define GFA_KV4_CHUNK_INST(DD)                                                      \
  template __global__ void kv4_chunk_kernel<DD, true, true>(const Kv4AttnParams);   \
  template __global__ void kv4_chunk_kernel<DD, true, false>(const Kv4AttnParams);  \
  template __global__ void kv4_chunk_kernel<DD, false, true>(const Kv4AttnParams);  \
  template __global__ void kv4_chunk_kernel<DD, false, false>(const Kv4AttnParams);
GFA_KV4_CHUNK_INST(64)
GFA_KV4_CHUNK_INST(128)
GFA_KV4_CHUNK_INST(256)
GFA_KV4_CHUNK_INST(512)
#undef GFA_KV4_CHUNK_INST

hipError_t launch_kv4_chunk(const Kv4AttnParams& p, int D, bool bf16, bool cap, hipStream_t stream) {
  auto go = [&](auto d, auto b, auto c) {
    constexpr int DD = decltype(d)::value;
    constexpr bool BB = decltype(b)::value, CC = decltype(c)::value;
    hipLaunchKernelGGL((kv4_chunk_kernel<DD, BB, CC>), dim3((unsigned)p.nblocks), dim3(256), 0, stream, p);
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
