// Pieces that the two kernels of attend_tree share.
#pragma once

#include "kernels.cuh"
#include "ptx.cuh"

namespace wv {

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar,
                                            int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// hi + lo = (x, y) to 2^-22 of each.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = pack_half2(x, y);
  const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&hi));
  lo = pack_half2(x - f.x, y - f.y);
}

// The pair with zeros for infinities and NaN.
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  if ((v & 0x7c00u) == 0x7c00u) v &= 0xffff0000u;
  if ((v & 0x7c000000u) == 0x7c000000u) v &= 0x0000ffffu;
  return v;
}

}  // namespace wv
