// Pieces that the two kernels of attend_tree share.
#pragma once

#include "kernels.cuh"
#include "ptx.cuh"
#include "softmax.cuh"

namespace wv {

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar,
                                            int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// hi + lo = (x, y) to 2^-22 of each, or to 2^-25 where lo is subnormal.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = pack_half2(x, y);
  const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&hi));
  lo = pack_half2(x - f.x, y - f.y);
}

// Probabilities meet V in f16, at most 2^kLift, near the top of f16's range, which leaves 29 binary
// orders below it at full precision and 10 more with less. (At most 1 they are 14 and 10: a
// probability of 1e-5 keeps three digits and one below 3e-8 none, while the sum that divides keeps
// both.) One f16 part: the exponents' reference is that much lower, and the sum carries the factor
// too. Two parts: the products alone carry it (an exponent near 15 is rounded to 2^-21, which f32
// would show).
constexpr int kLift = 15;
constexpr float kLowUp = 2048.0f;

// hi + lo / 2^11 = (x, y) UP to 2^-22 of each, or to 2^-36 where lo is subnormal.
template <int UP>
__device__ __forceinline__ void split2_up(float x, float y, uint32_t &hi, uint32_t &lo) {
  constexpr float up = float(1 << UP);
  float a, b;
  fma2(a, b, x, y, up, up, 0.0f, 0.0f);
  hi = pack_half2(a, b);
  const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&hi));
  add2(a, b, a, b, -f.x, -f.y);
  fma2(a, b, a, b, kLowUp, kLowUp, 0.0f, 0.0f);
  lo = pack_half2(a, b);
}

// The pair with zeros for infinities and NaN.
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  if ((v & 0x7c00u) == 0x7c00u) v &= 0xffff0000u;
  if ((v & 0x7c000000u) == 0x7c000000u) v &= 0x0000ffffu;
  return v;
}

}  // namespace wv
