// The order of logits as whole numbers, and sums and order statistics of a
// wave: what beam selection (qs_beam.hip) and the log probabilities of tokens
// (qs_logprobs.hip) share.
#pragma once

#include "qs_chunk_dev.h"

namespace qs {

// Order-preserving bits of a float; -0 counts as 0, NaN as -inf.
__device__ __forceinline__ uint32_t order_bits(float f) {
  f = f != f ? -INFINITY : f + 0.0f;
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_float(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

__device__ __forceinline__ double wave_sum64(double v, LaneX lx) {
  auto add = [&](auto other) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(other(__uint_as_float((uint32_t)u))), hi = __float_as_uint(other(__uint_as_float((uint32_t)(u >> 32))));
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  add([&](float x) { return lane_xor<32>(x, lx); });
  add([&](float x) { return lane_xor<16>(x, lx); });
  add([&](float x) { return lane_xor<8>(x, lx); });
  add([&](float x) { return lane_xor<4>(x, lx); });
  add([&](float x) { return lane_xor<2>(x, lx); });
  add([&](float x) { return lane_xor<1>(x, lx); });
  return v;
}

// The largest u such that at least n lanes (1 .. 64) have a key of u or more.
__device__ __forceinline__ uint32_t nth_key(uint32_t key, int n) {
  uint32_t u = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t v = u | 1u << bit;
    if (__popcll(__ballot(key >= v)) >= n) u = v;
  }
  return u;
}

}  // namespace qs
