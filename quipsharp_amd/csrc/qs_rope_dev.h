// RMSNorm over a 128-wide head and the rotary embedding, with one arithmetic
// wherever they run: the decode-step kernels (qs_decoder.hip) and the paged
// cache's append (qs_pages.hip).
#pragma once

#include "qs_chunk_dev.h"

namespace qs {

__device__ __forceinline__ float bf(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ float rbf(float f) { return bf(f32_to_bf16(f)); }  // round through bf16

// cos and sin of the rotary embedding at one position, dims l and l + 64.
struct Rot {
  float c0, c1, s0, s1;
};

__device__ __forceinline__ Rot load_rot(const uint16_t* cos_r, const uint16_t* sin_r, int l) {
  return Rot{bf(cos_r[l]), bf(cos_r[l + 64]), bf(sin_r[l]), bf(sin_r[l + 64])};
}

// q_norm / k_norm (RMSNorm over the head dim) and the rotary embedding of
// one 128-wide head, one wave: lane l holds dims l and l + 64 (x0, x1; the
// pair rotate_half mixes) and the norm weights there (w0, w1); o0 / o1 the
// bf16 results.  The sum of squares is a lane-local fma then a fixed
// butterfly, so every kernel that calls this gets the same bits.
__device__ __forceinline__ void norm_rope(float x0, float x1, float w0, float w1, const Rot& r, float eps, LaneX lx,
                                          uint16_t& o0, uint16_t& o1) {
  float ss = __builtin_fmaf(x1, x1, x0 * x0);
  ss += lane_xor<32>(ss, lx);
  ss += lane_xor<16>(ss, lx);
  ss += lane_xor<8>(ss, lx);
  ss += lane_xor<4>(ss, lx);
  ss += lane_xor<2>(ss, lx);
  ss += lane_xor<1>(ss, lx);
  const float rs = 1.0f / sqrtf(__builtin_fmaf(ss, 1.0f / 128.0f, eps));
  const float y0 = rbf(w0 * rbf(x0 * rs)), y1 = rbf(w1 * rbf(x1 * rs));
  // q * cos + rotate_half(q) * sin, rotate_half(q) = (-q[64:], q[:64])
  o0 = f32_to_bf16(rbf(y0 * r.c0) + (-rbf(y1 * r.s0)));
  o1 = f32_to_bf16(rbf(y1 * r.c1) + rbf(y0 * r.s1));
}

}  // namespace qs
