// Attention over a paged key-value cache: what the kernels for single tokens
// (qs_attend_token.hip) and for several (qs_attend_chunk.hip) share, and the
// step of one wave for a single token.
//
// A cache page holds `page` positions (a power of two, 16 or more) of every
// kv head: element (id, head, position, d) of the key pool is
// k[id * k_page + head * k_head + position * k_pos + d]; values likewise.
// Row r keeps position p on page table[r][p / page]; an entry outside the
// pool, or a column outside the table, leaves the 16 positions read there out.
#pragma once

#include "qs_chunk_dev.h"

namespace qs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct PagePool {
  const uint16_t *k, *v;
  int64_t k_page, k_head, v_page, v_head;
  int k_pos, v_pos;
  int pages, shift;  // pages of the pool; log2 of the positions of a page
  const int32_t* table;
  int64_t table_ld;
  int cols;
  const int32_t* lengths;
};

// What a query at position `last` sees: positions low .. last and those below
// sinks (sinks <= low; zero without a window).
struct Span {
  int low, last, sinks;
};

__device__ __forceinline__ Span span_of(int last, int window, int sinks) {
  Span s;
  s.last = last;
  s.low = window > 0 && last >= window ? last - window + 1 : 0;
  s.sinks = sinks < s.low ? sinks : s.low;
  return s;
}

// The positions that a span touches, in tiles of T positions: first the
// sinks' tiles, then the window's (a tile of both is one of the window's).
template <int T>
struct TileList {
  int sink, low, count;
  __device__ __forceinline__ explicit TileList(const Span& s) {
    low = s.low / T;
    sink = (s.sinks + T - 1) / T;
    if (sink > low) sink = low;
    count = s.last < 0 ? 0 : sink + s.last / T - low + 1;
  }
  __device__ __forceinline__ int at(int u) const { return u < sink ? u : low + u - sink; }
};

template <bool BF>
__device__ __forceinline__ f32x4 mma_16x16x32(const uint4& a, const uint4& b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two floats to the 16-bit type, to nearest even: lo in bits 0-15.
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF) {
    return f32x2_to_bf16x2(lo, hi);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2));
  }
}

// The weight of a score that lies `below` the maximum; scale holds log2(e).
// The difference is taken before the product, which could leave the range of
// fp32 for scores near its end.
__device__ __forceinline__ float weight(float below, float scale) { return __builtin_amdgcn_exp2f(below * scale); }

// The same times 2^14 in fp16, where it is rounded to the cache's type: without
// it weights below 2^-14 of the largest would be subnormal there.  The sums
// and the outputs carry the factor until they are divided.
template <bool BF>
__device__ __forceinline__ float lifted_weight(float below, float scale) {
  return __builtin_amdgcn_exp2f(BF ? below * scale : __builtin_fmaf(below, scale, 14.0f));
}

// A query as it is, or its negative (flip = 0x80008000) where the scale is
// negative: the kernels' scale is positive, so that the largest product has
// the largest weight.
__device__ __forceinline__ uint4 flipped(uint4 x, uint32_t flip) {
  return make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
}

// One wave's attention of 16 query columns (the heads of a token) over
// tiles of 32 positions, with the running maximum and sum of the softmax.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that
// the column of a query is the lane's own (lane & 15) all the way through:
// the 16x16x32 result of S^T leaves lane (qd = lane / 16) with positions 4 qd
// + j of each 16, which is what it hands to the second product as its 8 of 32
// positions -- the order of the positions inside a sum is free -- and the
// maximum, the sum and the rescaling of O are the lane's own registers.
// Values are read as they lie, 16 lanes to a row; the operand wants 8
// positions of one dimension, so the lane takes rows 4 qd + j and 16 + 4 qd +
// j and puts halves together, and the dimension of operand row m of tile j is
// DPL m + j.  Nothing goes through LDS.
//
// All columns are heads of one token and see the same positions.
template <bool BF, int HD>
struct WaveAttend {
  static constexpr int DPL = HD / 16;  // dimensions per lane of a value row
  static constexpr int KS = HD / 32;   // steps of the score product
  uint4 q[KS];
  f32x4 o[DPL];
  float top, sum;  // of the products q k; the sum is over this lane's positions

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    top = -INFINITY, sum = 0.f;
  }

  // Positions p0 .. p0 + 31 (p0 a multiple of 32) of kv head g; s is the
  // column's span, `all` (uniform) that every column sees every position.
  __device__ __forceinline__ void step(const PagePool& pp, const int32_t* trow, int g, int p0, const Span& s, bool all,
                                       float scale, LaneX lx) {
    const int lane = __lane_id(), r16 = lane & 15, qd = lane >> 4;
    const int mask = (1 << pp.shift) - 1;
    int64_t id[2];
    bool ok[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int col = (p0 + 16 * t) >> pp.shift;
      const int e = col < pp.cols ? trow[col] : -1;
      ok[t] = e >= 0 && e < pp.pages;
      id[t] = ok[t] ? e : 0;
    }
    uint4 kf[2][KS];
    uint32_t vr[8][DPL / 2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* kb = pp.k + id[t] * pp.k_page + g * pp.k_head + (int64_t)((p0 + 16 * t) & mask) * pp.k_pos;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[t][ks] = *reinterpret_cast<const uint4*>(kb + r16 * pp.k_pos + 32 * ks + 8 * qd);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* vb = pp.v + id[t] * pp.v_page + g * pp.v_head + (int64_t)((p0 + 16 * t) & mask) * pp.v_pos;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint16_t* a = vb + (4 * qd + j) * pp.v_pos + DPL * r16;
        uint32_t* to = vr[4 * t + j];
        if constexpr (DPL == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(a);
          to[0] = x.x, to[1] = x.y;
        } else {
#pragma unroll
          for (int i = 0; i < DPL / 8; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(a + 8 * i);
            to[4 * i] = x.x, to[4 * i + 1] = x.y, to[4 * i + 2] = x.z, to[4 * i + 3] = x.w;
          }
        }
      }
    }
    f32x4 st[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) st[t] = mma_16x16x32<BF>(kf[t][ks], q[ks], st[t]);
    }
    if (!all || !ok[0] || !ok[1]) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = p0 + 16 * t + 4 * qd + j;
          const bool see = ok[t] && p <= s.last && (p >= s.low || p < s.sinks);
          st[t][j] = see ? st[t][j] : -INFINITY;
          // what lies in a place that is not seen may be no number, and 0 times it would be none either
#pragma unroll
          for (int i = 0; i < DPL / 2; ++i) vr[4 * t + j][i] = see ? vr[4 * t + j][i] : 0u;
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                     fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
    mx = fmaxf(mx, lane_xor<16>(mx, lx));
    mx = fmaxf(mx, lane_xor<32>(mx, lx));
    mx = fmaxf(mx, top);
    const float base = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every weight below is 0
    const float f = weight(top - base, scale);
    top = mx;
    float pr[2][4], t8 = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pr[t][j] = lifted_weight<BF>(st[t][j] - base, scale);
        t8 += pr[t][j];
      }
    sum = sum * f + t8;
    // the weights in the cache's type, as the matrix instructions take them: half a step of at most 1
    const uint4 pb = make_uint4(pack16<BF>(pr[0][0], pr[0][1]), pack16<BF>(pr[0][2], pr[0][3]),
                                pack16<BF>(pr[1][0], pr[1][1]), pack16<BF>(pr[1][2], pr[1][3]));
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
      const uint4 a = make_uint4(__builtin_amdgcn_perm(vr[1][j / 2], vr[0][j / 2], sel),
                                 __builtin_amdgcn_perm(vr[3][j / 2], vr[2][j / 2], sel),
                                 __builtin_amdgcn_perm(vr[5][j / 2], vr[4][j / 2], sel),
                                 __builtin_amdgcn_perm(vr[7][j / 2], vr[6][j / 2], sel));
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] *= f;
      o[j] = mma_16x16x32<BF>(a, pb, o[j]);
    }
  }

  // The sum over the whole column (every lane of it gets it).
  __device__ __forceinline__ float total(LaneX lx) const {
    float t = sum + lane_xor<16>(sum, lx);
    return t + lane_xor<32>(t, lx);
  }
};

// The argument checks of the attention calls; fills `out`.
int page_pool_checks(const char* fn, const qs_page_pool* p, int dtype, int64_t rows, int heads, int kv_heads,
                     int head_dim, float scale, int window, int sinks, PagePool& out);

}  // namespace qs
