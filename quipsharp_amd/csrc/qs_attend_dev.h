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
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct PagePool {
  const uint16_t *k, *v;
  int64_t k_page, k_head, v_page, v_head;
  int k_pos, v_pos;
  int pages, shift;  // pages of the pool; log2 of the positions of a page
  const int32_t* table;
  int64_t table_ld;
  int cols;
  const int32_t *lengths, *over;  // over: per row, or null
};

// Where a row's tokens end, which may lie beyond the `most` positions that its
// table has room for: at its length, or where that is the table's end, `over`
// further.
__device__ __forceinline__ int end_of(const int32_t* lengths, const int32_t* over, int most, int64_t row) {
  const int n = lengths[row] < 0 ? 0 : lengths[row];
  if (!over || n != most) return n;
  const int o = over[row] < 0 ? 0 : over[row];
  return o < INT32_MAX - n ? n + o : INT32_MAX;
}

// What a query at position `at` sees of a table with room for `most`
// positions: positions low .. last and those below sinks (sinks <= low; zero
// without a window).  The window goes by where the query is; of what it holds,
// positions beyond the table are left out here, so that no kernel looks for
// them (low may lie beyond last then).
struct Span {
  int low, last, sinks;
};

__device__ __forceinline__ Span span_of(int at, int window, int sinks, int most) {
  Span s;
  s.last = at < most ? at : most - 1;
  s.low = window > 0 && at >= window ? at - window + 1 : 0;
  s.sinks = sinks < s.low ? sinks : s.low;
  if (s.sinks > most) s.sinks = most;
  return s;
}

// The positions that a span touches, in tiles of T positions: first the
// sinks' tiles, then the window's (a tile of both is one of the window's).
template <int T>
struct TileList {
  int sink, low, count;
  __device__ __forceinline__ explicit TileList(const Span& s) {
    const bool window = s.low <= s.last;
    low = s.low / T;
    sink = (s.sinks + T - 1) / T;
    if (window && sink > low) sink = low;
    count = sink + (window ? s.last / T - low + 1 : 0);
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

constexpr float kLog2E = 1.44269504088896340736f;

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

// 16 bytes per lane from base + off straight to LDS, at `lds` + AT + 16 lane.  The
// compiler does not count this load: wait_loads before the bytes are read.
// (Its own form would have it wait for all such loads before the next read of
// LDS, whatever place that reads.)
template <int AT>
__device__ __forceinline__ void load_to_lds(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base), "n"(AT)
               : "memory", "m0", "scc");
}
// N loads whose lanes' places behind base are off, one after the other in LDS.
template <int N, int AT = 0>
__device__ __forceinline__ void load_rows(const char* base, const unsigned (&off)[N], unsigned lds) {
  if constexpr (AT < N) {
    load_to_lds<1024 * AT>(base, off[AT], lds);
    load_rows<N, AT + 1>(base, off, lds);
  }
}
// All but the last N of the wave's loads are there (loads that are written in
// the program between two of these calls stay between them).
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)(p);
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
//
// The loads are the whole cost, so each of them takes whole rows: keys go
// straight to the wave's own part of LDS (a lane's operand is 16 bytes of each
// of 16 rows, and loads in that shape took 288 us instead of 281 over 1.6 GB,
// 10.3 instead of 8.0 us over 577 positions), values lie as they are used, 16
// lanes to a row: the operand wants 8 positions of one dimension, so the lane
// takes rows 4 qd + j and 16 + 4 qd + j and puts halves together, and the
// dimension of operand row m of tile j is DPL m + j.
//
// All columns are heads of one token and see the same positions.  NT: values
// are loaded past the caches.
template <bool BF, int HD, bool NT>
struct WaveAttend {
  static constexpr int DPL = HD / 16;   // dimensions per lane of a value row
  static constexpr int KS = HD / 32;    // steps of the score product
  static constexpr int kRow = HD * 2;   // bytes of a position in LDS
  static constexpr int kKeys = 32 * kRow;
  static constexpr int CPR = HD / 8;    // 16-byte pieces of a position
  static constexpr int NJ = 16 * CPR / 64, RJ = 64 / CPR;  // loads of 16 positions, positions of a load
  static constexpr int kSwz = CPR < 16 ? 7 : 15;
  static constexpr int NV = DPL == 4 ? 8 : DPL;  // loads of the values
  uint4 q[KS];
  f32x4 o[DPL];
  float top, sum;   // of the products q k; the sum is over this lane's positions
  unsigned ko[NJ];  // where the lane's piece of a load lies behind the first of 16 positions
  unsigned lds;     // the wave's part
  const char* keys;

  __device__ __forceinline__ void init(const PagePool& pp, const char* at) {
    const int lane = __lane_id();
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int r = j * RJ + lane / CPR;
      ko[j] = 2u * (r * pp.k_pos + 8 * ((lane % CPR) ^ (r & kSwz)));
    }
    keys = at;
    lds = __builtin_amdgcn_readfirstlane(lds_address(at));
  }

  // Positions p0 .. p0 + 31 (p0 a multiple of 32) of kv head g, the pages of
  // whose halves are e (-1: none); s is the columns' span, `all` that it
  // holds every position.  e, p0, s and all are the same for the whole wave.
  __device__ __forceinline__ void step(const PagePool& pp, const int (&e)[2], int g, int p0, const Span& s, bool all,
                                       float scale, LaneX lx) {
    const int lane = __lane_id(), r16 = lane & 15, qd = lane >> 4;
    const int mask = (1 << pp.shift) - 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t id = e[t] < 0 ? 0 : e[t];
      const char* kb = reinterpret_cast<const char*>(pp.k + id * pp.k_page + g * pp.k_head + (int64_t)((p0 + 16 * t) & mask) * pp.k_pos);
      load_rows<NJ>(kb, ko, lds + 16 * t * kRow);
    }
    uint32_t vr[8][DPL / 2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t id = e[t] < 0 ? 0 : e[t];
      const uint16_t* vb = pp.v + id * pp.v_page + g * pp.v_head + (int64_t)((p0 + 16 * t) & mask) * pp.v_pos;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint16_t* a = vb + (unsigned)((4 * qd + j) * pp.v_pos + DPL * r16);
        uint32_t* to = vr[4 * t + j];
        if constexpr (DPL == 4) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(a);
          to[0] = x[0], to[1] = x[1];
        } else {
#pragma unroll
          for (int i = 0; i < DPL / 8; ++i) {
            const u32x4* from = reinterpret_cast<const u32x4*>(a + 8 * i);
            u32x4 x;
            if constexpr (NT) x = __builtin_nontemporal_load(from);
            else x = *from;
            to[4 * i] = x[0], to[4 * i + 1] = x[1], to[4 * i + 2] = x[2], to[4 * i + 3] = x[3];
          }
        }
      }
    }
    wait_loads<NV>();
    f32x4 st[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint4 kf = *reinterpret_cast<const uint4*>(keys + (16 * t + r16) * kRow + 16 * ((4 * ks + qd) ^ (r16 & kSwz)));
        st[t] = mma_16x16x32<BF>(kf, q[ks], st[t]);
      }
    }
    if (!all || (e[0] | e[1]) < 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = p0 + 16 * t + 4 * qd + j;
          const bool see = e[t] >= 0 && p <= s.last && (p >= s.low || p < s.sinks);
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
    // the weights in the cache's type, as the matrix instructions take them (half a step of each, in their sum none):
    // an output is off by 0.20 % in the 2-norm in bf16, its own rounding alone is 0.165 %
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

// The positions that `span` + 1 tokens in a row see at most, of `room`.
inline int64_t seen_positions(int64_t room, int window, int sinks, int64_t span) {
  const int64_t n = (int64_t)window + sinks + span;
  return window > 0 && n < room ? n : room;
}

// A part of a token's head: its maximum, its sum, two words that keep what
// follows 16-byte aligned, and head_dim sums of weighted values.
constexpr int kPartHead = 4;
constexpr int part_floats(int head_dim) { return kPartHead + head_dim; }

// The tiles of one share of a single token's: at least one for each wave, so
// that a short row in a table of many columns uses few of the shares.
constexpr int kShareTiles = 4;
__host__ __device__ __forceinline__ int share_tiles(int count, int splits) {
  const int n = (count + splits - 1) / splits;
  return n < kShareTiles ? kShareTiles : n;
}

// Which parts of a single token's head there are: those of its row's tiles.
struct Used {
  const int32_t *lengths, *over;
  int most;  // positions that the table has room for
  int window, sinks;
};

// The parts (part[token][head][split]) of `tokens` tokens' heads together;
// used: null where all are there.
int join_parts(const float* part, int splits, const Used* used, int64_t tokens, int heads, int head_dim, bool bf, float scale,
               uint16_t* out, int64_t out_token, hipStream_t stream);

// The argument checks of the attention calls; fills `out`.
int page_pool_checks(const char* fn, const qs_page_pool* p, int dtype, int64_t rows, int heads, int kv_heads,
                     int head_dim, float scale, int window, int sinks, const int32_t* over, PagePool& out);

}  // namespace qs
