// Causal attention of several new tokens per row over the row's cache pages
// (qs_attend_chunk).  The tokens of row r are q[starts[r]] .. q[starts[r + 1]
// - 1]; the last of them is at position lengths[r] - 1.
#include <cmath>
#include <type_traits>

#include "qs_attend_dev.h"

namespace qs {
namespace {

constexpr int kWaves = 4;
constexpr int kCols = 32 * kWaves;  // query columns (a head of a token each) of a work-group

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_token, q_head;
  uint16_t* out;
  int64_t out_token;
  const int32_t* starts;
  int tokens, rows, heads, kv_heads, window, sinks;
  float* part;
  int splits;
  float scale;    // its size, times log2(e)
  uint32_t flip;  // its sign, for a pair of elements
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <bool BF>
__device__ __forceinline__ f32x16 mma_32x32x16(const uint4& a, const uint4& b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF>
__device__ __forceinline__ float from16(uint16_t x) {
  if constexpr (BF) return __uint_as_float((uint32_t)x << 16);
  else return (float)__builtin_bit_cast(_Float16, x);
}

// The bits of two elements' exponents: all of them set for infinities and no
// numbers.
template <bool BF>
constexpr uint32_t exponents() { return BF ? 0x7F807F80u : 0x7C007C00u; }

// Two elements as finite ones (0 for the others) and ones at +inf and at -inf;
// no number counts as both, whose sum is none.
template <bool BF>
struct Parted {
  uint32_t finite, plus, minus;
  __device__ __forceinline__ explicit Parted(uint32_t two) {
    const uint32_t lack = ~two & exponents<BF>(), one = BF ? 0x3F80u : 0x3C00u;
    const uint32_t odd = (lack - 0x00010001u) & ~lack & 0x80008000u;  // bits 15 and 31: nothing lacks
    const uint32_t none = odd & ((two & (BF ? 0x007F007Fu : 0x03FF03FFu)) + 0x7FFF7FFFu);
    finite = two & ~((odd >> 15) * 0xFFFFu);
    plus = ((odd & (~two | none)) >> 15) * one;
    minus = ((odd & (two | none)) >> 15) * one;
  }
};

// 4 rows of 16 elements from LDS, transposed: lane i of 16 gives the address
// of elements 4 (i % 4) .. + 3 of row i / 4 and gets element i of the rows.
__device__ __forceinline__ uint2 read_transposed(const char* at) {
  typedef __attribute__((address_space(3))) s16x4* lds_t;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(at)));
}

__device__ __forceinline__ int wave_total(int v, LaneX lx) {
  auto other = [&](auto x) { return __builtin_bit_cast(int, x); };
  auto f = [&]() { return __builtin_bit_cast(float, v); };
  v += other(lane_xor<32>(f(), lx));
  v += other(lane_xor<16>(f(), lx));
  v += other(lane_xor<8>(f(), lx));
  v += other(lane_xor<4>(f(), lx));
  v += other(lane_xor<2>(f(), lx));
  v += other(lane_xor<1>(f(), lx));
  return __builtin_amdgcn_readfirstlane(v);
}

// The query columns of a work-group: columns 128 b .. of row `row`, whose
// tokens are first .. first + count - 1.
struct Block {
  int row, b, first, count;
};

// Row r's tokens are first .. first + count - 1.
__device__ __forceinline__ int first_of(const ChunkArgs& a, int r) {
  const int x = a.starts[r];
  return x < 0 ? 0 : x > a.tokens ? a.tokens : x;
}

// The k-th block of the call; false where there are fewer.  Up to 64 rows are
// looked at together, a lane for each, and their blocks are taken in the order
// of their ends, the latest position first: a long one that begins last would
// have the chip wait for it (six rows of up to 1500 new tokens behind up to
// 4000: 288 us instead of 300).  The block at hand is found by its end: the
// largest x such that more than k blocks end at x or beyond.
__device__ __forceinline__ bool find_block(const ChunkArgs& a, const PagePool& pp, int k, int group, LaneX lx, Block& out) {
  const int lane = __lane_id();
  if (a.rows > 64) {
    // Row by row, the end of each first.  The numbers from base(r) on are the
    // row's: as many as it has blocks, or one more that stands for none.
    auto base = [&](int r) { return (int)((int64_t)first_of(a, r) * group / kCols) + r; };
    int lo = 0, hi = a.rows;
    if (k < base(0)) return false;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, r = lo + lane * step;
      const uint64_t at = __ballot(r < hi && base(r < hi ? r : lo) <= k);
      lo += (63 - __clzll((unsigned long long)(at | 1))) * step;
      hi = lo + step < hi ? lo + step : hi;
    }
    const int first = first_of(a, lo), count = first_of(a, lo + 1) - first, n = (count * group + kCols - 1) / kCols;
    out = Block{lo, n - 1 - (k - base(lo)), first, count};
    return count > 0 && out.b >= 0;
  }
  // a lane's row: its tokens, its blocks, the position of its first token
  int first = 0, count = 0, n = 0, p0 = 0;
  if (lane < a.rows) {
    first = first_of(a, lane);
    const int end = first_of(a, lane + 1);
    count = end > first ? end - first : 0;
    n = (count * group + kCols - 1) / kCols;
    // for the order alone: a row that ends beyond its table counts as one that ends with it
    const int len = pp.lengths[lane] < 0 ? 0 : pp.lengths[lane], most = pp.cols << pp.shift;
    p0 = (len < most ? len : most) - count;
  }
  if (a.rows == 1) {
    out = Block{0, __builtin_amdgcn_readfirstlane(n) - 1 - k, __builtin_amdgcn_readfirstlane(first), __builtin_amdgcn_readfirstlane(count)};
    return out.b >= 0;
  }
  // how many of the row's blocks end at position x or beyond
  auto from = [&](int64_t x) {
    const int64_t t = x - p0;  // from this token on
    return t <= 0 ? n : t >= count ? 0 : n - (int)t * group / kCols;
  };
  auto blocks_from = [&](int64_t x) { return wave_total(from(x), lx); };
  // blocks_from(lo) > k >= blocks_from(hi)
  int64_t lo = -a.tokens, hi = ((int64_t)pp.cols << pp.shift) + 1;
  if (k >= blocks_from(lo)) return false;
  while (hi - lo > 1) {
    const int64_t mid = lo + (hi - lo) / 2;
    if (blocks_from(mid) > k) lo = mid; else hi = mid;
  }
  k -= blocks_from(hi);  // among those that end at lo, by row
  const int beyond = from(hi), here = from(lo) - beyond;
  int upto = here;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(upto, d, 64);
    if (lane >= d) upto += y;
  }
  const uint64_t over = __ballot(k < upto);
  if (!over) return false;
  const int l = __ffsll((unsigned long long)over) - 1;
  out.row = l;
  out.b = __builtin_amdgcn_readlane(n - beyond - here + upto, l) - 1 - k;
  out.first = __builtin_amdgcn_readlane(first, l);
  out.count = __builtin_amdgcn_readlane(count, l);
  return true;
}

// out[t][h] = sum_p w_p v_p, w = softmax(scale q_t,h . k_p) over the positions
// that token t sees, in one pass with the running maximum and sum.
//
// One work-group per kv head and 128 columns of a row, column c being head c %
// group of the row's token c / group; one wave per 32 of them, whose sums stay
// in its registers.  Tiles of kT positions go through LDS, which all four
// waves read, past the registers; the next tile is on its way while one is
// worked on.  8192 tokens under a window of 1024 took 616 us with every wave
// loading every tile from the L1, 242 through the registers, 208 past them,
// and take 169 now.
// Two work-groups share a CU, so that one's softmax runs beside the other's
// products.  Both products are transposed, so that a column stays the lane's
// own (lane & 31): a 32x32 result of K Q^T leaves lane (hf = lane / 32) with
// positions 8 a + 4 hf + {0 .. 3}, and the second product takes 8 of them at a
// step, with the values read through LDS's transposing load.
//
// The weights refer to a base that follows the running maximum only where it
// has fallen 2^8 behind, so that most tiles rescale nothing; in fp16 they
// carry a factor of 2^7 too, which keeps 2^-21 of the largest from being
// subnormal and the largest below 2^15.  They are rounded to the cache's type
// for the second product, and their sum is that of the unrounded ones: an
// output is off by 0.20 to 0.22 % in the 2-norm in bf16 (fp16: an eighth),
// where its own rounding alone is 0.165 %.
//
// Bound by the matrix and vector instructions, which run nearly one after the
// other (of 365 k cycles matrix units are busy 138 k and vector units 167 k),
// at the clock that their power leaves: 129 GFLOP in 169 us (8192 tokens,
// window 1024) and 237 in 276 (six rows), 760 and 860 TFLOP/s, where the
// products alone would run at 1750.  Heads of 256 (one wave a SIMD, tiles of
// 32): 4096 tokens of 16 heads 236 us, 583 TFLOP/s.
//
// GR = 2: eight waves, of which the second four take every other tile; their
// results meet in LDS at the end.  For calls whose work-groups do not fill
// the chip, where a block's own tiles are what takes the time.
template <bool BF, int HD, int GR>
__global__ __launch_bounds__(64 * kWaves * GR, HD == 256 ? 1 : HD == 128 || GR == 2 ? 2 : 3) void attend_chunk_kernel(PagePool pp, ChunkArgs a) {
  constexpr int kT = HD == 256 ? 32 : 64;   // positions of a tile
  constexpr int RT = kT / 32, G = kT / 16;  // matrix rows of 32 positions; groups of 16, which lie on one page
  constexpr int KS = HD / 16, DT = HD / 32;
  constexpr int CPR = HD / 8;               // 16-byte pieces of a position
  constexpr int RW = kT / kWaves;           // positions that a wave brings: on one page
  constexpr int NJ = RW * CPR / 64;
  constexpr int RJ = 64 / CPR;              // positions of one load of the wave
  constexpr int kRow = HD * 2;
  constexpr int kSwz = CPR < 16 ? 7 : 15;
  // a transposing load of half a wave takes 64 bytes of four positions: all 64 banks once
  auto value_swizzle = [](int r) { return HD == 64 ? 2 * (r & 2) : 4 * (r & 3); };
  __shared__ __align__(16) char all_keys[GR][2][kT * kRow];
  __shared__ __align__(16) char all_values[GR][2][kT * kRow];
  __shared__ int odd[kWaves * GR];  // whether a wave has results that are infinite or no number
  const int group = a.heads / a.kv_heads, g = blockIdx.x % a.kv_heads;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave % kWaves, gr = wave / kWaves;
  const int lane = tid & 63, r32 = lane & 31, hf = lane >> 5;
  const LaneX lx = lane_x_init();
  auto& Ks = all_keys[gr];
  auto& Vs = all_values[gr];
  Block blk;
  if (!find_block(a, pp, blockIdx.x / a.kv_heads, group, lx, blk)) return;
  const int split = blockIdx.y;
  const int row = __builtin_amdgcn_readfirstlane(blk.row), count = __builtin_amdgcn_readfirstlane(blk.count), columns = count * group;
  const int b0 = __builtin_amdgcn_readfirstlane(blk.b) * kCols;
  const int most = pp.cols << pp.shift, len = __builtin_amdgcn_readfirstlane(end_of(pp.lengths, pp.over, most, row));
  const int cw = b0 + 32 * w, c = cw + r32;
  const bool column = c < columns;
  const int t = column ? c / group : count - 1;
  const int h = g * group + (column ? c % group : 0);
  const Span s = span_of(len - (count - t), a.window, a.sinks, most);  // last may be negative: sees nothing
  // the spans of the first and the last token of the wave and of the work-group
  auto span_at = [&](int col) {
    const int cc = __builtin_amdgcn_readfirstlane(col < columns ? col : columns - 1);
    return span_of(len - (count - cc / group), a.window, a.sinks, most);
  };
  const Span s0 = span_at(cw), s1 = span_at(cw + 31);  // a wave without columns has the last token's
  const Span g0 = span_at(b0), g1 = span_at(b0 + kCols - 1);
  TileList<kT> tiles(Span{g0.low, g1.last, g0.sinks});
  tiles.sink = __builtin_amdgcn_readfirstlane(tiles.sink), tiles.low = __builtin_amdgcn_readfirstlane(tiles.low);
  tiles.count = __builtin_amdgcn_readfirstlane(tiles.count);
  const int last_w = s1.last, low_w = s0.low, sinks_w = s0.sinks;
  // this split's share of the tiles
  const int u0 = (int)((int64_t)split * tiles.count / a.splits), n = (int)((int64_t)(split + 1) * tiles.count / a.splits);
  uint4 q[KS];
  const uint16_t* qp = a.q + (int64_t)(blk.first + t) * a.q_token + h * a.q_head;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = flipped(*reinterpret_cast<const uint4*>(qp + 16 * ks + 8 * hf), a.flip);
  const int32_t* trow = pp.table + row * pp.table_ld;

  // lane i < G: the table's entry for positions 16 i .. of the tile at p0
  const int lane_at = 16 * (lane < G ? lane : 0);
  auto entry = [&](int p0) {
    const int col = (p0 + lane_at) >> pp.shift;
    return col < pp.cols ? trow[col] : -1;
  };
  // which groups of 16 positions have a page (bits), and the page of this wave's
  auto valid = [&](int e) { return (unsigned)__ballot(lane < G && e >= 0 && e < pp.pages); };
  constexpr unsigned kAll = (1u << G) - 1;
  const int gw = w * RW / 16, mask = (1 << pp.shift) - 1;
  const int rl = lane / CPR, piece = lane % CPR;  // this lane's position of a load and its piece of it
  const unsigned k_lds = __builtin_amdgcn_readfirstlane(lds_address(Ks[0]) + w * RW * kRow);
  const unsigned v_lds = __builtin_amdgcn_readfirstlane(lds_address(Vs[0]) + w * RW * kRow);
  // Pieces lie swizzled in LDS (below), so a lane brings the piece that belongs at its place.
  unsigned ko[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = w * RW + j * RJ + rl;
    ko[j] = 2u * ((r & 15) * pp.k_pos + 8 * (piece ^ (r & kSwz)));
  }
  unsigned vo[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int r = w * RW + j * RJ + rl;
    vo[j] = 2u * ((r & 15) * pp.v_pos + 8 * (piece ^ value_swizzle(r)));
  }
  // the head's first page; bytes from page to page and from position to position
  const char* const k_head = reinterpret_cast<const char*>(pp.k + g * pp.k_head);
  const char* const v_head = reinterpret_cast<const char*>(pp.v + g * pp.v_head);
  const unsigned k_page = 2u * (unsigned)pp.k_page, v_page = 2u * (unsigned)pp.v_page;
  const unsigned k_pos = 2u * pp.k_pos, v_pos = 2u * pp.v_pos;
  // this wave's positions of the tile at p0
  auto fetch = [&](int p0, int buf, int e, unsigned ok) {
    const unsigned id = ok >> gw & 1 ? __builtin_amdgcn_readlane(e, gw) : 0;
    const unsigned at = (p0 + 16 * gw) & mask;
    load_rows(k_head + ((uint64_t)id * k_page + at * k_pos), ko, k_lds + buf * (kT * kRow));
    load_rows(v_head + ((uint64_t)id * v_page + at * v_pos), vo, v_lds + buf * (kT * kRow));
  };
  // What lies in a place that the row has not filled may be no number, and 0
  // times it would be none either: zeros there, by the wave that brought it.
  auto clear = [&](int p0, int buf, unsigned ok) {
    const int fill = ok >> gw & 1 ? len - (p0 + w * RW) : 0;
    if (fill < RW) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r = j * RJ + rl;
        if (r >= fill) *reinterpret_cast<uint4*>(Vs[buf] + (w * RW + r) * kRow + 16 * piece) = make_uint4(0, 0, 0, 0);
      }
    }
  };

  const int i16 = lane & 15;
  const unsigned k_at = r32 * kRow + 16 * (hf ^ (r32 & kSwz));
  const unsigned v_at = (4 * hf + (i16 >> 2)) * kRow + 16 * ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ value_swizzle(i16 >> 2)) + 8 * (i16 & 1);
  // In a tile that not every column sees all of, a value that is infinite or
  // no number must not meet the columns that do not see it, whose weight of 0
  // would make it NaN.  Where results are not finite the tiles are gone over
  // again (in a loop of its own: looking in the first one took 2 to 7 %), the
  // wave that brings such a value puts a zero in its place, and at the end
  // they are brought to the columns that see them.
  auto partial = [&](int p0) {
    return p0 + kT - 1 > g0.last || (p0 < g1.low && p0 + kT - 1 >= g0.sinks);
  };
  auto take_out = [&](int p0, int buf) {
    if (!partial(p0)) return;
    char* v = Vs[buf] + w * RW * kRow + 16 * lane;
    uint4 x[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) x[j] = *reinterpret_cast<const uint4*>(v + 1024 * j);
    // the least of what the exponents lack of all bits set: of the low elements and of the high ones
    u16x2 least = {0xFFFF, 0xFFFF};
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint32_t words[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, ~words[i] & exponents<BF>()));
    }
    if (!__any(least[0] == 0 || least[1] == 0)) return;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      *reinterpret_cast<uint4*>(v + 1024 * j) =
          make_uint4(Parted<BF>(x[j].x).finite, Parted<BF>(x[j].y).finite, Parted<BF>(x[j].z).finite, Parted<BF>(x[j].w).finite);
  };

  f32x16 o[DT];
  float top, sum;
  // One pass over the tiles; CLEAN: with values taken out.
  auto sweep = [&](auto clean_values) {
    constexpr bool CLEAN = decltype(clean_values)::value;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    top = -INFINITY, sum = 0.f;
    unsigned ok = 0;
    int e_next = 0, p0 = 0, p1 = 0, p2 = 0;  // the tile at hand, the next one (the last again), the one after it
    float back = BF ? 0.f : 7.f;             // what the scaled scores get added: the lift less the base of the weights
    bool far = false;                        // whether a base times scale could leave the range of fp32
    if (u0 < n) {
      const int first = u0 + gr < n ? u0 + gr : u0;
      p0 = kT * tiles.at(first), p1 = kT * tiles.at(first + GR < n ? first + GR : first);
      const int e = entry(p0);
      ok = valid(e);
      fetch(p0, 0, e, ok);
      e_next = entry(p1);
      wait_loads<0>();
      clear(p0, 0, ok);
      if (CLEAN) take_out(p0, 0);
    }
    __syncthreads();
    int buf = 0;
    for (int u = u0 + gr; u - gr < n; u += GR, buf ^= 1) {
      const unsigned ok_next = valid(e_next);
      fetch(p1, buf ^ 1, e_next, ok_next);
      p2 = u + 2 * GR < n ? kT * tiles.at(u + 2 * GR) : p1;
      e_next = entry(p2);
      if ((GR == 1 || u < n) && cw < columns && p0 <= last_w && (p0 + kT - 1 >= low_w || p0 < sinks_w)) {
        unsigned ka = k_at, va = v_at;
        asm volatile("" : "+v"(ka), "+v"(va));  // the addresses made of these are not kept over the loop
        f32x16 st[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[r][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint4 kf = *reinterpret_cast<const uint4*>(Ks[buf] + 32 * r * kRow + (ka ^ 32 * ks));
            st[r] = mma_32x32x16<BF>(kf, q[ks], st[r]);
          }
        const bool all = ok == kAll && p0 + kT - 1 <= s0.last && (p0 >= s1.low || p0 + kT - 1 < s0.sinks);
        if (!all) {
          // the span from this lane's first position on
          const int at = p0 + 4 * hf, hi = s.last - at, lo = s.low - at, sk = s.sinks - at;
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int p = 32 * r + 8 * (i / 4) + i % 4;
              const bool see = p <= (ok >> (2 * r + i / 8) & 1 ? hi : -1) && (p >= lo || p < sk);
              st[r][i] = see ? st[r][i] : -INFINITY;
            }
        }
        float mx = st[0][0];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[r][i]);
        mx = fmaxf(mx, lane_xor<32>(mx, lx));
        // the base of the weights follows the maximum only where it has fallen 2^8 behind
        if (__any((mx - top) * a.scale > 8.f)) {
          const float up = fmaxf(mx, top), f = up == -INFINITY ? 1.f : weight(top - up, a.scale);
          top = up;
          sum *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= f;
          const float base = top == -INFINITY ? 0.f : top;
          back = BF ? -base * a.scale : __builtin_fmaf(-base, a.scale, 7.f);
          far = __any(fabsf(base) > 1e36f);
        }
        float plus = back;
        if (far) {
          // the difference first
          const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 16; ++i) st[r][i] -= base;
          plus = BF ? 0.f : 7.f;
        }
        uint4 pb[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          float part = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            st[r][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r][i], a.scale, plus));
            part += st[r][i];
          }
          sum += part;
#pragma unroll
          for (int x = 0; x < 2; ++x)
            pb[r][x] = make_uint4(pack16<BF>(st[r][8 * x], st[r][8 * x + 1]), pack16<BF>(st[r][8 * x + 2], st[r][8 * x + 3]),
                                  pack16<BF>(st[r][8 * x + 4], st[r][8 * x + 5]), pack16<BF>(st[r][8 * x + 6], st[r][8 * x + 7]));
        }
        // positions 32 r + 16 x + 4 hf + {0 .. 3, 8 .. 11} are this lane's operand of a step
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const char* at = Vs[buf] + (32 * r + 16 * x) * kRow + (va ^ 64 * d);
              const uint2 lo = read_transposed(at), hi = read_transposed(at + 8 * kRow);
              o[d] = mma_32x32x16<BF>(make_uint4(lo.x, lo.y, hi.x, hi.y), pb[r][x], o[d]);
            }
      }
      wait_loads<0>();
      clear(p1, buf ^ 1, ok_next);
      if (CLEAN) take_out(p1, buf ^ 1);
      __syncthreads();
      p0 = p1, p1 = p2, ok = ok_next;
    }
  };
  sweep(std::false_type());
  // infinite or no number?
  float zero = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(o[d][i], 0.f, zero);
  if (lane == 0) odd[wave] = 0;
  if (zero != 0.f) odd[wave] = 1;
  __syncthreads();
  int some = odd[0];
#pragma unroll
  for (int i = 1; i < kWaves * GR; ++i) some |= odd[i];
  const bool again = __builtin_amdgcn_readfirstlane(some);
  if (again) sweep(std::true_type());
  if constexpr (GR == 2) {
    // a wave's sums lie register by register, its lanes side by side
    float* sums = reinterpret_cast<float*>(all_keys) + w * (DT * 16 * 64) + lane;
    float* tops = reinterpret_cast<float*>(all_values) + w * 128 + lane;
    static_assert(sizeof(all_keys) >= kWaves * DT * 16 * 64 * sizeof(float), "");
    if (gr == 1) {
      tops[0] = top, tops[64] = sum;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(16 * d + i) * 64] = o[d][i];
    }
    __syncthreads();
    if (gr == 0) {
      const float up = fmaxf(top, tops[0]), base = up == -INFINITY ? 0.f : up;
      const float f0 = weight(top - base, a.scale), f1 = weight(tops[0] - base, a.scale);
      top = up, sum = f0 * sum + f1 * tops[64];
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = f0 * o[d][i] + f1 * sums[(16 * d + i) * 64];
    }
  }
  const bool live = column && gr == 0;
  const float l = sum + lane_xor<32>(sum, lx);
  // element i of o[d] is dimension 32 d + 2 (i & ~3) + 4 hf + i % 4
  float* part = a.part + (((int64_t)(blk.first + t) * a.heads + h) * a.splits + split) * part_floats(HD) + kPartHead + 4 * hf;
  uint16_t* out = a.out + (int64_t)(blk.first + t) * a.out_token + (int64_t)h * HD + 4 * hf;
  if (live && a.splits > 1) {
    if (hf == 0) part[-kPartHead] = top, part[1 - kPartHead] = l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4*>(part + 32 * d + 2 * i) = f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
  } else if (live) {
    const float rcp = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<uint2*>(out + 32 * d + 2 * i) =
            make_uint2(pack16<BF>(o[d][i] * rcp, o[d][i + 1] * rcp), pack16<BF>(o[d][i + 2] * rcp, o[d][i + 3] * rcp));
  }
  if (!again) return;
  // Ones at the infinite values (no number counts as +inf and -inf) times
  // ones at the positions that a column sees say what its sums get.
  f32x16 up[DT], down[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) up[d][i] = down[d][i] = 0.f;
  for (int u = u0; u < n; ++u) {
    const int p0 = kT * tiles.at(u);
    if (!partial(p0)) continue;
    __syncthreads();
    const int e = entry(p0);
    fetch(p0, 0, e, valid(e));
    wait_loads<0>();
    clear(p0, 0, valid(e));
    __syncthreads();
    const int at = p0 + 4 * hf, hi = s.last - at, lo = s.low - at, sk = s.sinks - at;
    constexpr uint32_t one = BF ? 0x3F80u : 0x3C00u;
#pragma unroll 1
    for (int r = 0; r < 2 * RT; ++r) {
      uint32_t sees[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = 16 * r + 8 * (i / 4) + i % 4;
        sees[i / 2] |= p <= hi && (p >= lo || p < sk) ? one << 16 * (i % 2) : 0u;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const char* v = Vs[0] + 16 * r * kRow + (v_at ^ 64 * d);
        const uint2 x = read_transposed(v), y = read_transposed(v + 8 * kRow);
        const Parted<BF> x0(x.x), x1(x.y), y0(y.x), y1(y.y);
        const uint4 b = make_uint4(sees[0], sees[1], sees[2], sees[3]);
        up[d] = mma_32x32x16<BF>(make_uint4(x0.plus, x1.plus, y0.plus, y1.plus), b, up[d]);
        down[d] = mma_32x32x16<BF>(make_uint4(x0.minus, x1.minus, y0.minus, y1.minus), b, down[d]);
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (!(up[d][i] > 0.f || down[d][i] > 0.f)) continue;
      const int at = 32 * d + 2 * (i & ~3) + i % 4;
      const float gets = (up[d][i] > 0.f ? INFINITY : 0.f) - (down[d][i] > 0.f ? INFINITY : 0.f);
      if (a.splits > 1) part[at] += gets;
      else out[at] = (uint16_t)pack16<BF>(from16<BF>(out[at]) + gets, 0.f);
    }
}

int64_t chunk_blocks(int64_t tokens, int64_t rows, int heads, int kv_heads) {
  return (tokens * (heads / kv_heads) + kCols - 1) / kCols + rows;
}

// The blocks that there are if the rows' tokens fill theirs and every row has some.
int64_t likely_blocks(int64_t tokens, int64_t rows, int heads, int kv_heads) {
  const int64_t full = (tokens * (heads / kv_heads) + kCols - 1) / kCols, some = rows < tokens ? rows : tokens;
  return full > some ? full : some;
}

// Into how many shares the tiles of a block are cut.  A share is a work-group;
// a CU has room for two, so cutting pays where the blocks' heads are fewer
// than half the chip's CUs, and shares of less than 8 tiles do not repay the
// second launch and the parts that it joins (16 tokens of 8 kv heads behind
// 6000 positions: 136 us whole, 26 us in shares; a prompt of 512 with 64 heads:
// 21 us whole, 36 us in two, and 18 whole since it runs in eight waves).  Blocks that are not full leave few parts to
// join, so that twice the shares pay (16 rows of up to 8 tokens behind up to
// 4000 positions: 38.5 us instead of 45; full ones, 100 tokens behind 6000
// positions: 59 us instead of 41).
int chunk_splits(int64_t tokens, int64_t rows, int heads, int kv_heads, int64_t cols, int page, int window, int sinks) {
  const int64_t blocks = likely_blocks(tokens, rows, heads, kv_heads), wgs = blocks * kv_heads;
  const int64_t slots = tokens * (heads / kv_heads) * 4 <= blocks * kCols * 3 ? 512 : 256;
  const int64_t seen = seen_positions(cols * page, window, sinks, (tokens - 1 < kCols ? tokens - 1 : kCols));
  const int64_t most = seen / 512, n = slots / wgs;
  return (int)(n < 2 || most < 2 ? 1 : n < most ? n : most);
}

template <bool BF, int HD>
int launch_chunk(const PagePool& pp, const ChunkArgs& a, hipStream_t stream) {
  const int64_t blocks = chunk_blocks(a.tokens, a.rows, a.heads, a.kv_heads);
  const dim3 grid((unsigned)(blocks * a.kv_heads), (unsigned)a.splits);
  if constexpr (HD < 256) {  // whose registers leave no room for a second wave on a SIMD
    // One work-group for a CU at most, with tiles for both halves: eight waves
    // (a prompt of 512 with 64 heads: 19.2 us against 20.7, 300 tokens behind
    // 6000 positions 105 against 146; with one or two tiles the second half
    // only costs, 10.9 against 9.1 us for a prompt of 64; 64 rows of up to 2
    // tokens behind up to 1000 positions, 8 kv heads: 34 us, with eight waves 59).
    const int64_t seen = seen_positions((int64_t)pp.cols << pp.shift, a.window, a.sinks, a.tokens - 1 < kCols ? a.tokens - 1 : kCols);
    if (likely_blocks(a.tokens, a.rows, a.heads, a.kv_heads) * a.kv_heads * a.splits <= 256 && seen / a.splits >= 256) {
      hipLaunchKernelGGL((attend_chunk_kernel<BF, HD, 2>), grid, dim3(128 * kWaves), 0, stream, pp, a);
      QS_LAUNCHED("attend_chunk_kernel");
      if (a.splits > 1) return join_parts(a.part, a.splits, nullptr, a.tokens, a.heads, HD, BF, a.scale, a.out, a.out_token, stream);
      return QS_OK;
    }
  }
  hipLaunchKernelGGL((attend_chunk_kernel<BF, HD, 1>), grid, dim3(64 * kWaves), 0, stream, pp, a);
  QS_LAUNCHED("attend_chunk_kernel");
  if (a.splits > 1) return join_parts(a.part, a.splits, nullptr, a.tokens, a.heads, HD, BF, a.scale, a.out, a.out_token, stream);
  return QS_OK;
}

}  // namespace

int page_pool_checks(const char* fn, const qs_page_pool* p, int dtype, int64_t rows, int heads, int kv_heads,
                     int head_dim, float scale, int window, int sinks, const int32_t* over, PagePool& out) {
  QS_REQUIRE(std::isfinite(scale * kLog2E) && scale != 0.f, "%s: scale %g", fn, (double)scale);
  QS_SUPPORTED(dtype == QS_DTYPE_BF16 || dtype == QS_DTYPE_F16, "%s: dtype %d (bf16 and fp16 only)", fn, dtype);
  QS_SUPPORTED(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %d (64, 128 or 256)", fn, head_dim);
  QS_REQUIRE(p && p->k && p->v && p->table && p->lengths, "%s: null pointer", fn);
  QS_REQUIRE(rows >= 1 && rows <= 65535 && kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads <= 4096,
             "%s: rows %lld, heads %d / %d", fn, (long long)rows, heads, kv_heads);
  QS_SUPPORTED(p->page >= 16 && p->page <= 4096 && (p->page & (p->page - 1)) == 0,
               "%s: pages of %d positions (a power of two from 16 to 4096)", fn, p->page);
  QS_REQUIRE(p->pages >= 1 && p->pages <= INT32_MAX && p->cols >= 1 && p->table_ld >= p->cols &&
                 p->cols * p->page <= INT32_MAX - 4096,
             "%s: %lld pages, table of %lld columns (stride %lld)", fn, (long long)p->pages, (long long)p->cols,
             (long long)p->table_ld);
  QS_REQUIRE(window >= 0 && sinks >= 0 && (sinks == 0 || window > 0), "%s: window %d, sinks %d", fn, window, sinks);
  const int64_t st[6] = {p->k_page, p->k_head, p->k_pos, p->v_page, p->v_head, p->v_pos};
  for (int64_t x : st) QS_REQUIRE(x >= 0 && x % 8 == 0, "%s: pool strides must be multiples of 8 elements, got %lld", fn, (long long)x);
  QS_SUPPORTED(p->k_page < ((int64_t)1 << 31) && p->v_page < ((int64_t)1 << 31) && p->page * p->k_pos <= (1 << 30) &&
                   p->page * p->v_pos <= (1 << 30),
               "%s: pages %lld and %lld elements apart, positions %lld and %lld (at most 2^31, a page's 2^30)", fn,
               (long long)p->k_page, (long long)p->v_page, (long long)p->k_pos, (long long)p->v_pos);
  QS_REQUIRE(p->k_pos >= head_dim && p->k_pos <= (1 << 24) && p->v_pos >= head_dim && p->v_pos <= (1 << 24),
             "%s: position strides %lld, %lld", fn, (long long)p->k_pos, (long long)p->v_pos);
  QS_REQUIRE(((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15) == 0,
             "%s: the pools must be 16-byte aligned", fn);
  int shift = 0;
  while ((1 << shift) < p->page) ++shift;
  out = PagePool{static_cast<const uint16_t*>(p->k), static_cast<const uint16_t*>(p->v), p->k_page, p->k_head, p->v_page,
                 p->v_head, (int)p->k_pos, (int)p->v_pos, (int)p->pages, shift, p->table, p->table_ld, (int)p->cols, p->lengths, over};
  return QS_OK;
}

}  // namespace qs

using namespace qs;

extern "C" size_t qs_attend_chunk_workspace_bytes(int64_t tokens, int64_t rows, int heads, int kv_heads, int head_dim,
                                                  int64_t cols, int page, int window, int sinks) {
  if (tokens < 1 || rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || cols < 1 || page < 1) return 0;
  const int n = chunk_splits(tokens, rows, heads, kv_heads, cols, page, window, sinks);
  return n == 1 ? 0 : (size_t)tokens * heads * n * part_floats(head_dim) * sizeof(float);
}

extern "C" int qs_attend_chunk(const void* q, int dtype, int64_t tokens, int64_t rows, int heads, int kv_heads,
                               int head_dim, int64_t q_token, int64_t q_head, const int32_t* starts,
                               const qs_page_pool* pool, float scale, int window, int sinks, void* out,
                               int64_t out_token, qs_stream_t stream) {
  return qs_attend_chunk_over(q, dtype, tokens, rows, heads, kv_heads, head_dim, q_token, q_head, starts, pool, nullptr,
                              scale, window, sinks, out, out_token, nullptr, 0, stream);
}

extern "C" int qs_attend_chunk_ws(const void* q, int dtype, int64_t tokens, int64_t rows, int heads, int kv_heads,
                                  int head_dim, int64_t q_token, int64_t q_head, const int32_t* starts,
                                  const qs_page_pool* pool, float scale, int window, int sinks, void* out,
                                  int64_t out_token, void* workspace, size_t workspace_bytes, qs_stream_t stream) {
  return qs_attend_chunk_over(q, dtype, tokens, rows, heads, kv_heads, head_dim, q_token, q_head, starts, pool, nullptr,
                              scale, window, sinks, out, out_token, workspace, workspace_bytes, stream);
}

extern "C" int qs_attend_chunk_over(const void* q, int dtype, int64_t tokens, int64_t rows, int heads, int kv_heads,
                                    int head_dim, int64_t q_token, int64_t q_head, const int32_t* starts,
                                    const qs_page_pool* pool, const int32_t* over, float scale, int window, int sinks,
                                    void* out, int64_t out_token, void* workspace, size_t workspace_bytes,
                                    qs_stream_t stream) {
  if (tokens == 0) return QS_OK;
  QS_REQUIRE(rows != 0, "qs_attend_chunk: %lld tokens of no row", (long long)tokens);
  PagePool pp;
  if (const int rc = page_pool_checks("qs_attend_chunk", pool, dtype, rows, heads, kv_heads, head_dim, scale, window, sinks, over, pp)) return rc;
  QS_REQUIRE(q && out && starts, "qs_attend_chunk: null pointer");
  QS_REQUIRE(tokens >= 1 && tokens * heads <= INT32_MAX, "qs_attend_chunk: %lld tokens", (long long)tokens);
  QS_REQUIRE(q_head >= head_dim && q_head % 8 == 0 && q_token >= 0 && q_token % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
             "qs_attend_chunk: query rows must be 16-byte aligned (strides %lld, %lld)", (long long)q_token, (long long)q_head);
  QS_REQUIRE(out_token >= (int64_t)heads * head_dim && out_token % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
             "qs_attend_chunk: output rows of %lld elements must be 16-byte aligned", (long long)out_token);
  const size_t need = qs_attend_chunk_workspace_bytes(tokens, rows, heads, kv_heads, head_dim, pool->cols, pool->page, window, sinks);
  QS_REQUIRE(!workspace || (workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
             "qs_attend_chunk: workspace of %zu bytes (16-byte aligned), %zu needed", workspace_bytes, need);
  const int splits = workspace && need ? chunk_splits(tokens, rows, heads, kv_heads, pool->cols, pool->page, window, sinks) : 1;
  ChunkArgs a{static_cast<const uint16_t*>(q), q_token, q_head, static_cast<uint16_t*>(out), out_token, starts, (int)tokens,
              (int)rows, heads, kv_heads, window, sinks, static_cast<float*>(workspace), splits, fabsf(scale) * kLog2E, scale < 0 ? 0x80008000u : 0u};
  const bool bf = dtype == QS_DTYPE_BF16;
  const hipStream_t st = as_stream(stream);
  if (head_dim == 64) return bf ? launch_chunk<true, 64>(pp, a, st) : launch_chunk<false, 64>(pp, a, st);
  if (head_dim == 128) return bf ? launch_chunk<true, 128>(pp, a, st) : launch_chunk<false, 128>(pp, a, st);
  return bf ? launch_chunk<true, 256>(pp, a, st) : launch_chunk<false, 256>(pp, a, st);
}
