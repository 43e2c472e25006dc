// Low-rank adapters of many requests beside shared projections
// (qs_adapters_add): for up to four linears g that read the same rows,
//
//   out_g[t] = y_g[t] + scale_g[a] up_g[a] (down_g[a] x[t]),   a = which[t]
//
// with rows that have no adapter left as they are.  Two launches: the inner
// products with `down` (K = n is long, so it is split over work-groups, each
// split leaving its fp32 sums), then the ones with `up` (K = rank), in whose
// first step the splits are added.  The rows of `down` of all linears count as
// one matrix, so that x is read once for 128 of them.
//
// Both are bound by memory: single tokens by the weights of the adapters that
// they name, prompts by x, y and out.  Measured: 48 tokens that name 21 adapters of
// rank 64, 5120 inputs to two linears of 25600, 10 and 31 us for 28 and 147 MB (2.9
// and 4.7 TB/s; a large copy reaches 5.06); 10313 tokens of 3 prompts, 25600 inputs
// to 5120 at rank 64, 95 and 54 us for 747 MB (5.0 TB/s); 4260 of 6, 3584 inputs to
// 3584 + 512 + 512 at rank 24, 16 and 24 us for 113 MB (2.8 TB/s: short loops behind
// each work-group's start); one token, 4096 inputs to 4096 + 1024 + 1024, 4 and 6 us.
//
// Tokens are taken 64 at a time.  In each 64 those of one adapter form a group
// (found by ballots: prompts come in runs, single tokens in any order), which
// reads that adapter once and is a block of matrix columns: 16x16x32 MFMA with
// the weights as rows and the tokens as columns, so that a lane's results lie
// together in a token's row.
//
// The inner products go on as two 16-bit numbers, the second the remainder of
// the first, after an exact scaling of each token's by a power of two: what is
// dropped lies 2^-16 (bf16) or 2^-22 (fp16) below the largest, and products
// beyond fp16's range work.  All sums are fp32; the output is rounded once.
#include "qs_attend_dev.h"
#include "qs_overlap.h"

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;     // tokens at a time
constexpr int kMaxRank = 128;
constexpr int64_t kMaxTokens = 1 << 19;
constexpr int kColumns = 256;  // output columns of a work-group of single tokens at a time, 64 a wave

struct Linear {
  const uint16_t *down, *up;
  const float* scale;
  const uint16_t* y;
  uint16_t* out;
  int64_t down_adapter, down_row, up_adapter, up_row, ldy, ldo, m;
  int rank, offset;  // offset: of its ranks among those of all linears
  int first;         // its first work-group column of the second launch
};

struct AdapterArgs {
  const uint16_t* x;
  int64_t ldx, tokens, n;
  const int32_t* which;
  int adapters, count, ranks;  // ranks: of all linears together
  int tiles, runs, splits, steps;  // runs: work-groups for all ranks; steps of 256 inputs of a split
  int slots, span;             // work-groups that share a tile's groups, a power of two; columns of one of the second launch
  float* part;                 // [splits][tokens][ranks]
  Linear linear[QS_MAX_GROUP];
};

// The tokens of a group, by column: lane c has the place in the tile of the c-th.
struct Group {
  int adapter, size, inverse;
};

// Calls use(Group) for the groups of a tile that fall to this slot.  `none`:
// tokens without an adapter form a group too.  Every wave of a work-group runs
// through the same groups.
template <typename F>
__device__ __forceinline__ void each_group(const AdapterArgs& a, int64_t t0, int slot, bool none, F use) {
  const int lane = threadIdx.x & 63;
  int id = -2;
  if (t0 + lane < a.tokens) {
    id = a.which[t0 + lane];
    if (id < 0 || id >= a.adapters) id = -1;
  }
  uint64_t todo = __ballot(id >= (none ? -1 : 0));
  for (int nth = 0; todo; ++nth) {
    const int adapter = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == adapter);
    todo &= ~mine;
    if ((nth & (a.slots - 1)) != slot) continue;
    // a permutation of the lanes: the group's first, in order
    const uint64_t below = (1ull << lane) - 1;
    const int size = __popcll(mine);
    const int to = mine >> lane & 1 ? __popcll(mine & below) : size + __popcll(~mine & below);
    use(Group{adapter, size, __builtin_amdgcn_ds_permute(to * 4, lane)});
  }
}

// Place in the tile of a group's column c, the last one's beyond them.
__device__ __forceinline__ int place_in_tile(const Group& g, int c) {
  c = c < g.size ? c : g.size - 1;
  return __builtin_amdgcn_ds_bpermute(c * 4, g.inverse);
}

// Row `rank` of an adapter's `down`, those of all linears one after the other;
// rows beyond repeat the last.
__device__ __forceinline__ const char* down_row(const AdapterArgs& a, int adapter, int rank) {
  rank = rank < a.ranks ? rank : a.ranks - 1;
  const char* row = nullptr;
#pragma unroll
  for (int g = 0; g < QS_MAX_GROUP; ++g)
    if (g < a.count && rank >= a.linear[g].offset) {
      const Linear& l = a.linear[g];
      row = reinterpret_cast<const char*>(l.down + adapter * l.down_adapter) + (uint64_t)(uint32_t)(rank - l.offset) * (2u * (uint32_t)l.down_row);
    }
  return row;
}

// One group of the first launch, of up to 16 tokens: RB blocks of 16 ranks from
// rank0 on, the inputs shared out over the waves.
template <bool BF, int RB>
__device__ __forceinline__ void down_group(const AdapterArgs& a, const Group& g, int64_t t0, int split, int rank0, f32x4 (*sums)[64]) {
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  const char *x = reinterpret_cast<const char*>(a.x + (t0 + place_in_tile(g, r)) * a.ldx + 8 * q), *down[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) down[i] = down_row(a, g.adapter, rank0 + 16 * i + r) + 16 * q;
  f32x4 acc[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int n = (int)a.n, k0 = split * a.steps * 256, k1 = k0 + a.steps * 256 < n ? k0 + a.steps * 256 : n;
  // 64 inputs at a time, 32 for each of two products
  uint4 xv[2], av[RB][2];
  auto multiply = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < RB; ++i) acc[i] = mma_16x16x32<BF>(av[i][j], xv[j], acc[i]);
  };
  int k = k0 + 64 * w;
  for (; k + 64 <= k1; k += 256) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      xv[j] = *reinterpret_cast<const uint4*>(x + 2 * (int64_t)k + 64 * j);
#pragma unroll
      for (int i = 0; i < RB; ++i) av[i][j] = *reinterpret_cast<const uint4*>(down[i] + 2 * (int64_t)k + 64 * j);
    }
    multiply();
  }
  if (k < k1) {
    // fewer than 64 are left: zeros behind them
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool in = k + 32 * j + 8 * q < k1;
      xv[j] = in ? *reinterpret_cast<const uint4*>(x + 2 * (int64_t)k + 64 * j) : uint4{};
#pragma unroll
      for (int i = 0; i < RB; ++i) av[i][j] = in ? *reinterpret_cast<const uint4*>(down[i] + 2 * (int64_t)k + 64 * j) : uint4{};
    }
    multiply();
  }
  // the waves' sums together, a block of ranks at a time
  float* part = a.part + ((int64_t)split * a.tokens + t0) * a.ranks;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    sums[w][lane] = acc[i];
    __syncthreads();
    if (w == 0) {
      const int rank = rank0 + 16 * i + 4 * q;
      const f32x4 s = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
      const int place = place_in_tile(g, r);  // an exchange of all lanes
      if (r < g.size && rank < a.ranks) *reinterpret_cast<f32x4*>(part + place * a.ranks + rank) = s;
    }
    __syncthreads();
  }
}

// The same for more than 16 tokens: 64 tokens and 16 RB ranks by 64 inputs at a
// time go straight to LDS, kAhead such stages ahead of their use, and each wave
// multiplies its 16 tokens.  A row of a stage is eight pieces of 16 bytes, of
// which piece p lies at place p ^ (row & 7), so that a wave's operands (one
// piece of each of 16 rows) come from all banks.
constexpr int kStageRow = 128;
template <int RB>
constexpr int kAhead = RB > 4 ? 2 : 3;
template <int RB>
constexpr int stage_bytes() {
  return (kTile + 16 * RB) * kStageRow;
}

template <bool BF, int RB>
__device__ __forceinline__ void down_tile(const AdapterArgs& a, const Group& g, int64_t t0, int split, int rank0, char* stages) {
  constexpr int NX = kTile / 32, NW = RB / 2, NL = NX + NW, A = kAhead<RB>;  // loads of a wave in a stage, of 8 rows each
  static_assert(RB % 2 == 0, "every wave brings as many rows");
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  const int n = (int)a.n, k0 = split * a.steps * 256, k1 = k0 + a.steps * 256 < n ? k0 + a.steps * 256 : n;
  const int count = (k1 - k0 + 63) / 64, left = k1 - k0 - 64 * (count - 1);  // stages, inputs of the last
  const int row8 = lane >> 3;  // of a load; every load begins at a multiple of 8 rows
  const unsigned piece = 16 * ((lane & 7) ^ row8);
  unsigned x_row[NX], w_row[NW], x_at[NX], w_at[NW];
  const char* down[NW];  // a load's rows are of one linear: ranks are multiples of 8
#pragma unroll
  for (int j = 0; j < NX; ++j) x_row[j] = 2u * (uint32_t)place_in_tile(g, 8 * (NX * w + j) + row8) * (uint32_t)a.ldx, x_at[j] = x_row[j] + piece;
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    int rank = rank0 + 8 * (NW * w + j), gi = 0;  // the sums of rows beyond go nowhere
    rank = rank < a.ranks ? rank : a.ranks - 8;
    while (gi + 1 < a.count && rank >= a.linear[gi + 1].offset) ++gi;
    const Linear& l = a.linear[gi];
    down[j] = reinterpret_cast<const char*>(l.down + g.adapter * l.down_adapter + (rank - l.offset) * l.down_row + k0);
    w_row[j] = 2u * (uint32_t)row8 * (uint32_t)l.down_row, w_at[j] = w_row[j] + piece;
  }
  const char* x = reinterpret_cast<const char*>(a.x + t0 * a.ldx + k0);
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_address(stages));
  auto fetch = [&](int s) {
    const unsigned to = lds + (unsigned)(s % (A + 1)) * stage_bytes<RB>();
    if (s == count - 1 && left < 64) {
      // pieces behind the last input: the last one again, which is not used
      const unsigned end = 2u * (left - 8), p = piece < end ? piece : end;
#pragma unroll
      for (int j = 0; j < NX; ++j) x_at[j] = x_row[j] + p;
#pragma unroll
      for (int j = 0; j < NW; ++j) w_at[j] = w_row[j] + p;
    }
    load_rows(x + 128 * (int64_t)s, x_at, to + w * (NX * 1024));
#pragma unroll
    for (int j = 0; j < NW; ++j) load_to_lds<0>(down[j] + 128 * (int64_t)s, w_at[j], to + kTile * kStageRow + (NW * w + j) * 1024);
  };
  f32x4 acc[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool busy = 16 * w < g.size;
#pragma unroll
  for (int s = 0; s < A; ++s)
    if (s < count) fetch(s);
  for (int s = 0; s < count; ++s) {
    if (s + A <= count) wait_loads<(A - 1) * NL>();
    else wait_loads<0>();
    __syncthreads();
    if (s + A < count) fetch(s + A);
    if (busy) {
      const char* at = stages + (s % (A + 1)) * stage_bytes<RB>();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int p = 16 * ((4 * j + q) ^ (r & 7));
        uint4 xv = *reinterpret_cast<const uint4*>(at + (16 * w + r) * kStageRow + p), av[RB];
#pragma unroll
        for (int i = 0; i < RB; ++i) av[i] = *reinterpret_cast<const uint4*>(at + (kTile + 16 * i + r) * kStageRow + p);
        if (s == count - 1 && left < 64 && 32 * j + 8 * q >= left) {
          xv = uint4{};
#pragma unroll
          for (int i = 0; i < RB; ++i) av[i] = uint4{};
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i] = mma_16x16x32<BF>(av[i], xv, acc[i]);
      }
    }
  }
  const int c = 16 * w + r, place = place_in_tile(g, c);
  float* part = a.part + ((int64_t)split * a.tokens + t0 + place) * a.ranks;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int rank = rank0 + 16 * i + 4 * q;
    if (c < g.size && rank < a.ranks) *reinterpret_cast<f32x4*>(part + rank) = acc[i];
  }
  __syncthreads();  // the next group's stages lie where these did
}

// A work-group: (slot, tile, split, run of 16 RB ranks).  Work-groups go to the
// eight XCDs in turn.  The runs of a tile's split, which read the same x, go to
// one XCD, one after the other (5768 tokens, 5120 inputs, three runs of 128: 74 us
// with the runs on XCDs beside each other, 67 so), and the slot is slowest, so that
// slots without a group do not fall to the same XCDs (14 tiles in 4 slots: 18.3 us
// with the slot fastest, 13.9 so).  One tile has its work-groups in plain order.
template <bool BF, int RB, bool MANY>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterArgs a) {
  constexpr int kSums = 4 * 64 * sizeof(f32x4), kStages = MANY ? (kAhead<RB> + 1) * stage_bytes<RB>() : 0;
  __shared__ __align__(16) char room[kStages > kSums ? kStages : kSums];
  int unit = blockIdx.x / a.runs, run = blockIdx.x % a.runs;
  if (a.tiles > 1) {
    unit = (int)(blockIdx.x / 8) / a.runs * 8 + (int)(blockIdx.x % 8), run = (int)(blockIdx.x / 8) % a.runs;
    if (unit >= a.slots * a.tiles * a.splits) return;
  }
  const int split = unit % a.splits, rank0 = run * (16 * RB);
  const int64_t t0 = (int64_t)(unit / a.splits % a.tiles) * kTile;
  each_group(a, t0, unit / a.splits / a.tiles, false, [&](const Group& g) {
    if constexpr (MANY) {
      if (g.size > 16) return down_tile<BF, RB>(a, g, t0, split, rank0, room);
    }
    down_group<BF, RB>(a, g, t0, split, rank0, reinterpret_cast<f32x4(*)[64]>(room));
  });
}

template <bool BF>
__device__ __forceinline__ float float_of(uint32_t u) {
  if constexpr (BF) return __uint_as_float(u << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}

// Rows of y and out may begin anywhere: 16 bytes from a place that is aligned to
// an element only, which a global access takes on this target.
typedef u32x4 Loose __attribute__((aligned(2)));
__device__ __forceinline__ uint4 get_loose(const char* p) { return __builtin_bit_cast(uint4, (u32x4)*reinterpret_cast<const Loose*>(p)); }
__device__ __forceinline__ void put_loose(char* p, const uint4& v) { *reinterpret_cast<Loose*>(p) = __builtin_bit_cast(u32x4, v); }
// The first n of 8 elements, 0 < n < 8.
__device__ __forceinline__ uint4 get_some(const char* p, int n) {
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) v[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16 * (i & 1);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put_some(char* p, const uint4& x, int n) {
  const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(v[i / 2] >> 16 * (i & 1));
}

// 8 columns of a token: y + scale * d.
template <bool BF>
__device__ __forceinline__ uint4 add_8(uint4 y, const f32x4& d0, const f32x4& d1, float scale) {
  const uint32_t in[4] = {y.x, y.y, y.z, y.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4& d = i < 2 ? d0 : d1;
    o[i] = pack16<BF>(__builtin_fmaf(d[2 * (i & 1)], scale, float_of<BF>(in[i] & 0xFFFF)),
                      __builtin_fmaf(d[2 * (i & 1) + 1], scale, float_of<BF>(in[i] >> 16)));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// An exact power of two that brings a largest size near 1, and its inverse.
// Within 2^64 either way, so that the inverse times an adapter's scale neither
// overflows nor loses bits: inner products of fp16 numbers are (products from
// 2^-48 to 2^32, at most 2^24 of them added), and those of bf16 numbers go on as
// bf16, which has fp32's exponents.
__device__ __forceinline__ float powers(float most, float& inverse) {
  int e = (int)(__float_as_uint(most) >> 23);
  e = e < 127 - 64 ? 127 - 64 : e > 127 + 64 ? 127 + 64 : e;
  inverse = __uint_as_float((uint32_t)e << 23);
  return __uint_as_float((uint32_t)(254 - e) << 23);
}
// Two numbers as 16 bits and the remainder in 16 more; an infinite one has none.
template <bool BF>
__device__ __forceinline__ void two_parts(float f0, float f1, uint32_t& hi, uint32_t& lo) {
  hi = pack16<BF>(f0, f1);
  const float h0 = float_of<BF>(hi & 0xFFFF), h1 = float_of<BF>(hi >> 16);
  lo = pack16<BF>(fabsf(h0) < INFINITY ? f0 - h0 : 0.f, fabsf(h1) < INFINITY ? f1 - h1 : 0.f);
}

// The inner products of up to 16 tokens of a group, summed over the splits, as two
// 16-bit numbers: four ranks a thread, a token's R / 4 threads in one wave.
// Splits on their way together: 9 tokens of rank 112 take 10.8 us with a loop
// that the compiler unrolls by four, 7.0 with eight at a time; 48 tokens of rank 64
// to 2 x 25600 34 and 32, with sixteen 37.  Ranks up to 32 keep the loop: few
// splits of prompts 24 us with it, 29 without.
template <bool BF, int R, int kRow>
__device__ __forceinline__ void inner_products(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, uint4* high,
                                               uint4* low, float* factor) {
  constexpr int T = R == 96 ? 32 : R / 4;  // a power of two
  constexpr int U = T == 32 ? 2 : 1, P = 8 / U;  // tokens of a thread, splits at a time
  const int tid = threadIdx.x;
  if (16 * T < kThreads && tid >= 16 * T) return;  // whole waves: 16 T is a multiple of 64
  const float* base = a.part + t0 * a.ranks + l.offset;
  const int64_t next = a.tokens * a.ranks;
  const int rank = tid % T * 4;
  const float scale = l.scale[g.adapter];
  f32x4 s[U];
  uint32_t from[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    from[i] = (uint32_t)place_in_tile(g, i * (kThreads / T) + tid / T) * (uint32_t)a.ranks + (rank < l.rank ? rank : 0);
    s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if constexpr (R == 32) {
#pragma unroll 4
    for (int p = 0; p < a.splits; ++p) s[0] += *reinterpret_cast<const f32x4*>(base + p * next + from[0]);
  } else {
    for (int p0 = 0; p0 < a.splits; p0 += P) {
      f32x4 v[P][U];  // on their way together
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < U; ++i)
          v[p][i] = p0 + p < a.splits ? *reinterpret_cast<const f32x4*>(base + (p0 + p) * next + from[i]) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < U; ++i) s[i] += v[p][i];
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = i * (kThreads / T) + tid / T;
    if (rank >= l.rank) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float most = fmaxf(fmaxf(fabsf(s[i][0]), fabsf(s[i][1])), fmaxf(fabsf(s[i][2]), fabsf(s[i][3])));
#pragma unroll
    for (int x = 1; x < T; x *= 2) most = fmaxf(most, __shfl_xor(most, x));
    float grow;
    const float shrink = powers(most, grow);
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) two_parts<BF>(s[i][2 * x] * shrink, s[i][2 * x + 1] * shrink, hi[x], lo[x]);
    const int at = (c * kRow + rank) / 4;
    if (R < 4 * T && rank >= R) continue;
    reinterpret_cast<uint2*>(high)[at] = make_uint2(hi[0], hi[1]), reinterpret_cast<uint2*>(low)[at] = make_uint2(lo[0], lo[1]);
    if (rank == 0) factor[c] = grow * scale;
  }
}

// What a lane's part of the products reads and writes of y and out: columns m0
// + 8 q .. + 7 and m0 + 32 + 8 q .. + 7 of a token, so that an access of the
// wave takes 64 bytes together of 16 rows.  left: columns from m0 + 8 q on.
__device__ __forceinline__ void load_y(const char* from, int left, uint4 (&y)[2]) {
  if (left >= 40) {
    y[0] = get_loose(from), y[1] = get_loose(from + 64);
  } else {
    if (left > 0) y[0] = left < 8 ? get_some(from, left) : get_loose(from);
    if (left > 32) y[1] = get_some(from + 64, left - 32);
  }
}
__device__ __forceinline__ void store_out(char* to, int left, const uint4 (&o)[2]) {
  if (left >= 40) {
    put_loose(to, o[0]), put_loose(to + 64, o[1]);
  } else {
    if (left >= 8) put_loose(to, o[0]);
    else if (left > 0) put_some(to, o[0], left);
    if (left > 32) put_some(to + 64, o[1], left - 32);
  }
}
// The column of row r of the j-th of the four products over 64 columns.
__device__ __forceinline__ int column_of(int j, int r) { return 32 * (j >> 1) + 8 * (r >> 2) + 4 * (j & 1) + (r & 3); }

// The second launch for a group of up to 16 tokens: each wave takes 64 columns
// at a time, whose weights go to its registers, the next ones on their way.
template <bool BF, int KB>
__device__ __forceinline__ void up_group(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, int64_t m_begin,
                                         int64_t m_end, char* room) {
  constexpr int R = 32 * KB, kRow = R + 8;  // 16-bit elements of a token's row, 16 bytes more than the products need
  uint4 *high = reinterpret_cast<uint4*>(room), *low = high + 16 * kRow / 8;
  float* factor = reinterpret_cast<float*>(low + 16 * kRow / 8);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  const char* up = reinterpret_cast<const char*>(l.up + g.adapter * l.up_adapter);
  uint32_t w_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w_at[j] = 2u * ((uint32_t)column_of(j, r) * (uint32_t)l.up_row + 8 * q);
  auto weights = [&](int64_t m0, uint4 (&wv)[4][KB]) {
    const char* from = up + 2 * m0 * l.up_row;
    const int last = m0 + 64 <= l.m ? 63 : (int)(l.m - m0) - 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = column_of(j, r) <= last ? w_at[j] : 2u * ((uint32_t)last * (uint32_t)l.up_row + 8 * q);
#pragma unroll
      for (int k = 0; k < KB; ++k)
        wv[j][k] = 32 * k + 8 * q < l.rank ? *reinterpret_cast<const uint4*>(from + at + 64 * k) : uint4{};
    }
  };
  const uint32_t place = place_in_tile(g, r);
  const char* y0 = reinterpret_cast<const char*>(l.y + t0 * l.ldy) + 2u * (place * (uint32_t)l.ldy + 8 * q);
  char* out0 = reinterpret_cast<char*>(l.out + t0 * l.ldo) + 2u * (place * (uint32_t)l.ldo + 8 * q);
  auto left_of = [&](int64_t m0) { return (int)(l.m - m0 < 64 ? l.m - m0 : 64) - 8 * q; };
  uint4 wv[4][KB], y[2];
  int64_t m0 = m_begin + 64 * w;
  if (m0 < m_end) weights(m0, wv), load_y(y0 + 2 * m0, left_of(m0), y);
  __syncthreads();  // the group before is done with the tables
  inner_products<BF, R, kRow>(a, l, g, t0, high, low, factor);
  __syncthreads();
  uint4 h[KB], o[KB];
#pragma unroll
  for (int k = 0; k < KB; ++k) h[k] = high[(r * kRow + 32 * k + 8 * q) / 8], o[k] = low[(r * kRow + 32 * k + 8 * q) / 8];
  const float scale = factor[r];
  for (; m0 < m_end; m0 += kColumns) {
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = mma_16x16x32<BF>(wv[j][k], o[k], mma_16x16x32<BF>(wv[j][k], h[k], acc[j]));
    const uint4 o8[2] = {add_8<BF>(y[0], acc[0], acc[1], scale), add_8<BF>(y[1], acc[2], acc[3], scale)};
    if (m0 + kColumns < m_end) weights(m0 + kColumns, wv), load_y(y0 + 2 * (m0 + kColumns), left_of(m0 + kColumns), y);
    if (r < g.size) store_out(out0 + 2 * m0, left_of(m0), o8);
  }
}

// The same for more tokens: a wave has 16 of them, whose inner products stay in
// its registers as the operand that they are, and the weights of 64 columns at
// a time lie in LDS for all four, the next ones on their way.  y is on its way two
// steps ahead, asked for before the step's results are stored, since a wait for
// it is one for the stores before it too (one step ahead: 10313 tokens to 5120
// at rank 64 58 us, so 55; 24287 to 5664 169 and 158).  (Through up_group's
// way, with the inner products in LDS and the weights in registers, 142 tokens of
// rank 72 took 23 us in place of 16, long prompts as much as here.)
template <int KB>
constexpr int tile_row() {
  return 64 * KB + 16;  // bytes of a row of weights: an odd number of pieces, so that 8 rows' same pieces come from all banks
}
template <bool BF, int KB>
__device__ __forceinline__ void up_tile(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, int64_t m_begin,
                                        int64_t m_end, char* room) {
  constexpr int kRow = tile_row<KB>(), kBuffer = 64 * kRow;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  // thread: row tid / 4 of 64, pieces tid % 4 + 4 k
  const int row = tid >> 2, piece = tid & 3, column = column_of(row >> 4, row & 15);
  const char* up = reinterpret_cast<const char*>(l.up + g.adapter * l.up_adapter) + 16 * piece;
  uint4 wn[KB];
  auto fetch = [&](int64_t m0) {
    int64_t m = m0 + column;
    m = m < l.m ? m : l.m - 1;  // the results of columns beyond go nowhere
    const char* from = up + 2 * m * l.up_row;
#pragma unroll
    for (int k = 0; k < KB; ++k) wn[k] = 32 * k + 8 * piece < l.rank ? *reinterpret_cast<const uint4*>(from + 64 * k) : uint4{};
  };
  auto keep = [&](int buffer) {
#pragma unroll
    for (int k = 0; k < KB; ++k) *reinterpret_cast<uint4*>(room + buffer * kBuffer + row * kRow + 64 * k + 16 * piece) = wn[k];
  };
  fetch(m_begin);
  const int c = 16 * w + r;
  const uint32_t place = place_in_tile(g, c);
  const char* y0 = reinterpret_cast<const char*>(l.y + t0 * l.ldy) + 2u * (place * (uint32_t)l.ldy + 8 * q);
  char* out0 = reinterpret_cast<char*>(l.out + t0 * l.ldo) + 2u * (place * (uint32_t)l.ldo + 8 * q);
  auto left_of = [&](int64_t m0) { return (int)(l.m - m0 < 64 ? l.m - m0 : 64) - 8 * q; };
  const bool mine = c < g.size;
  uint4 y[2][2], h[KB], o[KB];
  if (mine) load_y(y0 + 2 * m_begin, left_of(m_begin), y[0]);
  if (mine && m_begin + 64 < m_end) load_y(y0 + 2 * (m_begin + 64), left_of(m_begin + 64), y[1]);
  float scale;
  {
    const float* from = a.part + (t0 + place) * a.ranks + l.offset;
    f32x4 s[KB][2];
#pragma unroll
    for (int k = 0; k < KB; ++k) s[k][0] = s[k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t next = a.tokens * a.ranks;
#pragma unroll 8
    for (int p = 0; p < a.splits; ++p)
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int rank = 32 * k + 8 * q;
        const float* at = from + p * next + (rank < l.rank ? rank : 0);
        s[k][0] += *reinterpret_cast<const f32x4*>(at), s[k][1] += *reinterpret_cast<const f32x4*>(at + 4);
      }
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (32 * k + 8 * q >= l.rank) s[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(s[k][i][e]));
      }
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    float grow;
    const float shrink = powers(most, grow);
    scale = grow * l.scale[g.adapter];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) two_parts<BF>(s[k][x >> 1][2 * (x & 1)] * shrink, s[k][x >> 1][2 * (x & 1) + 1] * shrink, hi[x], lo[x]);
      h[k] = make_uint4(hi[0], hi[1], hi[2], hi[3]), o[k] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
  __syncthreads();  // the group before is done with the room
  keep(0);
  if (m_begin + 64 < m_end) fetch(m_begin + 64);
  __syncthreads();
  auto step = [&](int64_t m0, int buffer, uint4 (&yb)[2]) {
    if (16 * w < g.size) {
      f32x4 acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      const char* at = room + buffer * kBuffer + r * kRow + 16 * q;
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 wv = *reinterpret_cast<const uint4*>(at + 16 * j * kRow + 64 * k);
          acc[j] = mma_16x16x32<BF>(wv, o[k], mma_16x16x32<BF>(wv, h[k], acc[j]));
        }
      const uint4 o8[2] = {add_8<BF>(yb[0], acc[0], acc[1], scale), add_8<BF>(yb[1], acc[2], acc[3], scale)};
      if (mine) {
        if (m0 + 128 < m_end) load_y(y0 + 2 * (m0 + 128), left_of(m0 + 128), yb);
        store_out(out0 + 2 * m0, left_of(m0), o8);
      }
    }
    if (m0 + 64 < m_end) keep(buffer ^ 1);  // all are done with it since the last barrier
    if (m0 + 128 < m_end) fetch(m0 + 128);
    __syncthreads();
  };
  for (int64_t m0 = m_begin; m0 < m_end; m0 += 128) {
    step(m0, 0, y[0]);
    if (m0 + 64 < m_end) step(m0 + 64, 1, y[1]);
  }
}

// y of the tokens without an adapter goes on as it is, four tokens of a wave at a time.
__device__ __forceinline__ void copy_group(const Linear& l, const Group& g, int64_t t0, int64_t m_begin, int64_t m_end) {
  constexpr int U = 4;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int c0 = w; c0 < g.size; c0 += 4 * U) {
    int64_t t[U];
#pragma unroll
    for (int i = 0; i < U; ++i) t[i] = t0 + place_in_tile(g, c0 + 4 * i);  // the last token again behind it
    for (int64_t m = m_begin + 8 * lane; m < m_end; m += 512) {
      if (m + 8 <= m_end) {
        u32x4 v[U];
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = *reinterpret_cast<const Loose*>(l.y + t[i] * l.ldy + m);
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (c0 + 4 * i < g.size) *reinterpret_cast<Loose*>(l.out + t[i] * l.ldo + m) = v[i];
      } else {
        for (int64_t e = m; e < m_end; ++e)
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (c0 + 4 * i < g.size) l.out[t[i] * l.ldo + e] = l.y[t[i] * l.ldy + e];
      }
    }
  }
}

// (For ranks up to 96 the compiler would take more than 256 registers by itself,
// and one wave a SIMD: 20719 tokens of rank 88 313 us, with two 222.)
template <bool BF, int KB, bool MANY>
__global__ __launch_bounds__(kThreads, MANY && KB == 3 ? 2 : 1) void adapter_up_kernel(AdapterArgs a) {
  constexpr int kFew = 16 * (32 * KB + 8) * 4 + 64, kMany = MANY ? 2 * 64 * tile_row<KB>() : 0;
  __shared__ __align__(16) char room[kMany > kFew ? kMany : kFew];
  int gi = 0;
  while (gi + 1 < a.count && (int)blockIdx.x >= a.linear[gi + 1].first) ++gi;
  const Linear& l = a.linear[gi];
  const int64_t m_begin = (int64_t)((int)blockIdx.x - l.first) * a.span;
  const int64_t m_end = m_begin + a.span < l.m ? m_begin + a.span : l.m;
  const int64_t t0 = (int64_t)(blockIdx.y % a.tiles) * kTile;
  each_group(a, t0, blockIdx.y / a.tiles, l.out != l.y, [&](const Group& g) {
    if (g.adapter < 0) return copy_group(l, g, t0, m_begin, m_end);
    if constexpr (MANY) {
      if (g.size > 16) return up_tile<BF, KB>(a, l, g, t0, m_begin, m_end, room);
    }
    up_group<BF, KB>(a, l, g, t0, m_begin, m_end, room);
  });
}

template <bool BF>
auto down_kernel(int blocks, bool many) {
  if (many) return blocks == 2 ? adapter_down_kernel<BF, 2, true> : blocks == 4 ? adapter_down_kernel<BF, 4, true>
                   : blocks == 6 ? adapter_down_kernel<BF, 6, true> : adapter_down_kernel<BF, 8, true>;
  return blocks == 1 ? adapter_down_kernel<BF, 1, false> : blocks == 2 ? adapter_down_kernel<BF, 2, false> : adapter_down_kernel<BF, 4, false>;
}
template <bool BF, bool MANY>
auto up_kernel(int rank) {
  return rank <= 32 ? adapter_up_kernel<BF, 1, MANY> : rank <= 64 ? adapter_up_kernel<BF, 2, MANY>
         : rank <= 96 ? adapter_up_kernel<BF, 3, MANY> : adapter_up_kernel<BF, 4, MANY>;
}

struct Plan {
  int64_t tiles;
  int slots, blocks, runs;  // blocks of 16 ranks of a work-group, and work-groups for all of them
  int splits, steps;
};

Plan plan_of(int64_t tokens, int64_t n, int64_t adapters, int count, const int* ranks) {
  Plan p;
  p.tiles = (tokens + kTile - 1) / kTile;
  const int64_t most = tokens < kTile ? tokens : kTile, share = p.tiles < 128 ? 128 / p.tiles : 1;
  const int64_t slots = most < share ? most : share;
  p.slots = 1;
  while (p.slots < slots && p.slots < adapters + 1) p.slots *= 2;
  int all = 0;
  for (int g = 0; g < count; ++g) all += ranks[g];
  const int blocks = (all + 15) / 16;
  const int64_t steps = (n + 255) / 256, groups = p.tiles * (p.slots < 8 ? 1 : p.slots / 2);
  // Few tokens need many narrow work-groups, many tokens wide ones that read x
  // once: one token's 48 ranks of 4096 inputs in blocks of 16 take 4.2 us, in one of
  // 64 5.1; 48 tokens that name 21 adapters of 128 ranks in blocks of 32 11.9, of 64 9.8;
  // 229 tokens with 128 ranks in blocks of 32 6.6, of 64 7.6, of 128 10.4; 848 with
  // 240 ranks 16.2, 13.8 and 16.3; 5641 with 160 ranks of 24296 inputs in blocks of
  // 64 254, of 96 194.
  auto widest = [&](int width) { p.runs = (blocks + width - 1) / width, p.blocks = (blocks + p.runs - 1) / p.runs; };
  if (p.tiles == 1) {
    int width = tokens > 16 ? 2 : 1;
    widest(width);
    while (width < 4 && groups * p.runs * (steps < 16 ? steps : 16) > 512) widest(width *= 2);
  } else {
    widest(p.tiles < 16 ? 2 : p.tiles < 64 ? 4 : 8);
  }
  if (p.blocks > 1 || tokens > 16) p.blocks += p.blocks & 1;
  // Splits fill the GPU, but each is read again by the second launch: 4260 tokens
  // of 6 prompts with 4 splits of 3584 inputs (268 work-groups) take 15 + 25 us, with 8 18
  // + 29, with 2 18 + 23.  Groups of single tokens have shorter loops and want four
  // times as many.
  int64_t splits = 1;
  if (p.tiles == 1) splits = (1024 + groups * p.runs - 1) / (groups * p.runs);
  else while (splits < 8 && groups * p.runs * splits < 256) splits *= 2;
  splits = splits < steps ? splits : steps;
  splits = splits < 16 ? splits : 16;
  p.steps = (int)((steps + splits - 1) / splits);
  p.splits = (int)((steps + p.steps - 1) / p.steps);
  return p;
}

// Columns of a work-group of the second launch, which splits up the inner
// products once for all of them.  Groups of single tokens take 256 at a time, 64 a
// wave, and 512 work-groups of them fill the GPU (48 tokens to 2 x 25600: 33 us with
// 1024 columns, 48 with 256).  Prompts take 64 at a time and are cut finer where
// there are few (142 tokens to 1315 columns: 8.5 us with 64, 12 with 256) and coarser
// where there are many (10313 to 5120: 58 us with 512, 62 with 256, 80 with 128; but
// 5641 to 12659 151 us with 1024, 128 with 512); work-groups of slots without a group
// cost their launch (74 tokens in 32 slots to 20507 columns: 20 us with 64, 9 with 256).
int span_of(const Plan& p, int64_t columns) {
  int span;
  if (p.tiles == 1) {
    const int64_t groups = p.slots < 8 ? 1 : p.slots / 2;
    span = kColumns;
    while (span < 8 * kColumns && groups * columns / (2 * span) >= 512) span *= 2;
  } else {
    span = 64;
    while (span < (p.slots > 1 ? 256 : 512) && p.tiles * p.slots * columns / (2 * span) >= 640) span *= 2;
  }
  return span;
}

// What linear g's output shares memory with of all that the call reads and
// writes, its own y at the same place aside; nullptr: nothing.
const char* meets(const AdapterArgs& a, const qs_adapter_job* jobs, int g) {
  auto rows = [&](const void* p, int64_t ld, int64_t width) { return Rows{p, a.tokens, 2 * ld, 2 * width}; };
  auto weights = [&](const void* p, int64_t adapter, int64_t rows, int64_t row, int64_t width, const Rows& out) {
    const Rows all{p, 1, 0, 2 * ((a.adapters - 1) * adapter + (rows - 1) * row + width)};
    if (!share_memory(all, out)) return false;
    for (int64_t i = 0; i < a.adapters; ++i)
      if (share_memory(Rows{static_cast<const uint16_t*>(p) + i * adapter, rows, 2 * row, 2 * width}, out)) return true;
    return false;
  };
  const qs_adapter_job& j = jobs[g];
  const Rows out = rows(j.out, j.ldo, j.m);
  if (share_memory(out, rows(a.x, a.ldx, a.n))) return "x";
  if (share_memory(out, Rows{a.which, 1, 0, 4 * a.tokens})) return "which";
  for (int h = 0; h < a.count; ++h) {
    const qs_adapter_job& k = jobs[h];
    if (!(h == g && k.y == j.out) && share_memory(out, rows(k.y, k.ldy, k.m))) return "a y";
    if (h != g && share_memory(out, rows(k.out, k.ldo, k.m))) return "another output";
    if (weights(k.down, k.down_adapter, k.rank, k.down_row, a.n, out) || weights(k.up, k.up_adapter, k.m, k.up_row, k.rank, out) ||
        share_memory(out, Rows{k.scale, 1, 0, 4 * (int64_t)a.adapters}))
      return "weights";
  }
  return nullptr;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_adapters_workspace_bytes(int64_t tokens, int64_t n, int64_t adapters, int count, const int* ranks) {
  if (tokens < 1 || n < 1 || adapters < 1 || count < 1 || count > QS_MAX_GROUP || !ranks) return 0;
  int64_t all = 0;
  for (int g = 0; g < count; ++g) {
    if (ranks[g] < 1 || ranks[g] > kMaxRank) return 0;
    all += ranks[g];
  }
  if (tokens > kMaxTokens) return 0;
  // What any number of tokens up to this takes, of any number of adapters: fewer
  // tokens may be cut into more splits.  One tile has up to 16, several up to 8, and
  // fewer than 512 work-groups if more than one.
  const int64_t steps = (n + 255) / 256, one = tokens < kTile ? tokens : kTile;
  int64_t rows = one * (steps < 16 ? steps : 16);
  if (tokens > kTile) {
    int64_t more = tokens * (steps < 8 ? steps : 8);
    more = more < 512 * kTile ? more : 512 * kTile;
    more = more > tokens ? more : tokens;
    rows = rows > more ? rows : more;
  }
  return (size_t)(rows * all) * sizeof(float);
}

extern "C" int qs_adapters_plan(int64_t tokens, int64_t n, int64_t adapters, int count, const int* ranks, const int64_t* ms, int* plan) {
  QS_REQUIRE(ranks && ms && plan, "qs_adapters_plan: null pointer");
  QS_REQUIRE(qs_adapters_workspace_bytes(tokens, n, adapters, count, ranks) > 0, "qs_adapters_plan: no such call");
  int64_t columns = 0;
  for (int g = 0; g < count; ++g) columns += ms[g];
  const Plan p = plan_of(tokens, n, adapters, count, ranks);
  plan[0] = p.slots, plan[1] = p.blocks, plan[2] = p.runs, plan[3] = p.splits, plan[4] = span_of(p, columns);
  return QS_OK;
}

extern "C" int qs_adapters_add(const void* x, int dtype, int64_t ldx, int64_t tokens, int64_t n, const int32_t* which,
                               int64_t adapters, int count, const qs_adapter_job* jobs, void* workspace,
                               size_t workspace_bytes, qs_stream_t stream) {
  const char* fn = "qs_adapters_add";
  if (tokens == 0) return QS_OK;
  QS_REQUIRE(x && which && jobs, "%s: null pointer", fn);
  QS_REQUIRE(dtype == QS_DTYPE_F16 || dtype == QS_DTYPE_BF16, "%s: dtype %d", fn, dtype);
  QS_REQUIRE(count >= 1 && count <= QS_MAX_GROUP, "%s: %d linears (at most %d)", fn, count, QS_MAX_GROUP);
  QS_REQUIRE(tokens >= 1 && n >= 8 && n % 8 == 0 && adapters >= 1 && adapters <= INT32_MAX && (tokens == 1 || ldx >= n) && ldx % 8 == 0 &&
                 (reinterpret_cast<uintptr_t>(x) & 15) == 0,
             "%s: %lld rows of %lld (a multiple of 8), %lld apart, %lld adapters; rows must be 16-byte aligned", fn,
             (long long)tokens, (long long)n, (long long)ldx, (long long)adapters);
  QS_SUPPORTED(tokens <= kMaxTokens && ldx <= (1 << 24), "%s: %lld rows of %lld, %lld apart", fn, (long long)tokens, (long long)n, (long long)ldx);
  AdapterArgs a{};
  a.x = static_cast<const uint16_t*>(x), a.ldx = tokens == 1 ? 0 : ldx, a.tokens = tokens, a.n = n, a.which = which;
  a.adapters = (int)adapters, a.count = count;
  int most = 0, ranks[QS_MAX_GROUP];
  int64_t columns = 0;
  for (int g = 0; g < count; ++g) {
    const qs_adapter_job& j = jobs[g];
    QS_REQUIRE(j.down && j.up && j.scale && j.y && j.out, "%s: linear %d: null pointer", fn, g);
    QS_REQUIRE(j.rank >= 8 && j.rank % 8 == 0 && j.rank <= kMaxRank, "%s: linear %d: rank %d (a multiple of 8 up to %d)", fn, g, j.rank, kMaxRank);
    QS_REQUIRE(j.m >= 1 && j.m <= (1 << 30) && (tokens == 1 || (j.ldy >= j.m && j.ldo >= j.m)), "%s: linear %d: rows of %lld outputs, %lld and %lld apart",
               fn, g, (long long)j.m, (long long)j.ldy, (long long)j.ldo);
    QS_REQUIRE(j.down_row >= n && j.up_row >= j.rank && j.down_adapter >= 0 && j.up_adapter >= 0 &&
                   (j.down_row | j.up_row | j.down_adapter | j.up_adapter) % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(j.down) | reinterpret_cast<uintptr_t>(j.up)) & 15) == 0,
               "%s: linear %d: weights must be 16-byte aligned, rows %lld and %lld apart", fn, g, (long long)j.down_row, (long long)j.up_row);
    QS_SUPPORTED(j.down_row <= (1 << 24) && j.up_row <= (1 << 24) && (tokens == 1 || (j.ldy <= (1 << 24) && j.ldo <= (1 << 24))),
                 "%s: linear %d: weights' rows %lld and %lld apart, y and out %lld and %lld", fn, g, (long long)j.down_row, (long long)j.up_row, (long long)j.ldy, (long long)j.ldo);
    QS_REQUIRE(((reinterpret_cast<uintptr_t>(j.y) | reinterpret_cast<uintptr_t>(j.out)) & 1) == 0 && (reinterpret_cast<uintptr_t>(j.scale) & 3) == 0,
               "%s: linear %d: tensors must be aligned to their elements", fn, g);
    QS_REQUIRE(j.y != j.out || tokens == 1 || j.ldy == j.ldo, "%s: linear %d: y and out share memory with rows %lld and %lld apart", fn, g,
               (long long)j.ldy, (long long)j.ldo);
    for (int h = 0; h < count; ++h)
      QS_REQUIRE(h == g || (j.out != jobs[h].y && j.out != jobs[h].out), "%s: the output of linear %d is linear %d's y or output", fn, g, h);
    QS_REQUIRE(j.out != x, "%s: the output of linear %d is x", fn, g);
    a.linear[g] = Linear{static_cast<const uint16_t*>(j.down), static_cast<const uint16_t*>(j.up), j.scale,
                         static_cast<const uint16_t*>(j.y), static_cast<uint16_t*>(j.out), j.down_adapter, j.down_row,
                         j.up_adapter, j.up_row, tokens == 1 ? 0 : j.ldy, tokens == 1 ? 0 : j.ldo, j.m, j.rank, a.ranks, 0};
    a.ranks += j.rank, ranks[g] = j.rank;
    most = j.rank > most ? j.rank : most;
    columns += j.m;
  }
  for (int g = 0; g < count; ++g) {
    const char* with = meets(a, jobs, g);
    QS_REQUIRE(!with, "%s: the output of linear %d shares memory with %s", fn, g, with);
  }
  const Plan p = plan_of(tokens, n, adapters, count, ranks);
  a.tiles = (int)p.tiles, a.runs = p.runs, a.splits = p.splits, a.steps = p.steps;
  const size_t need = (size_t)p.splits * tokens * a.ranks * sizeof(float);
  QS_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "%s: workspace of %zu bytes (16-byte aligned), %zu needed", fn, workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  a.span = span_of(p, columns);
  int grid = 0;
  for (int g = 0; g < count; ++g) {
    a.linear[g].first = grid;
    grid += (int)((a.linear[g].m + a.span - 1) / a.span);
  }
  const bool bf = dtype == QS_DTYPE_BF16;
  const auto down = bf ? down_kernel<true>(p.blocks, tokens > 16) : down_kernel<false>(p.blocks, tokens > 16);
  // at a boundary of two prompts the second one's tokens go to work-groups of
  // their own: 15 us in place of 21 where 4260 tokens of 6 prompts have 72 ranks of
  // 3584 inputs.  (The second launch has many more, of which half would be empty.)
  a.slots = p.tiles > 1 && p.slots < 2 ? 2 : p.slots;
  const int64_t units = p.tiles > 1 ? (p.tiles * a.slots * p.splits + 7) / 8 * 8 : a.slots * p.splits;
  hipLaunchKernelGGL(down, dim3((unsigned)units * p.runs), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("adapter_down_kernel");
  const auto up = tokens > 16 ? (bf ? up_kernel<true, true>(most) : up_kernel<false, true>(most))
                              : (bf ? up_kernel<true, false>(most) : up_kernel<false, false>(most));
  a.slots = p.slots;
  hipLaunchKernelGGL(up, dim3((unsigned)grid, (unsigned)(p.tiles * p.slots)), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("adapter_up_kernel");
  return QS_OK;
}
