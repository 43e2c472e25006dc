// Low-rank adapters of many requests beside shared projections
// (qs_adapters_add): for up to four linears g that read the same rows,
//
//   out_g[t] = y_g[t] + scale_g[a] up_g[a] (down_g[a] x[t]),   a = which[t]
//
// with rows that have no adapter left as they are.  Two launches: the inner
// products with `down` (K = n is long, so it is split over work-groups, each
// split leaving its fp32 sums), then the ones with `up` (K = rank), in whose
// first step the splits are added.
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

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;     // tokens at a time
constexpr int kMaxRank = 128;
constexpr int kColumns = 256;  // output columns of a work-group at a time, 64 a wave

struct Linear {
  const uint16_t *down, *up;
  const float* scale;
  const uint16_t* y;
  uint16_t* out;
  int64_t down_adapter, down_row, up_adapter, up_row, ldy, ldo, m;
  int rank, offset;  // offset: of its ranks among those of all linears
  int first_run, first;  // its first work-group column of the first and the second launch
};

struct AdapterArgs {
  const uint16_t* x;
  int64_t ldx, tokens, n;
  const int32_t* which;
  int adapters, count, ranks;  // ranks: of all linears together
  int splits, steps;           // steps of 256 inputs of a split
  int slots, chunks;           // work-groups that share a tile's groups, a power of two; runs of kColumns of a work-group
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

// One group of the first launch: NB blocks of 16 tokens, RB of 16 ranks from
// rank0 on.  All that changes along the inputs is a scalar; a lane's places in
// the rows are 32-bit offsets.
template <bool BF, int RB, int NB>
__device__ __forceinline__ void down_group(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, int split, int rank0,
                                           f32x4 (*sums)[NB][64]) {
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  const char* x = reinterpret_cast<const char*>(a.x + t0 * a.ldx);
  const char* down = reinterpret_cast<const char*>(l.down + g.adapter * l.down_adapter);
  uint32_t x_at[NB], down_at[RB];
#pragma unroll
  for (int b = 0; b < NB; ++b) x_at[b] = 2u * ((uint32_t)place_in_tile(g, 16 * b + r) * (uint32_t)a.ldx + 8 * q);
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int rank = rank0 + 16 * i + r;  // the sums of rows beyond go nowhere
    down_at[i] = 2u * ((uint32_t)(rank < l.rank ? rank : l.rank - 1) * (uint32_t)l.down_row + 8 * q);
  }
  f32x4 acc[RB][NB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int n = (int)a.n, k0 = split * a.steps * 256, k1 = k0 + a.steps * 256 < n ? k0 + a.steps * 256 : n;
  // 64 inputs at a time, 32 for each of two products
  uint4 xv[NB][2], av[RB][2];
  auto load = [&](int k) {
    const char *xk = x + 2 * (int64_t)k, *dk = down + 2 * (int64_t)k;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int b = 0; b < NB; ++b) xv[b][j] = *reinterpret_cast<const uint4*>(xk + x_at[b] + 64 * j);
#pragma unroll
      for (int i = 0; i < RB; ++i) av[i][j] = *reinterpret_cast<const uint4*>(dk + down_at[i] + 64 * j);
    }
  };
  auto multiply = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[i][b] = mma_16x16x32<BF>(av[i][j], xv[b][j], acc[i][b]);
  };
  int k = k0 + 64 * w;
  for (; k + 64 <= k1; k += 256) load(k), multiply();
  if (k < k1) {
    // fewer than 64 are left: zeros behind them
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool in = k + 32 * j + 8 * q < k1;
#pragma unroll
      for (int b = 0; b < NB; ++b) xv[b][j] = in ? *reinterpret_cast<const uint4*>(x + 2 * (int64_t)k + x_at[b] + 64 * j) : uint4{};
#pragma unroll
      for (int i = 0; i < RB; ++i) av[i][j] = in ? *reinterpret_cast<const uint4*>(down + 2 * (int64_t)k + down_at[i] + 64 * j) : uint4{};
    }
    multiply();
  }
  // the waves' sums together, a block of ranks at a time
  float* part = a.part + ((int64_t)split * a.tokens + t0) * a.ranks + l.offset;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
#pragma unroll
    for (int b = 0; b < NB; ++b) sums[w][b][lane] = acc[i][b];
    __syncthreads();
    if (NB == 4 || w < NB) {
      const int c = 16 * w + r, rank = rank0 + 16 * i + 4 * q;
      const f32x4 s = (sums[0][w][lane] + sums[1][w][lane]) + (sums[2][w][lane] + sums[3][w][lane]);
      const int place = place_in_tile(g, c);  // an exchange of all lanes
      if (c < g.size && rank < l.rank) *reinterpret_cast<f32x4*>(part + place * a.ranks + rank) = s;
    }
    __syncthreads();
  }
}

// The same for more than 16 tokens: 64 tokens and 16 RB ranks by 64 inputs at a
// time go straight to LDS, kAhead such stages ahead of their use, and each wave
// multiplies its 16 tokens.  A row of a stage is eight pieces of 16 bytes, of
// which piece p lies at place p ^ (row & 7), so that a wave's operands (one
// piece of each of 16 rows) come from all banks.
constexpr int kStageRow = 128, kAhead = 3;
template <int RB>
constexpr int stage_bytes() {
  return (kTile + 16 * RB) * kStageRow;
}

template <bool BF, int RB>
__device__ __forceinline__ void down_tile(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, int split, int rank0, char* stages) {
  constexpr int NX = kTile / 32, NW = RB / 2, NL = NX + NW;  // loads of a wave in a stage, of 8 rows each
  static_assert(RB % 2 == 0, "every wave brings as many rows");
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  const int n = (int)a.n, k0 = split * a.steps * 256, k1 = k0 + a.steps * 256 < n ? k0 + a.steps * 256 : n;
  const int count = (k1 - k0 + 63) / 64, left = k1 - k0 - 64 * (count - 1);  // stages, inputs of the last
  const int row8 = lane >> 3;  // of a load; every load begins at a multiple of 8 rows
  const unsigned piece = 16 * ((lane & 7) ^ row8);
  unsigned x_row[NX], down_row[NW], x_at[NX], down_at[NW];
#pragma unroll
  for (int j = 0; j < NX; ++j) x_row[j] = 2u * (uint32_t)place_in_tile(g, 8 * (NX * w + j) + row8) * (uint32_t)a.ldx, x_at[j] = x_row[j] + piece;
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    const int rank = rank0 + 8 * (NW * w + j) + row8;  // the sums of rows beyond go nowhere
    down_row[j] = 2u * (uint32_t)(rank < l.rank ? rank : l.rank - 1) * (uint32_t)l.down_row, down_at[j] = down_row[j] + piece;
  }
  const char* x = reinterpret_cast<const char*>(a.x + t0 * a.ldx + k0);
  const char* down = reinterpret_cast<const char*>(l.down + g.adapter * l.down_adapter + k0);
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_address(stages));
  auto fetch = [&](int s) {
    const unsigned to = lds + (unsigned)(s % (kAhead + 1)) * stage_bytes<RB>();
    if (s == count - 1 && left < 64) {
      // pieces behind the last input: the last one again, which is not used
      const unsigned end = 2u * (left - 8), p = piece < end ? piece : end;
#pragma unroll
      for (int j = 0; j < NX; ++j) x_at[j] = x_row[j] + p;
#pragma unroll
      for (int j = 0; j < NW; ++j) down_at[j] = down_row[j] + p;
    }
    load_rows(x + 128 * (int64_t)s, x_at, to + w * (NX * 1024));
    load_rows(down + 128 * (int64_t)s, down_at, to + kTile * kStageRow + w * (NW * 1024));
  };
  f32x4 acc[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool busy = 16 * w < g.size;
#pragma unroll
  for (int s = 0; s < kAhead; ++s)
    if (s < count) fetch(s);
  for (int s = 0; s < count; ++s) {
    if (s + kAhead <= count) wait_loads<(kAhead - 1) * NL>();
    else wait_loads<0>();
    __syncthreads();
    if (s + kAhead < count) fetch(s + kAhead);
    if (busy) {
      const char* at = stages + (s % (kAhead + 1)) * stage_bytes<RB>();
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
  float* part = a.part + ((int64_t)split * a.tokens + t0 + place) * a.ranks + l.offset;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int rank = rank0 + 16 * i + 4 * q;
    if (c < g.size && rank < l.rank) *reinterpret_cast<f32x4*>(part + rank) = acc[i];
  }
  __syncthreads();  // the next group's stages lie where these did
}

// blockIdx.x: (linear, its run of 16 RB ranks, split), the split fastest.
template <bool BF, int RB, bool MANY>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterArgs a) {
  constexpr int kSums = 4 * 64 * sizeof(f32x4), kStages = MANY ? (kAhead + 1) * stage_bytes<RB>() : 0;
  __shared__ __align__(16) char room[kStages > kSums ? kStages : kSums];
  const int split = blockIdx.x % a.splits, run = blockIdx.x / a.splits;
  int gi = 0;
  while (gi + 1 < a.count && run >= a.linear[gi + 1].first_run) ++gi;
  const Linear& l = a.linear[gi];
  const int rank0 = (run - l.first_run) * (16 * RB);
  const int64_t t0 = (int64_t)(blockIdx.y / a.slots) * kTile;
  each_group(a, t0, blockIdx.y & (a.slots - 1), false, [&](const Group& g) {
    if constexpr (MANY) {
      if (g.size > 16) return down_tile<BF, RB>(a, l, g, t0, split, rank0, room);
    }
    down_group<BF, RB, 1>(a, l, g, t0, split, rank0, reinterpret_cast<f32x4(*)[1][64]>(room));
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

// The inner products of N tokens of a group, summed over the splits, as two
// 16-bit numbers: four ranks a thread, a token's R / 4 threads in one wave.
template <bool BF, int R, int kRow, int N>
__device__ __forceinline__ void inner_products(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, uint4* high,
                                               uint4* low, float* factor) {
  constexpr int T = R / 4, I = N * T / kThreads > 0 ? N * T / kThreads : 1, U = I < 2 ? 1 : 2;
  const int tid = threadIdx.x;
  if (N * T < kThreads && tid >= N * T) return;  // whole waves: N T is a multiple of 64
  const float* base = a.part + t0 * a.ranks + l.offset;
  const int64_t next = a.tokens * a.ranks;
  const int rank = tid % T * 4;
  const float scale = l.scale[g.adapter];
#pragma unroll
  for (int i0 = 0; i0 < I; i0 += U) {
    f32x4 s[U];
    uint32_t from[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      from[i] = (uint32_t)place_in_tile(g, (i0 + i) * (kThreads / T) + tid / T) * (uint32_t)a.ranks + (rank < l.rank ? rank : 0);
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll 4
    for (int p = 0; p < a.splits; ++p)
#pragma unroll
      for (int i = 0; i < U; ++i) s[i] += *reinterpret_cast<const f32x4*>(base + p * next + from[i]);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = (i0 + i) * (kThreads / T) + tid / T;
      if (rank >= l.rank) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      float most = fmaxf(fmaxf(fabsf(s[i][0]), fabsf(s[i][1])), fmaxf(fabsf(s[i][2]), fabsf(s[i][3])));
#pragma unroll
      for (int x = 1; x < T; x *= 2) most = fmaxf(most, __shfl_xor(most, x));
      int e = (int)(__float_as_uint(most) >> 23);
      e = e < 2 ? 2 : e > 252 ? 252 : e;
      const float shrink = __uint_as_float((uint32_t)(254 - e) << 23);
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f0 = s[i][2 * x] * shrink, f1 = s[i][2 * x + 1] * shrink;
        hi[x] = pack16<BF>(f0, f1);
        const float h0 = float_of<BF>(hi[x] & 0xFFFF), h1 = float_of<BF>(hi[x] >> 16);
        // an infinite product has no remainder
        lo[x] = pack16<BF>(fabsf(h0) < INFINITY ? f0 - h0 : 0.f, fabsf(h1) < INFINITY ? f1 - h1 : 0.f);
      }
      const int at = (c * kRow + rank) / 4;
      reinterpret_cast<uint2*>(high)[at] = make_uint2(hi[0], hi[1]), reinterpret_cast<uint2*>(low)[at] = make_uint2(lo[0], lo[1]);
      if (rank == 0) factor[c] = __uint_as_float((uint32_t)e << 23) * scale;
    }
    __builtin_amdgcn_sched_barrier(0);  // more at a time would take more registers than the products
  }
}

// The second launch: a group's tokens, NB blocks of 16, against 64 columns a
// wave at a time.
template <bool BF, int KB, int NB>
__device__ __forceinline__ void up_group(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, int64_t m_begin,
                                         int64_t m_end, uint4* high, uint4* low, float* factor) {
  constexpr int R = 32 * KB, kRow = R + 8;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4, r = lane & 15;
  const char* up = reinterpret_cast<const char*>(l.up + g.adapter * l.up_adapter);
  auto row_of = [&](int j) { return 32 * (j >> 1) + 8 * (r >> 2) + 4 * (j & 1) + (r & 3); };
  uint32_t w_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w_at[j] = 2u * ((uint32_t)row_of(j) * (uint32_t)l.up_row + 8 * q);
  auto weights = [&](int64_t m0, uint4 (&wv)[4][KB]) {
    const char* from = up + 2 * m0 * l.up_row;
    const int last = m0 + 64 <= l.m ? 63 : (int)(l.m - m0) - 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = row_of(j) <= last ? w_at[j] : 2u * ((uint32_t)last * (uint32_t)l.up_row + 8 * q);
#pragma unroll
      for (int k = 0; k < KB; ++k)
        wv[j][k] = 32 * k + 8 * q < l.rank ? *reinterpret_cast<const uint4*>(from + at + 64 * k) : uint4{};
    }
  };
  // A lane's results of a token are columns m0 + 8 q .. + 7 and m0 + 32 + 8 q .. + 7, so that an access of the wave
  // takes 64 bytes together of 16 rows.
  const char* y0 = reinterpret_cast<const char*>(l.y + t0 * l.ldy);
  char* out0 = reinterpret_cast<char*>(l.out + t0 * l.ldo);
  uint32_t y_at[NB], out_at[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t place = place_in_tile(g, 16 * b + r);
    y_at[b] = 2u * (place * (uint32_t)l.ldy + 8 * q), out_at[b] = 2u * (place * (uint32_t)l.ldo + 8 * q);
  }
  uint4 wv[4][KB], y[NB][2];
  auto load_y = [&](int b, int64_t m0) {
    const char* from = y0 + 2 * m0;
    if (m0 + 64 <= l.m) {
      y[b][0] = get_loose(from + y_at[b]), y[b][1] = get_loose(from + y_at[b] + 64);
    } else {
      const int left = (int)(l.m - m0) - 8 * q;  // columns from the lane's first on
      if (left > 0) y[b][0] = left < 8 ? get_some(from + y_at[b], left) : get_loose(from + y_at[b]);
      if (left > 32) y[b][1] = left < 40 ? get_some(from + y_at[b] + 64, left - 32) : get_loose(from + y_at[b] + 64);
    }
  };
  int64_t m0 = m_begin + 64 * w;
  if (m0 < m_end) {
    weights(m0, wv);
#pragma unroll
    for (int b = 0; b < NB; ++b) load_y(b, m0);
  }
  __syncthreads();  // the group before is done with the tables
  inner_products<BF, R, kRow, 16 * NB>(a, l, g, t0, high, low, factor);
  __syncthreads();
  for (; m0 < m_end; m0 += kColumns) {
    const bool more = m0 + kColumns < m_end;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int c = 16 * b + r;
      f32x4 acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const uint4 h = high[(c * kRow + 32 * k + 8 * q) / 8], o = low[(c * kRow + 32 * k + 8 * q) / 8];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = mma_16x16x32<BF>(wv[j][k], o, mma_16x16x32<BF>(wv[j][k], h, acc[j]));
      }
      if (b == NB - 1 && more) weights(m0 + kColumns, wv);
      if (c < g.size) {
        const float scale = factor[c];
        char* to = out0 + 2 * m0 + out_at[b];
        const uint4 o0 = add_8<BF>(y[b][0], acc[0], acc[1], scale), o1 = add_8<BF>(y[b][1], acc[2], acc[3], scale);
        if (m0 + 64 <= l.m) {
          put_loose(to, o0), put_loose(to + 64, o1);
        } else {
          const int left = (int)(l.m - m0) - 8 * q;
          if (left >= 8) put_loose(to, o0);
          else if (left > 0) put_some(to, o0, left);
          if (left >= 40) put_loose(to + 64, o1);
          else if (left > 32) put_some(to + 64, o1, left - 32);
        }
      }
      if (more) load_y(b, m0 + kColumns);
      __builtin_amdgcn_sched_barrier(0);  // blocks that overlap would take twice the registers
    }
  }
}

// y of the tokens without an adapter goes on as it is, eight tokens of a wave at a time.
__device__ __forceinline__ void copy_group(const Linear& l, const Group& g, int64_t t0, int64_t m_begin, int64_t m_end) {
  constexpr int U = 8;
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

template <bool BF, int KB, int NB>
__global__ __launch_bounds__(kThreads, NB == 1 ? 1 : KB == 4 ? 2 : 3) void adapter_up_kernel(AdapterArgs a) {
  constexpr int kRow = 32 * KB + 8;  // 16-bit elements of a token's row, 16 bytes more than the products need
  __shared__ uint4 high[16 * NB * kRow / 8], low[16 * NB * kRow / 8];
  __shared__ float factor[16 * NB];
  int gi = 0;
  while (gi + 1 < a.count && (int)blockIdx.x >= a.linear[gi + 1].first) ++gi;
  const Linear& l = a.linear[gi];
  const int64_t m_begin = (int64_t)((int)blockIdx.x - l.first) * a.chunks * kColumns;
  const int64_t m_end = m_begin + a.chunks * kColumns < l.m ? m_begin + a.chunks * kColumns : l.m;
  const int64_t t0 = (int64_t)(blockIdx.y / a.slots) * kTile;
  each_group(a, t0, blockIdx.y % a.slots, l.out != l.y, [&](const Group& g) {
    if (g.adapter < 0) return copy_group(l, g, t0, m_begin, m_end);
    if constexpr (NB > 1) {
      if (g.size <= 16) return up_group<BF, KB, 1>(a, l, g, t0, m_begin, m_end, high, low, factor);
    }
    up_group<BF, KB, NB>(a, l, g, t0, m_begin, m_end, high, low, factor);
  });
}

template <bool BF>
auto down_kernel(int blocks, bool many) {
  if (many) return blocks <= 2 ? adapter_down_kernel<BF, 2, true> : adapter_down_kernel<BF, 4, true>;
  return blocks == 1 ? adapter_down_kernel<BF, 1, false> : blocks == 2 ? adapter_down_kernel<BF, 2, false> : adapter_down_kernel<BF, 4, false>;
}
template <bool BF, int NB>
auto up_kernel(int rank) {
  return rank <= 32 ? adapter_up_kernel<BF, 1, NB> : rank <= 64 ? adapter_up_kernel<BF, 2, NB> : adapter_up_kernel<BF, 4, NB>;
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
  int high = 0;
  for (int g = 0; g < count; ++g) high = ranks[g] > high ? ranks[g] : high;
  p.blocks = high > 32 ? 4 : high > 16 || tokens > 16 ? 2 : 1;
  p.runs = 0;
  for (int g = 0; g < count; ++g) p.runs += (ranks[g] + 16 * p.blocks - 1) / (16 * p.blocks);
  const int64_t steps = (n + 255) / 256, groups = p.tiles * (p.slots < 8 ? 1 : p.slots / 2) * p.runs;
  int64_t splits = 1;
  if (p.tiles == 1) splits = (1024 + groups - 1) / groups;
  else while (splits < 8 && groups * splits < (n <= 8192 ? 512 : 256)) splits *= 2;
  splits = splits < steps ? splits : steps;
  splits = splits < 16 ? splits : 16;
  p.steps = (int)((steps + splits - 1) / splits);
  p.splits = (int)((steps + p.steps - 1) / p.steps);
  return p;
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
  return (size_t)plan_of(tokens, n, adapters, count, ranks).splits * tokens * all * sizeof(float);
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
  QS_SUPPORTED(tokens <= (1 << 19) && ldx <= (1 << 24), "%s: %lld rows of %lld, %lld apart", fn, (long long)tokens, (long long)n, (long long)ldx);
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
    a.linear[g] = Linear{static_cast<const uint16_t*>(j.down), static_cast<const uint16_t*>(j.up), j.scale,
                         static_cast<const uint16_t*>(j.y), static_cast<uint16_t*>(j.out), j.down_adapter, j.down_row,
                         j.up_adapter, j.up_row, tokens == 1 ? 0 : j.ldy, tokens == 1 ? 0 : j.ldo, j.m, j.rank, a.ranks, 0, 0};
    a.ranks += j.rank, ranks[g] = j.rank;
    most = j.rank > most ? j.rank : most;
    columns += (j.m + kColumns - 1) / kColumns;
  }
  const Plan p = plan_of(tokens, n, adapters, count, ranks);
  a.slots = p.slots, a.splits = p.splits, a.steps = p.steps;
  const size_t need = (size_t)p.splits * tokens * a.ranks * sizeof(float);
  QS_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "%s: workspace of %zu bytes (16-byte aligned), %zu needed", fn, workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  // a work-group takes several runs of columns where there are tiles enough
  a.chunks = 1;
  const int64_t groups = p.tiles * (p.slots < 8 ? 1 : p.slots / 2);
  while (a.chunks < 8 && groups * columns / (2 * a.chunks) >= 512) a.chunks *= 2;
  int grid = 0, run = 0;
  for (int g = 0; g < count; ++g) {
    a.linear[g].first_run = run;
    run += (ranks[g] + 16 * p.blocks - 1) / (16 * p.blocks);
    a.linear[g].first = grid;
    grid += (int)((a.linear[g].m + (int64_t)a.chunks * kColumns - 1) / ((int64_t)a.chunks * kColumns));
  }
  const bool bf = dtype == QS_DTYPE_BF16;
  const auto down = bf ? down_kernel<true>(p.blocks, tokens > 16) : down_kernel<false>(p.blocks, tokens > 16);
  const unsigned rows = (unsigned)(p.tiles * p.slots);
  hipLaunchKernelGGL(down, dim3((unsigned)(p.runs * p.splits), rows), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("adapter_down_kernel");
  const auto up = tokens <= 16 ? (bf ? up_kernel<true, 1>(most) : up_kernel<false, 1>(most))
                               : (bf ? up_kernel<true, 4>(most) : up_kernel<false, 4>(most));
  hipLaunchKernelGGL(up, dim3((unsigned)grid, rows), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("adapter_up_kernel");
  return QS_OK;
}
