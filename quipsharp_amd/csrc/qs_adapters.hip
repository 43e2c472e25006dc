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
  int first;         // its first work-group column of the second launch
  int wide;          // y and out take 16-byte accesses
};

struct AdapterArgs {
  const uint16_t* x;
  int64_t ldx, tokens, n;
  const int32_t* which;
  int adapters, count, ranks;  // ranks: of all linears together
  int splits, steps;           // steps of 256 inputs of a split
  int slots, chunks;           // work-groups that share a tile's groups; runs of kColumns of a work-group
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
    if (nth % a.slots != slot) continue;
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

// One group of the first launch: NB blocks of 16 tokens, RB of 16 ranks.
template <bool BF, int RB, int NB>
__device__ __forceinline__ void down_group(const AdapterArgs& a, const Linear& l, const Group& g, int64_t t0, int split,
                                           f32x4 (*sums)[NB][64]) {
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, q = lane >> 4, r = lane & 15;
  const uint16_t* rows[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) rows[b] = a.x + (t0 + place_in_tile(g, 16 * b + r)) * a.ldx;
  const uint16_t* down = l.down + g.adapter * l.down_adapter;
  f32x4 acc[RB][NB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t k0 = (int64_t)split * a.steps * 256, k1 = k0 + a.steps * 256 < a.n ? k0 + a.steps * 256 : a.n;
  // 64 inputs at a time: a lane's 16 lie together, 8 for each of two products
  for (int64_t k = k0 + 64 * w; k < k1; k += 256) {
    uint4 av[RB][2], xv[NB][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t at = k + 16 * q + 8 * j;
      const bool in = at < k1;
#pragma unroll
      for (int i = 0; i < RB; ++i)
        av[i][j] = in && 16 * i + r < l.rank ? *reinterpret_cast<const uint4*>(down + (16 * i + r) * l.down_row + at) : uint4{};
#pragma unroll
      for (int b = 0; b < NB; ++b) xv[b][j] = in ? *reinterpret_cast<const uint4*>(rows[b] + at) : uint4{};
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[i][b] = mma_16x16x32<BF>(av[i][j], xv[b][j], acc[i][b]);
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) {
#pragma unroll
    for (int b = 0; b < NB; ++b) sums[w][b][lane] = acc[i][b];
    __syncthreads();
    for (int e = tid; e < NB * 64; e += kThreads) {
      const int b = e >> 6, c = 16 * b + (e & 15), rank = 16 * i + 4 * (e >> 4 & 3);
      const f32x4 s = (sums[0][b][e & 63] + sums[1][b][e & 63]) + (sums[2][b][e & 63] + sums[3][b][e & 63]);
      // all lanes take part in the exchange; e is a multiple of 64 and the lane
      const int place = place_in_tile(g, c);
      if (c < g.size && rank < l.rank)
        *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.tokens + t0 + place) * a.ranks + l.offset + rank) = s;
    }
    __syncthreads();
  }
}

template <bool BF, int RB, int NB>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterArgs a) {
  __shared__ f32x4 sums[4][NB][64];
  const Linear& l = a.linear[blockIdx.x / a.splits];
  const int split = blockIdx.x % a.splits;
  const int64_t t0 = (int64_t)(blockIdx.y / a.slots) * kTile;
  each_group(a, t0, blockIdx.y % a.slots, false, [&](const Group& g) {
    if constexpr (NB > 1) {
      if (g.size <= 16) return down_group<BF, RB, 1>(a, l, g, t0, split, reinterpret_cast<f32x4(*)[1][64]>(&sums[0][0][0]));
    }
    down_group<BF, RB, NB>(a, l, g, t0, split, sums);
  });
}

template <bool BF>
__device__ __forceinline__ float float_of(uint32_t u) {
  if constexpr (BF) return __uint_as_float(u << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}

// 16 columns of a token: y + scale * d in 16-byte pieces.
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

// The second launch: a group's tokens against 64 columns a wave at a time.
template <bool BF, int KB>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterArgs a) {
  constexpr int R = 32 * KB, kRow = R + 8;  // 16-bit elements of a token's row, 16 bytes further than the products need
  __shared__ uint4 high[kTile * kRow / 8], low[kTile * kRow / 8];
  __shared__ float factor[kTile];
  __shared__ int token[kTile];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, q = lane >> 4, r = lane & 15;
  int gi = 0;
  while (gi + 1 < a.count && (int)blockIdx.x >= a.linear[gi + 1].first) ++gi;
  const Linear& l = a.linear[gi];
  const int64_t m_begin = (int64_t)((int)blockIdx.x - l.first) * a.chunks * kColumns;
  const int64_t m_end = m_begin + a.chunks * kColumns < l.m ? m_begin + a.chunks * kColumns : l.m;
  const int64_t t0 = (int64_t)(blockIdx.y / a.slots) * kTile;
  each_group(a, t0, blockIdx.y % a.slots, l.out != l.y, [&](const Group& g) {
    if (g.adapter < 0) {
      for (int c = w; c < g.size; c += 4) {
        const int64_t t = t0 + place_in_tile(g, c);
        for (int64_t m = m_begin + lane; m < m_end; m += 64) l.out[t * l.ldo + m] = l.y[t * l.ldy + m];
      }
      return;
    }
    __syncthreads();  // the group before is done with the tables
    {
      // four threads a token: its products, summed over the splits, each its quarter of the ranks
      const int c = tid >> 2, j = tid & 3;
      const int place = place_in_tile(g, c);
      float v[R / 4], most = 0.f;
#pragma unroll
      for (int i = 0; i < R / 4; i += 4) {
        f32x4 s{0.f, 0.f, 0.f, 0.f};
        const int rank = j * (R / 4) + i;
        if (c < g.size && rank < l.rank)
          for (int p = 0; p < a.splits; ++p)
            s += *reinterpret_cast<const f32x4*>(a.part + ((int64_t)p * a.tokens + t0 + place) * a.ranks + l.offset + rank);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i + e] = s[e], most = fmaxf(most, fabsf(s[e]));
      }
      most = fmaxf(most, __shfl_xor(most, 1));
      most = fmaxf(most, __shfl_xor(most, 2));
      int e = (int)(__float_as_uint(most) >> 23);
      e = e < 2 ? 2 : e > 252 ? 252 : e;
      const float shrink = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
      for (int i = 0; i < R / 4; i += 8) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float f0 = v[i + 2 * x] * shrink, f1 = v[i + 2 * x + 1] * shrink;
          hi[x] = pack16<BF>(f0, f1);
          const float h0 = float_of<BF>(hi[x] & 0xFFFF), h1 = float_of<BF>(hi[x] >> 16);
          // an infinite product has no remainder
          lo[x] = pack16<BF>(fabsf(h0) < INFINITY ? f0 - h0 : 0.f, fabsf(h1) < INFINITY ? f1 - h1 : 0.f);
        }
        const int at = (c * kRow + j * (R / 4) + i) / 8;
        high[at] = make_uint4(hi[0], hi[1], hi[2], hi[3]), low[at] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      if (j == 0) factor[c] = __uint_as_float((uint32_t)e << 23) * l.scale[g.adapter], token[c] = place;
    }
    __syncthreads();
    const uint16_t* up = l.up + g.adapter * l.up_adapter;
    const int blocks = (g.size + 15) / 16;
    for (int64_t m0 = m_begin + 64 * w; m0 < m_end; m0 += kColumns) {
      uint4 wv[4][KB];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int64_t m = m0 + 16 * (r >> 2) + 4 * j + (r & 3);
        m = m < l.m ? m : l.m - 1;
#pragma unroll
        for (int k = 0; k < KB; ++k)
          wv[j][k] = 32 * k + 8 * q < l.rank ? *reinterpret_cast<const uint4*>(up + m * l.up_row + 32 * k + 8 * q) : uint4{};
      }
      const int64_t m = m0 + 16 * q;
      for (int b = 0; b < blocks; ++b) {
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
        if (c < g.size && m < l.m) {
          const int64_t t = t0 + token[c];
          const float scale = factor[c];
          const uint16_t* from = l.y + t * l.ldy + m;
          uint16_t* to = l.out + t * l.ldo + m;
          if (l.wide && m + 16 <= l.m) {
            const uint4 y0 = *reinterpret_cast<const uint4*>(from), y1 = *reinterpret_cast<const uint4*>(from + 8);
            *reinterpret_cast<uint4*>(to) = add_8<BF>(y0, acc[0], acc[1], scale);
            *reinterpret_cast<uint4*>(to + 8) = add_8<BF>(y1, acc[2], acc[3], scale);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (m + i < l.m) to[i] = (uint16_t)pack16<BF>(__builtin_fmaf(acc[i >> 2][i & 3], scale, float_of<BF>(from[i])), 0.f);
          }
        }
      }
    }
  });
}

template <bool BF, int NB>
auto down_kernel(int rank) {
  return rank <= 16 ? adapter_down_kernel<BF, 1, NB> : rank <= 32 ? adapter_down_kernel<BF, 2, NB>
         : rank <= 64 ? adapter_down_kernel<BF, 4, NB> : adapter_down_kernel<BF, 8, NB>;
}
template <bool BF>
auto up_kernel(int rank) {
  return rank <= 32 ? adapter_up_kernel<BF, 1> : rank <= 64 ? adapter_up_kernel<BF, 2> : adapter_up_kernel<BF, 4>;
}

struct Plan {
  int64_t tiles;
  int slots, splits, steps;
};

Plan plan_of(int64_t tokens, int64_t n, int64_t adapters, int count) {
  Plan p;
  p.tiles = (tokens + kTile - 1) / kTile;
  const int64_t most = tokens < kTile ? tokens : kTile, share = 64 / p.tiles > 4 ? 64 / p.tiles : 4;
  int64_t slots = most < share ? most : share;
  slots = slots < adapters + 1 ? slots : adapters + 1;
  p.slots = (int)slots;
  const int64_t steps = (n + 255) / 256, groups = p.tiles * (p.slots < 8 ? 1 : p.slots / 2) * count;
  int64_t splits = (1024 + groups - 1) / groups;
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
  return (size_t)plan_of(tokens, n, adapters, count).splits * tokens * all * sizeof(float);
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
  QS_SUPPORTED(tokens <= (1 << 19) && n <= (1 << 24), "%s: %lld rows of %lld", fn, (long long)tokens, (long long)n);
  AdapterArgs a{};
  a.x = static_cast<const uint16_t*>(x), a.ldx = tokens == 1 ? 0 : ldx, a.tokens = tokens, a.n = n, a.which = which;
  a.adapters = (int)adapters, a.count = count;
  int most = 0;
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
    QS_REQUIRE(((reinterpret_cast<uintptr_t>(j.y) | reinterpret_cast<uintptr_t>(j.out)) & 1) == 0 && (reinterpret_cast<uintptr_t>(j.scale) & 3) == 0,
               "%s: linear %d: tensors must be aligned to their elements", fn, g);
    QS_REQUIRE(j.y != j.out || tokens == 1 || j.ldy == j.ldo, "%s: linear %d: y and out share memory with rows %lld and %lld apart", fn, g,
               (long long)j.ldy, (long long)j.ldo);
    const bool wide = ((reinterpret_cast<uintptr_t>(j.y) | reinterpret_cast<uintptr_t>(j.out)) & 15) == 0 && (j.ldy | j.ldo) % 8 == 0;
    a.linear[g] = Linear{static_cast<const uint16_t*>(j.down), static_cast<const uint16_t*>(j.up), j.scale,
                         static_cast<const uint16_t*>(j.y), static_cast<uint16_t*>(j.out), j.down_adapter, j.down_row,
                         j.up_adapter, j.up_row, tokens == 1 ? 0 : j.ldy, tokens == 1 ? 0 : j.ldo, j.m, j.rank, a.ranks, 0, wide};
    a.ranks += j.rank;
    most = j.rank > most ? j.rank : most;
    columns += (j.m + kColumns - 1) / kColumns;
  }
  const Plan p = plan_of(tokens, n, adapters, count);
  a.slots = p.slots, a.splits = p.splits, a.steps = p.steps;
  const size_t need = (size_t)p.splits * tokens * a.ranks * sizeof(float);
  QS_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "%s: workspace of %zu bytes (16-byte aligned), %zu needed", fn, workspace_bytes, need);
  a.part = static_cast<float*>(workspace);
  // a work-group takes several runs of columns where there are tiles enough
  a.chunks = 1;
  while (a.chunks < 8 && p.tiles * columns / (2 * a.chunks) >= 2048) a.chunks *= 2;
  int grid = 0;
  for (int g = 0; g < count; ++g) {
    a.linear[g].first = grid;
    grid += (int)((a.linear[g].m + (int64_t)a.chunks * kColumns - 1) / ((int64_t)a.chunks * kColumns));
  }
  const bool bf = dtype == QS_DTYPE_BF16;
  const auto down = tokens <= 16 ? (bf ? down_kernel<true, 1>(most) : down_kernel<false, 1>(most))
                                 : (bf ? down_kernel<true, 4>(most) : down_kernel<false, 4>(most));
  const unsigned rows = (unsigned)(p.tiles * p.slots);
  hipLaunchKernelGGL(down, dim3((unsigned)(count * p.splits), rows), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("adapter_down_kernel");
  const auto up = bf ? up_kernel<true>(most) : up_kernel<false>(most);
  hipLaunchKernelGGL(up, dim3((unsigned)grid, rows), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("adapter_up_kernel");
  return QS_OK;
}
