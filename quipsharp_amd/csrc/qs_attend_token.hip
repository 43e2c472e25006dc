// Attention of one new token per row over the row's cache pages
// (qs_attend_token): out[r][h] = sum_p w_p v_p, w = softmax(scale q_h . k_p)
// over the positions p that the token at position lengths[r] - 1 sees.
#include "qs_attend_dev.h"

namespace qs {
namespace {

constexpr int kTile = 32;  // positions of one step of a wave
// Waves of a work-group, whose results meet in LDS.  A few where a row's
// tiles are split over work-groups, many where one work-group takes them all.
constexpr int few_waves(int hd) { return hd == 256 ? 2 : 4; }
constexpr int many_waves(int hd) { return hd == 256 ? 8 : 16; }

struct TokenArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t out_row;
  float* part;
  int heads, kv_heads, splits, window, sinks;
  float scale;    // its size, times log2(e)
  uint32_t flip;  // its sign, for a pair of elements
};

// One work-group per (split, kv head and block of 16 of its heads, row): the
// row's visible tiles are dealt in runs of ceil(tiles / splits), within a run
// wave by wave.
template <bool BF, int HD, int kWavesT, bool NT>
__global__ __launch_bounds__(64 * kWavesT) void attend_token_kernel(PagePool pp, TokenArgs a) {
  typedef WaveAttend<BF, HD, NT> W;
  // the keys at hand, a part for every wave; at the end the waves' results
  union Shared {
    char keys[kWavesT][W::kKeys];
    float Os[kWavesT][16][HD + 4];
  };
  __shared__ __align__(16) Shared sh;
  __shared__ float Ms[kWavesT][16], Ls[kWavesT][16];
  auto& Os = sh.Os;
  const int group = a.heads / a.kv_heads, blocks = (group + 15) / 16;
  const int split = blockIdx.x, g = blockIdx.y / blocks, hb = blockIdx.y % blocks, row = blockIdx.z;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r16 = lane & 15, qd = lane >> 4;
  const LaneX lx = lane_x_init();
  const int most = pp.cols << pp.shift;
  const int len = __builtin_amdgcn_readfirstlane(end_of(pp.lengths, pp.over, most, row));
  const Span s = span_of(len - 1, a.window, a.sinks, most);
  const TileList<kTile> tiles(s);
  const int run = share_tiles(tiles.count, a.splits);
  if (split > 0 && split * run >= tiles.count) return;  // the join does not look for it
  const int u0 = split * run, u1 = u0 + run < tiles.count ? u0 + run : tiles.count;
  const int nh = group - 16 * hb < 16 ? group - 16 * hb : 16;
  const int h0 = g * group + 16 * hb;
  W wv;
  wv.init(pp, sh.keys[w]);
#pragma unroll
  for (int ks = 0; ks < W::KS; ++ks) {
    wv.q[ks] = make_uint4(0, 0, 0, 0);
    if (r16 < nh) wv.q[ks] = flipped(*reinterpret_cast<const uint4*>(a.q + row * a.q_row + (h0 + r16) * a.q_head + 32 * ks + 8 * qd), a.flip);
  }
  typedef const __attribute__((address_space(4))) int32_t* const_t;  // the same for the wave: scalar loads
  const const_t trow = (const_t)(pp.table + row * pp.table_ld);
  auto look_up = [&](int u, int (&e)[2]) {
    const int p0 = kTile * tiles.at(u);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int col = (p0 + 16 * t) >> pp.shift;
      const int x = trow[col < pp.cols ? col : pp.cols - 1];
      e[t] = col < pp.cols && x >= 0 && x < pp.pages ? x : -1;
    }
  };
  int e[2], next[2];
  if (u0 + w < u1) look_up(u0 + w, next);
  for (int u = u0 + w; u < u1; u += kWavesT) {
    const int p0 = kTile * tiles.at(u);
    const bool all = p0 + kTile - 1 <= s.last && (p0 >= s.low || p0 + kTile - 1 < s.sinks);
    e[0] = next[0], e[1] = next[1];
    if (u + kWavesT < u1) look_up(u + kWavesT, next);
    wv.step(pp, e, g, p0, s, all, a.scale, lx);
  }
  // the waves' results together
  const float sum = wv.total(lx);
  __syncthreads();  // other waves' keys lie where the results go
  if (qd == 0) Ms[w][r16] = wv.top, Ls[w][r16] = sum;
#pragma unroll
  for (int j = 0; j < W::DPL; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) Os[w][r16][W::DPL * (4 * qd + i) + j] = wv.o[j][i];
  __syncthreads();
  for (int e = tid; e < nh * HD; e += 64 * kWavesT) {
    const int h = e / HD, d = e % HD;
    float m = Ms[0][h];
#pragma unroll
    for (int i = 1; i < kWavesT; ++i) m = fmaxf(m, Ms[i][h]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int i = 0; i < kWavesT; ++i) {
      const float f = weight(Ms[i][h] - base, a.scale);
      l += f * Ls[i][h], o += f * Os[i][h][d];
    }
    if (a.splits == 1) {
      const float r = l == 0.f ? 0.f : o / l;
      a.out[row * a.out_row + (int64_t)(h0 + h) * HD + d] = (uint16_t)pack16<BF>(r, r);
    } else {
      float* to = a.part + (((int64_t)row * a.heads + h0 + h) * a.splits + split) * part_floats(HD);
      to[kPartHead + d] = o;
      if (d == 0) to[0] = m, to[1] = l;
    }
  }
}

template <int N, typename V>
__device__ __forceinline__ float vec_at(const V& x, int i) {
  if constexpr (N == 1) return x[0];
  else return x[i];
}

// One wave per head of a token: lane i has the weights of splits i, i + 64
// .., and HD / 64 dimensions.
template <bool BF, int HD>
__global__ __launch_bounds__(256) void join_kernel(const float* part, int splits, Used used, int64_t pairs, int heads,
                                                   float scale, uint16_t* out, int64_t out_token) {
  constexpr int N = HD / 64, kAhead = 8;
  typedef float vec __attribute__((ext_vector_type(N)));
  const LaneX lx = lane_x_init();
  const int lane = threadIdx.x & 63;
  const int64_t pair = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (pair >= pairs) return;
  const float* from = part + pair * splits * part_floats(HD);
  // kAhead parts' values at a time, whose loads do not wait for each other
  auto bring = [&](vec (&x)[kAhead], int s) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      x[j] = *reinterpret_cast<const vec*>(from + (int64_t)(s + j < splits ? s + j : splits - 1) * part_floats(HD) + kPartHead + N * lane);
  };
  // the first parts, before it is known how many there are
  vec x[kAhead];
  bring(x, 0);
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < splits) ml = *reinterpret_cast<const float2*>(from + (int64_t)lane * part_floats(HD));
  if (used.lengths) {
    const int len = end_of(used.lengths, used.over, used.most, pair / heads);
    const int count = TileList<kTile>(span_of(len - 1, used.window, used.sinks, used.most)).count, run = share_tiles(count, splits);
    const int there = __builtin_amdgcn_readfirstlane((count + run - 1) / run);
    splits = there < 1 ? 1 : there;
  }
  float top = -INFINITY, sum = 0.f, o[N] = {};
  for (int s0 = 0; s0 < splits; s0 += 64) {
    const int left = splits - s0 < 64 ? splits - s0 : 64;
    if (s0 > 0 && lane < left) ml = *reinterpret_cast<const float2*>(from + (int64_t)(s0 + lane) * part_floats(HD));
    const float m = lane < left ? ml.x : -INFINITY, l = lane < left ? ml.y : 0.f;
    float mx = fmaxf(m, lane_xor<32>(m, lx));
    mx = fmaxf(mx, lane_xor<16>(mx, lx));
    mx = fmaxf(mx, lane_xor<8>(mx, lx));
    mx = fmaxf(mx, lane_xor<4>(mx, lx));
    mx = fmaxf(mx, lane_xor<2>(mx, lx));
    mx = fmaxf(mx, lane_xor<1>(mx, lx));
    mx = fmaxf(mx, top);
    const float base = mx == -INFINITY ? 0.f : mx;
    const float back = weight(top - base, scale), f = weight(m - base, scale);
    top = mx;
    sum = sum * back + wave_sum(f * l, lx);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= back;
    for (int s = 0; s < left; s += kAhead) {
      vec next[kAhead] = {};
      if (s0 + s + kAhead < splits) bring(next, s0 + s + kAhead);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float fj = s + j < left ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s + j)) : 0.f;
        // a part without weight may hold no number where its values do
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fj == 0.f ? o[i] : o[i] + fj * vec_at<N>(x[j], i);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) x[j] = next[j];
    }
  }
  const float r = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* to = out + pair / heads * out_token + pair % heads * HD + N * lane;
  if constexpr (N == 1) {
    *to = (uint16_t)pack16<BF>(o[0] * r, 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(to + i) = pack16<BF>(o[i] * r, o[i + 1] * r);
  }
}

// How many work-groups share a row's tiles, and whether they have many waves.
struct Shares {
  int splits;
  bool many;
};

// A work-group of many waves takes all of a short row in one launch (32 rows
// of up to 577 positions 12.5 us against 16.3 with shares and their join, one
// row 8.0 against 9.2); from about 700 positions on its waves' turns take
// longer than the join (1000: 14.4 against 9.2).  Shares: as many as make 4096
// work-groups, which even out rows of different lengths (48 rows of up to
// 16384: 273 us, with 1024 304), of 8 tiles or more (of 16: 12.4 us instead of
// 10 for one row of 2000).
Shares token_shares(int64_t rows, int heads, int kv_heads, int64_t cols, int page, int window, int sinks) {
  const int64_t wgs = rows * kv_heads * ((heads / kv_heads + 15) / 16);
  const int64_t tiles = seen_positions(cols * page, window, sinks, 0) / kTile + 2;
  if (wgs <= 256 && tiles <= 24) return {1, true};
  int64_t n = (4096 + wgs - 1) / wgs;
  const int64_t most = (tiles + 7) / 8;
  n = n < most ? n : most;
  return {(int)(n < 1 ? 1 : n), false};
}

template <bool BF, int HD>
int launch_token(const PagePool& pp, const TokenArgs& a, int64_t rows, bool many, bool past_caches, hipStream_t stream) {
  const int blocks = (a.heads / a.kv_heads + 15) / 16;
  const dim3 grid((unsigned)a.splits, (unsigned)(a.kv_heads * blocks), (unsigned)rows);
  const dim3 few(64 * few_waves(HD));
  if (many) hipLaunchKernelGGL((attend_token_kernel<BF, HD, many_waves(HD), false>), grid, dim3(64 * many_waves(HD)), 0, stream, pp, a);
  else if (past_caches) hipLaunchKernelGGL((attend_token_kernel<BF, HD, few_waves(HD), true>), grid, few, 0, stream, pp, a);
  else hipLaunchKernelGGL((attend_token_kernel<BF, HD, few_waves(HD), false>), grid, few, 0, stream, pp, a);
  QS_LAUNCHED("attend_token_kernel");
  const Used used{pp.lengths, pp.over, pp.cols << pp.shift, a.window, a.sinks};
  if (a.splits > 1) return join_parts(a.part, a.splits, &used, rows, a.heads, HD, BF, a.scale, a.out, a.out_row, stream);
  return QS_OK;
}

}  // namespace

int join_parts(const float* part, int splits, const Used* there, int64_t tokens, int heads, int head_dim, bool bf, float scale,
               uint16_t* out, int64_t out_token, hipStream_t stream) {
  const int64_t pairs = tokens * heads;
  const Used used = there ? *there : Used{nullptr, nullptr, 0, 0, 0};
  const dim3 grid((unsigned)((pairs + 3) / 4)), block(256);
  if (head_dim == 64) {
    if (bf) hipLaunchKernelGGL((join_kernel<true, 64>), grid, block, 0, stream, part, splits, used, pairs, heads, scale, out, out_token);
    else hipLaunchKernelGGL((join_kernel<false, 64>), grid, block, 0, stream, part, splits, used, pairs, heads, scale, out, out_token);
  } else if (head_dim == 128) {
    if (bf) hipLaunchKernelGGL((join_kernel<true, 128>), grid, block, 0, stream, part, splits, used, pairs, heads, scale, out, out_token);
    else hipLaunchKernelGGL((join_kernel<false, 128>), grid, block, 0, stream, part, splits, used, pairs, heads, scale, out, out_token);
  } else {
    if (bf) hipLaunchKernelGGL((join_kernel<true, 256>), grid, block, 0, stream, part, splits, used, pairs, heads, scale, out, out_token);
    else hipLaunchKernelGGL((join_kernel<false, 256>), grid, block, 0, stream, part, splits, used, pairs, heads, scale, out, out_token);
  }
  QS_LAUNCHED("join_kernel");
  return QS_OK;
}
}  // namespace qs

using namespace qs;

extern "C" size_t qs_attend_token_workspace_bytes(int64_t rows, int heads, int kv_heads, int head_dim, int64_t cols,
                                                  int page, int window, int sinks) {
  if (rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || cols < 1 || page < 1) return 0;
  const int n = token_shares(rows, heads, kv_heads, cols, page, window, sinks).splits;
  return n == 1 ? 0 : (size_t)rows * heads * n * part_floats(head_dim) * sizeof(float);
}

extern "C" int qs_attend_token(const void* q, int dtype, int64_t rows, int heads, int kv_heads, int head_dim,
                               int64_t q_row, int64_t q_head, const qs_page_pool* pool, float scale, int window,
                               int sinks, void* out, int64_t out_row, void* workspace, size_t workspace_bytes,
                               qs_stream_t stream) {
  return qs_attend_token_over(q, dtype, rows, heads, kv_heads, head_dim, q_row, q_head, pool, nullptr, scale, window,
                              sinks, out, out_row, workspace, workspace_bytes, stream);
}

extern "C" int qs_attend_token_over(const void* q, int dtype, int64_t rows, int heads, int kv_heads, int head_dim,
                                    int64_t q_row, int64_t q_head, const qs_page_pool* pool, const int32_t* over,
                                    float scale, int window, int sinks, void* out, int64_t out_row, void* workspace,
                                    size_t workspace_bytes, qs_stream_t stream) {
  if (rows == 0) return QS_OK;
  PagePool pp;
  if (const int rc = page_pool_checks("qs_attend_token", pool, dtype, rows, heads, kv_heads, head_dim, scale, window, sinks, over, pp)) return rc;
  QS_REQUIRE(q && out, "qs_attend_token: null pointer");
  QS_REQUIRE(q_head >= head_dim && q_head % 8 == 0 && q_row >= 0 && q_row % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
             "qs_attend_token: query rows must be 16-byte aligned (strides %lld, %lld)", (long long)q_row, (long long)q_head);
  QS_REQUIRE(out_row >= (int64_t)heads * head_dim && out_row % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
             "qs_attend_token: output rows of %lld elements must be 16-byte aligned", (long long)out_row);
  const size_t need = qs_attend_token_workspace_bytes(rows, heads, kv_heads, head_dim, pool->cols, pool->page, window, sinks);
  QS_REQUIRE(workspace_bytes >= need && (workspace || !need) && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "qs_attend_token: workspace of %zu bytes (16-byte aligned), %zu needed", workspace_bytes, need);
  const Shares sh = token_shares(rows, heads, kv_heads, pool->cols, pool->page, window, sinks);
  TokenArgs a{static_cast<const uint16_t*>(q), q_row, q_head, static_cast<uint16_t*>(out), out_row,
              static_cast<float*>(workspace), heads, kv_heads, sh.splits, window, sinks,
              fabsf(scale) * kLog2E, scale < 0 ? 0x80008000u : 0u};
  // A layer's pages that exceed the chip's 256 MB cache are not found in it by
  // the next call, and values that go past it leave it to the keys: 311 us
  // with, 287 us without over 1.6 GB; where they fit, 26.4 and 27.4 us over
  // 100 MB.
  const bool past_caches = (int64_t)pp.pages * pool->page * kv_heads * head_dim * 4 > (256 << 20);
  const bool bf = dtype == QS_DTYPE_BF16;
  const hipStream_t st = as_stream(stream);
  if (head_dim == 64) return bf ? launch_token<true, 64>(pp, a, rows, sh.many, past_caches, st) : launch_token<false, 64>(pp, a, rows, sh.many, past_caches, st);
  if (head_dim == 128) return bf ? launch_token<true, 128>(pp, a, rows, sh.many, past_caches, st) : launch_token<false, 128>(pp, a, rows, sh.many, past_caches, st);
  return bf ? launch_token<true, 256>(pp, a, rows, sh.many, past_caches, st) : launch_token<false, 256>(pp, a, rows, sh.many, past_caches, st);
}
