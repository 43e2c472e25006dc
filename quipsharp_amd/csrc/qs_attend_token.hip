// Attention of one new token per row over the row's cache pages
// (qs_attend_token): out[r][h] = sum_p w_p v_p, w = softmax(scale q_h . k_p)
// over the positions p that the token at position lengths[r] - 1 sees.
#include "qs_attend_dev.h"

namespace qs {
namespace {

constexpr int kTile = 32;  // positions of one step of a wave
// waves of a work-group: their results meet in LDS, 64 KB at most
constexpr int waves_of(int hd) { return hd == 256 ? 2 : 4; }

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
template <bool BF, int HD>
__global__ __launch_bounds__(64 * waves_of(HD)) void attend_token_kernel(PagePool pp, TokenArgs a) {
  typedef WaveAttend<BF, HD> W;
  constexpr int kWavesT = waves_of(HD);
  __shared__ float Os[kWavesT][16][HD + 4];
  __shared__ float Ms[kWavesT][16], Ls[kWavesT][16];
  const int group = a.heads / a.kv_heads, blocks = (group + 15) / 16;
  const int split = blockIdx.x, g = blockIdx.y / blocks, hb = blockIdx.y % blocks, row = blockIdx.z;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r16 = lane & 15, qd = lane >> 4;
  const LaneX lx = lane_x_init();
  int len = pp.lengths[row];
  const int64_t most = (int64_t)pp.cols << pp.shift;
  len = len > most ? (int)most : len;
  const Span s = span_of(len - 1, a.window, a.sinks);
  const TileList<kTile> tiles(s);
  const int run = (tiles.count + a.splits - 1) / a.splits;
  const int u0 = split * run, u1 = u0 + run < tiles.count ? u0 + run : tiles.count;
  const int nh = group - 16 * hb < 16 ? group - 16 * hb : 16;
  const int h0 = g * group + 16 * hb;
  W wv;
  wv.init();
#pragma unroll
  for (int ks = 0; ks < W::KS; ++ks) {
    wv.q[ks] = make_uint4(0, 0, 0, 0);
    if (r16 < nh) wv.q[ks] = flipped(*reinterpret_cast<const uint4*>(a.q + row * a.q_row + (h0 + r16) * a.q_head + 32 * ks + 8 * qd), a.flip);
  }
  const int32_t* trow = pp.table + row * pp.table_ld;
  for (int u = u0 + w; u < u1; u += kWavesT) {
    const int p0 = kTile * tiles.at(u);
    const bool all = p0 + kTile - 1 <= s.last && (p0 >= s.low || p0 + kTile - 1 < s.sinks);
    wv.step(pp, trow, g, p0, s, all, a.scale, lx);
  }
  // the waves' results together
  const float sum = wv.total(lx);
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
      float* to = a.part + (((int64_t)row * a.heads + h0 + h) * a.splits + split) * (HD + 2);
      to[2 + d] = o;
      if (d == 0) to[0] = m, to[1] = l;
    }
  }
}

// The splits' results of one head together.
template <bool BF, int HD>
__global__ __launch_bounds__(HD) void attend_join_kernel(TokenArgs a) {
  const int h = blockIdx.x, row = blockIdx.y, d = threadIdx.x;
  const float* from = a.part + ((int64_t)row * a.heads + h) * a.splits * (HD + 2);
  float m = -INFINITY;
  for (int i = 0; i < a.splits; ++i) m = fmaxf(m, from[i * (HD + 2)]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f, o = 0.f;
  for (int i = 0; i < a.splits; ++i) {
    const float* p = from + i * (HD + 2);
    const float f = weight(p[0] - base, a.scale);
    l += f * p[1], o += f * p[2 + d];
  }
  const float r = l == 0.f ? 0.f : o / l;
  a.out[row * a.out_row + (int64_t)h * HD + d] = (uint16_t)pack16<BF>(r, r);
}

int token_splits(int64_t rows, int heads, int kv_heads, int64_t cols, int page, int window, int sinks) {
  const int64_t wgs = rows * kv_heads * ((heads / kv_heads + 15) / 16);
  int64_t seen = cols * page;
  if (window > 0 && window + (int64_t)sinks < seen) seen = window + (int64_t)sinks;
  const int64_t tiles = seen / kTile + 2;
  int64_t n = (1024 + wgs - 1) / wgs;
  const int64_t most = (tiles + 3) / 4;
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : n);
}

template <bool BF, int HD>
int launch_token(const PagePool& pp, const TokenArgs& a, int64_t rows, hipStream_t stream) {
  const int blocks = (a.heads / a.kv_heads + 15) / 16;
  hipLaunchKernelGGL((attend_token_kernel<BF, HD>), dim3((unsigned)a.splits, (unsigned)(a.kv_heads * blocks), (unsigned)rows),
                     dim3(64 * waves_of(HD)), 0, stream, pp, a);
  QS_LAUNCHED("attend_token_kernel");
  if (a.splits > 1) {
    hipLaunchKernelGGL((attend_join_kernel<BF, HD>), dim3((unsigned)a.heads, (unsigned)rows), dim3(HD), 0, stream, a);
    QS_LAUNCHED("attend_join_kernel");
  }
  return QS_OK;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_attend_token_workspace_bytes(int64_t rows, int heads, int kv_heads, int head_dim, int64_t cols,
                                                  int page, int window, int sinks) {
  if (rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || cols < 1 || page < 1) return 0;
  const int n = token_splits(rows, heads, kv_heads, cols, page, window, sinks);
  return n == 1 ? 0 : (size_t)rows * heads * n * (head_dim + 2) * sizeof(float);
}

extern "C" int qs_attend_token(const void* q, int dtype, int64_t rows, int heads, int kv_heads, int head_dim,
                               int64_t q_row, int64_t q_head, const qs_page_pool* pool, float scale, int window,
                               int sinks, void* out, int64_t out_row, void* workspace, size_t workspace_bytes,
                               qs_stream_t stream) {
  if (rows == 0) return QS_OK;
  PagePool pp;
  if (const int rc = page_pool_checks("qs_attend_token", pool, dtype, rows, heads, kv_heads, head_dim, scale, window, sinks, pp)) return rc;
  QS_REQUIRE(q && out, "qs_attend_token: null pointer");
  QS_REQUIRE(q_head >= head_dim && q_head % 8 == 0 && q_row >= 0 && q_row % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
             "qs_attend_token: query rows must be 16-byte aligned (strides %lld, %lld)", (long long)q_row, (long long)q_head);
  QS_REQUIRE(out_row >= (int64_t)heads * head_dim && out_row % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
             "qs_attend_token: output rows of %lld elements must be 16-byte aligned", (long long)out_row);
  const size_t need = qs_attend_token_workspace_bytes(rows, heads, kv_heads, head_dim, pool->cols, pool->page, window, sinks);
  QS_REQUIRE(workspace_bytes >= need && (workspace || !need) && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "qs_attend_token: workspace of %zu bytes (16-byte aligned), %zu needed", workspace_bytes, need);
  TokenArgs a{static_cast<const uint16_t*>(q), q_row, q_head, static_cast<uint16_t*>(out), out_row,
              static_cast<float*>(workspace), heads, kv_heads,
              token_splits(rows, heads, kv_heads, pool->cols, pool->page, window, sinks), window, sinks,
              fabsf(scale) * 1.44269504088896340736f, scale < 0 ? 0x80008000u : 0u};
  const bool bf = dtype == QS_DTYPE_BF16;
  const hipStream_t st = as_stream(stream);
  if (head_dim == 64) return bf ? launch_token<true, 64>(pp, a, rows, st) : launch_token<false, 64>(pp, a, rows, st);
  if (head_dim == 128) return bf ? launch_token<true, 128>(pp, a, rows, st) : launch_token<false, 128>(pp, a, rows, st);
  return bf ? launch_token<true, 256>(pp, a, rows, st) : launch_token<false, 256>(pp, a, rows, st);
}
