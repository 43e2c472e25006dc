// Causal attention of several new tokens per row over the row's cache pages
// (qs_attend_chunk).  The tokens of row r are q[starts[r]] .. q[starts[r + 1]
// - 1]; the last of them is at position lengths[r] - 1.
#include <cmath>

#include "qs_attend_dev.h"

namespace qs {
namespace {

constexpr int kTile = 32;
constexpr int kWavesC = 4;
constexpr int kCols = 16 * kWavesC;  // query columns (a head of a token each) of a work-group

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_token, q_head;
  uint16_t* out;
  int64_t out_token;
  const int32_t* starts;
  int64_t tokens;
  int rows, heads, kv_heads, window, sinks;
  float scale;    // its size, times log2(e)
  uint32_t flip;  // its sign, for a pair of elements
};

// One work-group per kv head and 64 columns of a row, column c being head c %
// group of the row's token c / group; one wave per 16 of them.
template <bool BF, int HD>
__global__ __launch_bounds__(64 * kWavesC) void attend_chunk_kernel(PagePool pp, ChunkArgs a) {
  typedef WaveAttend<BF, HD, false> W;
  const int group = a.heads / a.kv_heads, g = blockIdx.y;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r16 = lane & 15, qd = lane >> 4;
  const LaneX lx = lane_x_init();
  // the row and its block of columns
  int64_t b = blockIdx.x, first = 0, count = 0;
  int row = 0;
  for (; row < a.rows; ++row) {
    first = a.starts[row];
    first = first < 0 ? 0 : first > a.tokens ? a.tokens : first;
    const int64_t end = a.starts[row + 1] > a.tokens ? a.tokens : a.starts[row + 1];
    count = end > first ? end - first : 0;
    const int64_t n = (count * group + kCols - 1) / kCols;
    if (b < n) break;
    b -= n;
  }
  if (row == a.rows) return;
  int len = pp.lengths[row];
  const int64_t most = (int64_t)pp.cols << pp.shift;
  len = len > most ? (int)most : len;
  const int64_t c = b * kCols + 16 * w + r16;
  if (b * kCols + 16 * w >= count * group) return;  // a whole wave without columns
  const bool live = c < count * group;
  const int64_t t = live ? c / group : count - 1;
  const int h = g * group + (int)(live ? c % group : 0);
  const int last = len - (int)(count - t);  // may be negative: sees nothing
  const Span s = span_of(last, a.window, a.sinks);
  // the wave's columns together: the first and the last token's spans
  const int64_t c0 = b * kCols + 16 * w, c1 = c0 + 15 < count * group ? c0 + 15 : count * group - 1;
  const Span s0 = span_of(len - (int)(count - c0 / group), a.window, a.sinks);
  const Span s1 = span_of(len - (int)(count - c1 / group), a.window, a.sinks);
  const Span both{s0.low, s1.last, a.window > 0 ? (a.sinks < s0.low ? a.sinks : s0.low) : 0};
  const TileList<kTile> tiles(both);
  W wv;
  wv.init();
  wv.filled = len;
  const uint16_t* qp = a.q + (first + t) * a.q_token + h * a.q_head;
#pragma unroll
  for (int ks = 0; ks < W::KS; ++ks) wv.q[ks] = flipped(*reinterpret_cast<const uint4*>(qp + 32 * ks + 8 * qd), a.flip);
  const int32_t* trow = pp.table + row * pp.table_ld;
  for (int u = 0; u < tiles.count; ++u) {
    const int p0 = kTile * tiles.at(u);
    const bool all = p0 + kTile - 1 <= s0.last && (p0 >= s1.low || p0 + kTile - 1 < s0.sinks);
    wv.step(pp, trow, g, p0, s, all, a.scale, lx);
  }
  const float l = wv.total(lx), r = l == 0.f ? 0.f : 1.f / l;
  if (!live) return;
  uint16_t* to = a.out + (first + t) * a.out_token + (int64_t)h * HD + 4 * W::DPL * qd;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < W::DPL; j += 2)
      *reinterpret_cast<uint32_t*>(to + W::DPL * i + j) = pack16<BF>(wv.o[j][i] * r, wv.o[j + 1][i] * r);
}

template <bool BF, int HD>
int launch_chunk(const PagePool& pp, const ChunkArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.tokens * (a.heads / a.kv_heads) + kCols - 1) / kCols + a.rows;
  hipLaunchKernelGGL((attend_chunk_kernel<BF, HD>), dim3((unsigned)blocks, (unsigned)a.kv_heads), dim3(64 * kWavesC), 0, stream, pp, a);
  QS_LAUNCHED("attend_chunk_kernel");
  return QS_OK;
}

}  // namespace

int page_pool_checks(const char* fn, const qs_page_pool* p, int dtype, int64_t rows, int heads, int kv_heads,
                     int head_dim, float scale, int window, int sinks, PagePool& out) {
  QS_REQUIRE(std::isfinite(scale) && scale != 0.f, "%s: scale %g", fn, (double)scale);
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
  QS_REQUIRE(p->k_pos >= head_dim && p->k_pos <= (1 << 24) && p->v_pos >= head_dim && p->v_pos <= (1 << 24),
             "%s: position strides %lld, %lld", fn, (long long)p->k_pos, (long long)p->v_pos);
  QS_REQUIRE(((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15) == 0,
             "%s: the pools must be 16-byte aligned", fn);
  int shift = 0;
  while ((1 << shift) < p->page) ++shift;
  out = PagePool{static_cast<const uint16_t*>(p->k), static_cast<const uint16_t*>(p->v), p->k_page, p->k_head, p->v_page,
                 p->v_head, (int)p->k_pos, (int)p->v_pos, (int)p->pages, shift, p->table, p->table_ld, (int)p->cols, p->lengths};
  return QS_OK;
}

}  // namespace qs

using namespace qs;

extern "C" int qs_attend_chunk(const void* q, int dtype, int64_t tokens, int64_t rows, int heads, int kv_heads,
                               int head_dim, int64_t q_token, int64_t q_head, const int32_t* starts,
                               const qs_page_pool* pool, float scale, int window, int sinks, void* out,
                               int64_t out_token, qs_stream_t stream) {
  if (tokens == 0 || rows == 0) return QS_OK;
  PagePool pp;
  if (const int rc = page_pool_checks("qs_attend_chunk", pool, dtype, rows, heads, kv_heads, head_dim, scale, window, sinks, pp)) return rc;
  QS_REQUIRE(q && out && starts, "qs_attend_chunk: null pointer");
  QS_REQUIRE(tokens >= 1 && tokens * heads <= INT32_MAX, "qs_attend_chunk: %lld tokens", (long long)tokens);
  QS_REQUIRE(q_head >= head_dim && q_head % 8 == 0 && q_token >= 0 && q_token % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
             "qs_attend_chunk: query rows must be 16-byte aligned (strides %lld, %lld)", (long long)q_token, (long long)q_head);
  QS_REQUIRE(out_token >= (int64_t)heads * head_dim && out_token % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
             "qs_attend_chunk: output rows of %lld elements must be 16-byte aligned", (long long)out_token);
  ChunkArgs a{static_cast<const uint16_t*>(q), q_token, q_head, static_cast<uint16_t*>(out), out_token, starts, tokens,
              (int)rows, heads, kv_heads, window, sinks, fabsf(scale) * 1.44269504088896340736f, scale < 0 ? 0x80008000u : 0u};
  const bool bf = dtype == QS_DTYPE_BF16;
  const hipStream_t st = as_stream(stream);
  if (head_dim == 64) return bf ? launch_chunk<true, 64>(pp, a, st) : launch_chunk<false, 64>(pp, a, st);
  if (head_dim == 128) return bf ? launch_chunk<true, 128>(pp, a, st) : launch_chunk<false, 128>(pp, a, st);
  return bf ? launch_chunk<true, 256>(pp, a, st) : launch_chunk<false, 256>(pp, a, st);
}
