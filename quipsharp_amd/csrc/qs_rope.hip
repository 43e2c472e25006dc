// Rotary positions of new tokens with the cache write (qs_page_append_rotated):
// every pair (a, b) of a query or key head's first 2 `pairs` elements becomes
// factor (a cos - b sin, b cos + a sin) at the angle position * frequency, the
// rest of the head stays as it is; queries go to q_out, keys and values to the
// token's place in the pages.
//
// The angle is one product in 64 bits, taken in turns, of which the fraction
// goes on in 32: at position 2^31 it is still right to 2^-21 of a radian, where
// a product in 32 bits would be off by whole turns.  A rotated element is
// rounded once, to the cache's type.
#include "qs_rope_dev.h"
#include "qs_attend_dev.h"
#include "qs_overlap.h"

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kTable = 1024;  // sines and cosines of a work-group: tokens x pairs
constexpr int kTokens = 64;   // of a work-group, at most

struct RotateArgs {
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, tokens;
  const int32_t *starts, *over;
  const double* frequencies;
  float factor;
  int rows, heads, kv_heads, head_dim, pairs;
  int block, lanes;  // tokens of a work-group; log2 of the threads of a head
};

// Where a token stands: its position (below 0: no row has it or it has none),
// the page and the place in it (page -1: it is stored nowhere).
struct Place {
  int64_t pos;
  int page, at;
};

__device__ __forceinline__ Place place_of(const qs_page_pool& pool, const RotateArgs& a, int64_t t, bool* mine) {
  int row = (int)t;
  int64_t back = 1;
  *mine = true;
  if (a.starts) {
    int lo = 0, hi = a.rows;  // the last row that starts at t or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid] <= t) lo = mid; else hi = mid;
    }
    row = lo;
    back = a.starts[row + 1] - t;
    if (a.starts[row] > t || back <= 0) {
      *mine = false;
      return Place{-1, -1, 0};
    }
  }
  int64_t n = pool.lengths[row];
  if (a.over && n == pool.cols * pool.page && a.over[row] > 0) n += a.over[row];
  Place p{n - back, -1, 0};
  if (p.pos >= 0 && p.pos < pool.cols * pool.page) {
    const int id = pool.table[row * pool.table_ld + p.pos / pool.page];
    if (id >= 0 && id < pool.pages) p.page = id, p.at = (int)(p.pos % pool.page);
  }
  return p;
}

template <bool BF>
__device__ __forceinline__ float wide_of(uint32_t u) {
  if constexpr (BF) return __uint_as_float(u << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}

// W elements, in one access.
template <int W>
struct Piece {
  typedef uint32_t type __attribute__((ext_vector_type(W / 2)));
};
template <>
struct Piece<1> {
  typedef uint16_t type;
};
template <int W>
using piece_t = typename Piece<W>::type;
template <int W>
__device__ __forceinline__ piece_t<W> get(const uint16_t* p) {
  return *reinterpret_cast<const piece_t<W>*>(p);
}
template <int W>
__device__ __forceinline__ void put(uint16_t* p, piece_t<W> v) {
  *reinterpret_cast<piece_t<W>*>(p) = v;
}

// a and b of a pair at the angle whose cosine and sine are r.x and r.y, in 16 bits each.
template <bool BF>
__device__ __forceinline__ uint32_t turned(float a, float b, float2 r) {
  return pack16<BF>(__builtin_fmaf(a, r.x, -b * r.y), __builtin_fmaf(b, r.x, a * r.y));
}

// W pairs, of which x and y are the 2 W elements in order: the first elements
// of the pairs and the second ones, or pair by pair.
template <bool BF, bool INTER, int W>
__device__ __forceinline__ void turn(piece_t<W>& x, piece_t<W>& y, const float2* cs) {
  if constexpr (W == 1) {
    const uint32_t o = turned<BF>(wide_of<BF>(x), wide_of<BF>(y), cs[0]);
    x = (uint16_t)o, y = (uint16_t)(o >> 16);
  } else if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      x[i] = turned<BF>(wide_of<BF>(x[i] & 0xFFFF), wide_of<BF>(x[i] >> 16), cs[i]);
      y[i] = turned<BF>(wide_of<BF>(y[i] & 0xFFFF), wide_of<BF>(y[i] >> 16), cs[W / 2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const uint32_t o0 = turned<BF>(wide_of<BF>(x[i] & 0xFFFF), wide_of<BF>(y[i] & 0xFFFF), cs[2 * i]);
      const uint32_t o1 = turned<BF>(wide_of<BF>(x[i] >> 16), wide_of<BF>(y[i] >> 16), cs[2 * i + 1]);
      x[i] = (o0 & 0xFFFF) | o1 << 16, y[i] = o0 >> 16 | (o1 & 0xFFFF0000u);
    }
  }
}

// A work-group has up to 64 tokens, whose places and angles (a table of up to
// 1024 sines and cosines in LDS, so that no head takes them again) come first,
// then their heads, dealt over gridDim.y where tokens are few; 2^lanes threads
// have a head, in accesses of W elements: 16 bytes where pairs and rest allow.
// Memory bounds it: 8192 tokens of 32 + 2 x 8 heads of 128 take 34 us (201 MB,
// 5.9 TB/s, some of it from the caches; 48 us with cold ones), 5394 tokens of 28 +
// 2 x 4 heads 19 us (99 MB, 5.2 TB/s); 48 single tokens 4.6 us, a chain of lookups,
// sines and the heads.
template <bool BF, bool INTER, int W>
__global__ __launch_bounds__(kThreads) void append_rotated_kernel(qs_page_pool pool, RotateArgs a) {
  __shared__ float2 table[kTable];
  __shared__ Place places[kTokens];
  __shared__ bool ours[kTokens];
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * a.block;
  const int n = a.tokens - t0 < a.block ? (int)(a.tokens - t0) : a.block;
  for (int i = tid; i < n; i += kThreads) {
    bool mine;
    places[i] = place_of(pool, a, t0 + i, &mine);
    ours[i] = mine;
  }
  __syncthreads();
  for (int i = tid; i < n * a.pairs; i += kThreads) {
    const double turns = (double)places[i / a.pairs].pos * a.frequencies[i % a.pairs] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    table[i] = make_float2(c * a.factor, s * a.factor);
  }
  __syncthreads();
  const int per = (a.head_dim - a.pairs * 2) / W + a.pairs / W;  // units of a turned head
  const int all = a.heads + 2 * a.kv_heads;
  // heads of this work-group: every gridDim.y-th, 2^lanes threads a head
  const int mine = (all - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y;
  const int step = kThreads >> a.lanes, pieces = a.pairs / W;
  int b = 0, i = tid >> a.lanes;
  for (;; i += step) {
    while (i >= mine) i -= mine, ++b;
    if (b >= n) break;
    if (!ours[b]) continue;
    const int h = i * (int)gridDim.y + (int)blockIdx.y;
    const Place p = places[b];
    const int64_t t = t0 + b;
    // the head's source and destination, and what is done on the way
    const bool query = h < a.heads, key = !query && h < a.heads + a.kv_heads;
    if (!query && p.page < 0) continue;
    const int g = query ? h : key ? h - a.heads : h - a.heads - a.kv_heads;
    const uint16_t* from = query ? a.q + t * a.q_token + g * a.q_head : key ? a.k + t * a.k_token + g * a.k_head : a.v + t * a.v_token + g * a.v_head;
    uint16_t* to = query ? a.q_out + t * a.out_token + (int64_t)g * a.head_dim
                   : key ? static_cast<uint16_t*>(pool.k) + p.page * pool.k_page + g * pool.k_head + p.at * pool.k_pos
                         : static_cast<uint16_t*>(pool.v) + p.page * pool.v_page + g * pool.v_head + p.at * pool.v_pos;
    const bool nothing = p.pos < 0;  // zero queries
    for (int u = tid & ((1 << a.lanes) - 1); u < per; u += 1 << a.lanes) {
      if (u < pieces) {
        // both are read before either is written, so queries may be turned in place
        const int at0 = INTER ? 2 * u * W : u * W, at1 = INTER ? 2 * u * W + W : u * W + a.pairs;
        piece_t<W> x = get<W>(from + at0), y = get<W>(from + at1);
        if (query || key) turn<BF, INTER, W>(x, y, table + b * a.pairs + u * W);
        if (nothing) x = piece_t<W>{}, y = piece_t<W>{};
        put<W>(to + at0, x), put<W>(to + at1, y);
      } else {
        const int at = 2 * a.pairs + (u - pieces) * W;
        piece_t<W> x = get<W>(from + at);
        if (nothing) x = piece_t<W>{};
        put<W>(to + at, x);
      }
    }
  }
}

template <bool BF, bool INTER>
auto rotated_kernel(int w) {
  return w == 8 ? append_rotated_kernel<BF, INTER, 8> : w == 4 ? append_rotated_kernel<BF, INTER, 4> : append_rotated_kernel<BF, INTER, 1>;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" int qs_page_append_rotated(const void* q, const void* k, const void* v, int dtype, int64_t tokens, int64_t rows,
                                      int heads, int kv_heads, int head_dim, int64_t q_token, int64_t q_head,
                                      int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                      const int32_t* starts, const qs_page_pool* pool, const int32_t* over,
                                      const double* frequencies, int pairs, int interleaved, float factor, void* q_out,
                                      int64_t out_token, qs_stream_t stream) {
  const char* fn = "qs_page_append_rotated";
  if (tokens == 0 || rows == 0) return QS_OK;
  QS_REQUIRE(q && k && v && q_out && frequencies && pool && pool->k && pool->v && pool->table && pool->lengths, "%s: null pointer", fn);
  QS_REQUIRE(dtype == QS_DTYPE_F16 || dtype == QS_DTYPE_BF16, "%s: dtype %d", fn, dtype);
  QS_REQUIRE(tokens >= 1 && tokens <= INT32_MAX && rows >= 1 && rows <= (1 << 20) && (starts || tokens == rows),
             "%s: %lld tokens of %lld rows", fn, (long long)tokens, (long long)rows);
  QS_REQUIRE(heads >= 1 && heads <= 65535 && kv_heads >= 1 && kv_heads <= 65535 && head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 4096,
             "%s: %d and %d heads of %d", fn, heads, kv_heads, head_dim);
  QS_REQUIRE(pairs >= 1 && 2 * pairs <= head_dim && pairs <= kMaxPairs, "%s: %d pairs of a head of %d (at most %d)", fn, pairs, head_dim, kMaxPairs);
  QS_REQUIRE(pool->pages >= 1 && pool->pages <= INT32_MAX && pool->page >= 1 && pool->cols >= 1 && pool->table_ld >= pool->cols &&
                 pool->cols * pool->page <= INT32_MAX,
             "%s: %lld pages of %d, table of %lld columns", fn, (long long)pool->pages, pool->page, (long long)pool->cols);
  const int64_t st[13] = {q_token, q_head, k_token, k_head, v_token, v_head, out_token, pool->k_page, pool->k_head, pool->k_pos, pool->v_page, pool->v_head, pool->v_pos};
  for (int64_t x : st) QS_REQUIRE(x >= 0 && x % 8 == 0, "%s: strides must be multiples of 8 elements, got %lld", fn, (long long)x);
  QS_REQUIRE(tokens == 1 || out_token >= (int64_t)heads * head_dim, "%s: rows of q_out %lld apart for %d heads of %d", fn, (long long)out_token, heads, head_dim);
  const void* ptr[6] = {q, k, v, q_out, pool->k, pool->v};
  for (const void* p : ptr) QS_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "%s: tensors must be 16-byte aligned", fn);
  QS_REQUIRE((reinterpret_cast<uintptr_t>(frequencies) & 7) == 0, "%s: frequencies must be 8-byte aligned", fn);
  const int all = heads + 2 * kv_heads;
  QS_SUPPORTED((int64_t)all * head_dim <= (1 << 24), "%s: %d heads of %d", fn, all, head_dim);
  // Queries may be turned where they lie, each element by the thread that reads it.
  const Rows to{q_out, tokens, 2 * out_token, 2 * (int64_t)heads * head_dim};
  auto meets = [&](const void* p, int64_t token, int64_t head, int count) {
    if (!share_memory(to, Rows{p, tokens, 2 * token, 2 * ((count - 1) * head + head_dim)})) return false;
    for (int h = 0; h < count; ++h)
      if (share_memory(to, Rows{static_cast<const uint16_t*>(p) + h * head, tokens, 2 * token, 2 * (int64_t)head_dim})) return true;
    return false;
  };
  const bool in_place = q == q_out && (tokens == 1 || q_token == out_token) && (heads == 1 || q_head == head_dim);
  QS_REQUIRE((in_place || !meets(q, q_token, q_head, heads)) && !meets(k, k_token, k_head, kv_heads) && !meets(v, v_token, v_head, kv_heads),
             "%s: q_out shares memory with q, k or v, and is not q itself", fn);
  int block = kTable / pairs < kTokens ? kTable / pairs : kTokens;
  while (block > 1 && (tokens < 512 * (int64_t)block || (int64_t)block * all * head_dim > (1 << 30))) block /= 2;
  const int64_t blocks = (tokens + block - 1) / block;
  QS_SUPPORTED(blocks < (1ll << 32) / kThreads, "%s: %lld tokens, %d of a work-group", fn, (long long)tokens, block);  // 2^32 threads
  int split = 1;
  while (split * 4 <= all && blocks * split < 512) split *= 2;
  const int rest = head_dim - 2 * pairs;
  const int w = pairs % 8 == 0 && rest % 8 == 0 ? 8 : pairs % 4 == 0 && rest % 4 == 0 ? 4 : 1;
  const int per = rest / w + pairs / w;
  int lanes = 0;
  while (lanes < 8 && 1 << lanes < per) ++lanes;
  const RotateArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                     static_cast<uint16_t*>(q_out), q_token, q_head, k_token, k_head, v_token, v_head, out_token, tokens,
                     starts, over, frequencies, factor, (int)rows, heads, kv_heads, head_dim, pairs, block, lanes};
  const auto kernel = dtype == QS_DTYPE_BF16 ? (interleaved ? rotated_kernel<true, true>(w) : rotated_kernel<true, false>(w))
                                             : (interleaved ? rotated_kernel<false, true>(w) : rotated_kernel<false, false>(w));
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)split), dim3(kThreads), 0, as_stream(stream), *pool, a);
  QS_LAUNCHED("append_rotated_kernel");
  return QS_OK;
}
