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

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kTable = 1024;  // sines and cosines of a work-group: tokens x pairs

struct RotateArgs {
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, tokens;
  const int32_t *starts, *over;
  const double* frequencies;
  float factor;
  int rows, heads, kv_heads, head_dim, pairs, block;  // block: tokens of a work-group
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
__device__ __forceinline__ float wide_of(uint16_t u) {
  if constexpr (BF) return __uint_as_float((uint32_t)u << 16);
  else return (float)__builtin_bit_cast(_Float16, u);
}

// W elements from one place (W 16-bit words, aligned to their size where that is a power of two).
template <int W>
struct Words {
  uint16_t w[W];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (W == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (W == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = p[i];
  }
  __device__ __forceinline__ void store(uint16_t* p) const {
    if constexpr (W == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
    else if constexpr (W == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(w);
    else
#pragma unroll
      for (int i = 0; i < W; ++i) p[i] = w[i];
  }
};

// One unit of a head: W pairs turned, or W elements copied.  A thread reads all
// of a unit before it writes it, so queries may be turned in place.
template <bool BF, bool INTER, int W>
__device__ __forceinline__ void turn_unit(const uint16_t* from, uint16_t* to, int u, int pairs, const float2* cs) {
  Words<W> x, y;
  const int n = pairs / W;
  if (u >= n) {
    const int at = 2 * pairs + (u - n) * W;
    x.load(from + at);
    x.store(to + at);
    return;
  }
  const int i = u * W;
  const int p0 = INTER ? 2 * i : i, p1 = INTER ? 2 * i + W : i + pairs;
  x.load(from + p0), y.load(from + p1);
#pragma unroll
  for (int e = 0; e < W; ++e) {
    // interleaved: pair e is elements 2 e and 2 e + 1 of the 2 W
    uint16_t* pa = INTER ? (2 * e < W ? &x.w[2 * e] : &y.w[2 * e - W]) : &x.w[e];
    uint16_t* pb = INTER ? (2 * e + 1 < W ? &x.w[2 * e + 1] : &y.w[2 * e + 1 - W]) : &y.w[e];
    const float a = wide_of<BF>(*pa), b = wide_of<BF>(*pb);
    const float2 r = cs[i + e];
    const uint32_t o = pack16<BF>(__builtin_fmaf(a, r.x, -b * r.y), __builtin_fmaf(b, r.x, a * r.y));
    *pa = (uint16_t)o, *pb = (uint16_t)(o >> 16);
  }
  x.store(to + p0), y.store(to + p1);
}

template <bool BF, bool INTER, int W>
__global__ __launch_bounds__(kThreads) void append_rotated_kernel(qs_page_pool pool, RotateArgs a) {
  __shared__ float2 table[kTable];
  __shared__ Place places[kTable];
  __shared__ bool ours[kTable];
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
  // heads of this work-group: every gridDim.y-th
  const int mine = (all - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y;
  const int units = n * mine * per;
  for (int i = tid; i < units; i += kThreads) {
    const int u = i % per, h = i / per % mine * (int)gridDim.y + (int)blockIdx.y, b = i / per / mine;
    if (!ours[b]) continue;
    const Place p = places[b];
    const int64_t t = t0 + b;
    if (h < a.heads) {
      uint16_t* to = a.q_out + t * a.out_token + (int64_t)h * a.head_dim;
      if (p.pos >= 0) {
        turn_unit<BF, INTER, W>(a.q + t * a.q_token + h * a.q_head, to, u, a.pairs, table + b * a.pairs);
      } else {
        const Words<W> zero{};
        const int m = a.pairs / W;
        if (u >= m) {
          zero.store(to + 2 * a.pairs + (u - m) * W);
        } else {
          zero.store(to + (INTER ? 2 * u * W : u * W));
          zero.store(to + (INTER ? 2 * u * W + W : u * W + a.pairs));
        }
      }
    } else if (p.page >= 0) {
      const int g = h - a.heads;
      if (g < a.kv_heads) {
        uint16_t* to = static_cast<uint16_t*>(pool.k) + p.page * pool.k_page + g * pool.k_head + p.at * pool.k_pos;
        turn_unit<BF, INTER, W>(a.k + t * a.k_token + g * a.k_head, to, u, a.pairs, table + b * a.pairs);
      } else {
        const int gv = g - a.kv_heads;
        uint16_t* to = static_cast<uint16_t*>(pool.v) + p.page * pool.v_page + gv * pool.v_head + p.at * pool.v_pos;
        const uint16_t* from = a.v + t * a.v_token + gv * a.v_head;
        const int m = a.pairs / W;
        Words<W> x;
        if (u >= m) {
          x.load(from + 2 * a.pairs + (u - m) * W), x.store(to + 2 * a.pairs + (u - m) * W);
        } else {
          x.load(from + 2 * u * W), x.store(to + 2 * u * W);
          x.load(from + 2 * u * W + W), x.store(to + 2 * u * W + W);
        }
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
  int block = kTable / pairs;
  while (block > 1 && (tokens < 512 * (int64_t)block || (int64_t)block * all * head_dim > (1 << 30))) block /= 2;
  const int64_t blocks = (tokens + block - 1) / block;
  int split = 1;
  while (split * 4 <= all && blocks * split < 512) split *= 2;
  const int rest = head_dim - 2 * pairs;
  const int w = pairs % 8 == 0 && rest % 8 == 0 ? 8 : pairs % 4 == 0 && rest % 4 == 0 ? 4 : 1;
  const RotateArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                     static_cast<uint16_t*>(q_out), q_token, q_head, k_token, k_head, v_token, v_head, out_token, tokens,
                     starts, over, frequencies, factor, (int)rows, heads, kv_heads, head_dim, pairs, block};
  const auto kernel = dtype == QS_DTYPE_BF16 ? (interleaved ? rotated_kernel<true, true>(w) : rotated_kernel<true, false>(w))
                                             : (interleaved ? rotated_kernel<false, true>(w) : rotated_kernel<false, false>(w));
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)split), dim3(kThreads), 0, as_stream(stream), *pool, a);
  QS_LAUNCHED("append_rotated_kernel");
  return QS_OK;
}
