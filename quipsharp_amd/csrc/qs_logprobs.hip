// Log probabilities of given tokens with entropy, rank and the best
// alternatives (qs_token_logprobs).  With m the row's largest logit and S = sum
// exp(x - m):
//
//   log p_t = x_t - m - log S
//   H       = log S - sum exp(x - m) (x - m) / S
//   rank    = #{j : x_j > x_t, or x_j = x_t and j < t}
//
// in one pass over the logits.  A thread keeps a level near the maximum of what
// it has seen, and both sums below it; they are turned to a new level when the
// maximum rises more than 1 above the old one, and joined at the end.
// Alternatives go by the logits alone, which no arithmetic touches.
//
// Exponentials are fp32, eight of a kind are added in fp32, and all else is
// fp64.  With units of 2^-24: a term D below its level is off by 2.25 D + 2 (the
// difference, log2(e), the product and the exponential), a turn adds D + 2, of
// which those after the first count for little (a sum is a third or less of
// itself after each), and there are two joins; eight added make 7.  The mean of
// D over a softmax is at most ln(vocab), so that a log sum is off by
// 3 ln(vocab) + 20 units (3.3e-6 for 151936 tokens) at most.
#include <type_traits>

#include "qs_order_dev.h"

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 64;
constexpr int kMaxParts = 128;  // of a row: its lists fit the join's room
constexpr int kGroup = 32;      // logits of a thread that have one maximum noted
constexpr int kRuns = 20;       // groups of a thread
constexpr int kListed = 256;    // groups that may be read again together
// Candidates at a time: above the exact edge there are fewer than 64 groups,
// and of those at it fewer than 64 are taken.
constexpr int kRoom = (kMaxTop - 1) * kGroup + kMaxTop;
static_assert(kRoom >= kMaxTop * (kMaxParts * kMaxTop / kThreads), "candidates of the join");
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Of a part of a row: its level, both sums below it and how many are ahead of
// the token; the token's logit (+inf where it is none), the same in all parts.
struct Stat {
  double sum, weighted;
  float top;
  int ahead;
  float xt;
};

struct ScoreArgs {
  const void* logits;
  int64_t ld, vocab;
  const void* tokens;
  int wide_tokens;  // int64
  int top, parts, slices, per;  // per: slices of a part
  Stat* stats;      // [rows][parts]
  uint64_t* lists;  // [rows][parts][top]: order bits << 32 | ~token, in descending order; 0 for none
  float *logp, *entropy, *top_logp;
  int32_t *ranks, *top_tokens;
};

// exp(d)
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504f); }

// Sums below the level `from` turned to the larger `to`.
__device__ __forceinline__ void turn(double& sum, double& weighted, float from, float to) {
  if (from == -INFINITY || !(from < to)) return;
  const double d = (double)from - (double)to;
  const double r = d < -200.0 ? 0.0 : (double)__builtin_amdgcn_exp2f((float)(d * 1.4426950408889634));
  weighted = r == 0.0 ? 0.0 : r * (weighted + d * sum);
  sum *= r;
}

__device__ __forceinline__ float wave_max(float v, LaneX lx) {
  v = fmaxf(v, lane_xor<32>(v, lx));
  v = fmaxf(v, lane_xor<16>(v, lx));
  v = fmaxf(v, lane_xor<8>(v, lx));
  v = fmaxf(v, lane_xor<4>(v, lx));
  v = fmaxf(v, lane_xor<2>(v, lx));
  v = fmaxf(v, lane_xor<1>(v, lx));
  return v;
}

template <typename T>
__device__ __forceinline__ float value_of(const T* row, int64_t t) {
  float f;
  if constexpr (sizeof(T) == 4) f = row[t];
  else if constexpr (std::is_same<T, _Float16>::value) f = (float)row[t];
  else f = __uint_as_float((uint32_t)row[t] << 16);
  return fmaxf(f, -INFINITY);  // NaN counts as -inf
}

__device__ __forceinline__ int64_t token_of(const ScoreArgs& a, int64_t row) {
  const int64_t t = a.wide_tokens ? static_cast<const int64_t*>(a.tokens)[row] : static_cast<const int32_t*>(a.tokens)[row];
  return t >= 0 && t < a.vocab ? t : -1;
}

// What is written for a row, from its level and sums: one thread.
__device__ __forceinline__ void write_row(const ScoreArgs& a, int64_t row, bool none, const Stat& s, double log_sum) {
  const bool runs = fabsf(s.top) < INFINITY;
  a.logp[row] = none ? 0.f : runs ? (float)(((double)s.xt - s.top) - log_sum) : -INFINITY;
  a.entropy[row] = runs ? (float)fmax(0.0, log_sum - s.weighted / s.sum) : 0.f;
  a.ranks[row] = none ? -1 : s.ahead;
}
__device__ __forceinline__ void write_alternative(const ScoreArgs& a, int64_t row, int i, uint64_t key, float top, double log_sum) {
  const bool has = key && fabsf(top) < INFINITY;
  a.top_logp[row * a.top + i] = has ? (float)(((double)order_float((uint32_t)(key >> 32)) - top) - log_sum) : -INFINITY;
  a.top_tokens[row * a.top + i] = has ? (int32_t)~(uint32_t)key : -1;
}

// Leaves the best `top` of n > top candidates, no two of which are alike, at
// the front of room: their least is found two at a time of the bits in which
// candidates differ, and no further than it takes to tell it from the next.
constexpr int kCounts = 97;  // three for every two bits, and one
__device__ void narrow(uint64_t* room, int n, int top, int* above) {
  constexpr int kEach = (kRoom + kThreads - 1) / kThreads;
  __shared__ uint64_t some[4], all[4];
  const int tid = threadIdx.x, w = tid >> 6;
  uint64_t mine[kEach], any = 0, every = ~0ull;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool is = i * kThreads + tid < n;
    mine[i] = is ? room[i * kThreads + tid] : 0;
    any |= mine[i], every &= is ? mine[i] : ~0ull;
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) any |= __shfl_xor(any, x), every &= __shfl_xor(every, x);
  if ((tid & 63) == 0) some[w] = any, all[w] = every;
  if (tid < kCounts) above[tid] = 0;
  __syncthreads();
  uint64_t least = all[0] & all[1] & all[2] & all[3], open = (some[0] | some[1] | some[2] | some[3]) & ~least;
  for (int* counts = above; open; counts += 3) {
    const uint64_t one = 1ull << (63 - __builtin_clzll(open));
    open &= ~one;
    const uint64_t two = open ? 1ull << (63 - __builtin_clzll(open)) : 0;
    open &= ~two;
    const uint64_t at[3] = {least | two, least | one, least | one | two};
    int many[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i * kThreads < n)
#pragma unroll
        for (int k = 0; k < 3; ++k) many[k] += __popcll(__ballot(mine[i] >= at[k]));
    if ((tid & 63) == 0)
#pragma unroll
      for (int k = 0; k < 3; ++k) atomicAdd(&counts[k], many[k]);
    __syncthreads();
    int have = 0;
#pragma unroll
    for (int k = 2; k >= 0; --k)
      if (!have && counts[k] >= top) have = counts[k], least = at[k];
    if (have == top) break;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (i * kThreads + tid < n && mine[i] >= least) room[atomicAdd(&above[kCounts - 1], 1)] = mine[i];
  __syncthreads();
}

// The best `top` of the first n candidates, in order, in best; zeros behind
// them.  More than kFew are narrowed first (2040 equal logits, 64 wanted: 12
// us in all, by their ranks alone 100).
constexpr int kFew = 192;
__device__ __forceinline__ void rank_all(uint64_t* room, int n, uint64_t* best, int top, int* above) {
  if (n > kFew) narrow(room, n, top, above), n = top;
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const uint64_t me = room[c];
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) place += room[i] > me;
    if (place < top) best[place] = me;
  }
  for (int c = n + threadIdx.x; c < top; c += kThreads) best[c] = 0;
}

// The maximum of a thread's group, in as few bytes as hold it.
template <typename T>
struct Note {
  typedef T type;
  __device__ __forceinline__ static type of(float f) { return (T)f; }
  __device__ __forceinline__ static float value(type t) { return (float)t; }
};
template <>
struct Note<uint16_t> {
  typedef uint16_t type;
  __device__ __forceinline__ static type of(float f) { return (uint16_t)(__float_as_uint(f) >> 16); }
  __device__ __forceinline__ static float value(type t) { return __uint_as_float((uint32_t)t << 16); }
};

// The W logits of a 16-byte piece.
template <typename T, int W = 16 / sizeof(T)>
__device__ __forceinline__ void unpack(const u32x4& u, float* x) {
#pragma unroll
  for (int e = 0; e < W; ++e) {
    if constexpr (sizeof(T) == 4) x[e] = __uint_as_float(u[e]);
    else if constexpr (std::is_same<T, _Float16>::value) x[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[e / 2] >> 16 * (e & 1)));
    else x[e] = __uint_as_float(e & 1 ? u[e / 2] & 0xFFFF0000u : u[e / 2] << 16);
    x[e] = fmaxf(x[e], -INFINITY);  // NaN counts as -inf
  }
}

// A part of a row as the selection of its best sees it: pieces of 16 bytes,
// piece (run * pieces + i) * 256 + thread is the i-th of the thread's group `run`.
template <typename T, int P>
struct Groups {
  static constexpr int W = 16 / sizeof(T);
  const u32x4* pieces;
  int64_t first, end, vocab;  // the part's first piece, elements of the row from the first piece on
  int lead, runs, limit;      // limit: pieces of the part for each thread (the last group may have fewer)
  const typename Note<T>::type* notes;

  // Calls use(logit, token) for the logits of a piece.
  template <typename F>
  __device__ __forceinline__ void each(int run, int i, int thread, F use) const {
    const int64_t at = first + ((int64_t)run * P + i) * kThreads + thread;
    if (run * P + i >= limit || at * W >= end) return;
    float x[W];
    unpack<T>(pieces[at], x);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int64_t token = at * W + e - lead;
      if (token >= 0 && token < vocab) use(x[e], (uint32_t)token);
    }
  }
};

struct Room {
  uint64_t keys[kRoom], best[kMaxTop];
  uint16_t listed[kListed];
  float red[4][4];
  int above[kCounts];  // of a search bit by bit
  int groups, count, sums[4];
};

__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) { return (uint64_t)order_bits(x) << 32 | (uint32_t)~token; }

// The best `top` of a part, in order, into r.best; zeros behind them.  The
// thread's largest logit is `largest`.  At least `top` groups have a maximum
// that is not below the edge, the largest of the waves' top-th largest
// maxima of threads or the least of their top / 4-th, and the best lie in groups
// of which that is so: those are read again.  (In a part of fewer pieces than
// threads, of which waves have nothing: the second of their top / 2-th or the third
// of their top / 3-th; 64 alternatives of 8 rows of 21818 24 us without, 9 so.)  Where they or their logits at
// the edge are too many, it is the top-th largest maximum of the groups: the
// logits above it lie in fewer than `top` groups, and of those at it the lowest
// tokens are taken.
//
// `own`: the part is one slice, which the threads still have: held(use) calls
// use(logit, token) for the thread's.
template <typename T, int P, typename Held>
__device__ __forceinline__ void select_best(const Groups<T, P>& g, float largest, int top, Room& r, bool own, Held held) {
  typedef Note<T> N;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const uint32_t bits = order_bits(largest);
  const float edge_w = order_float(nth_key(bits, top)), part_w = top > 8 ? order_float(nth_key(bits, (top + 3) / 4)) : -INFINITY;
  const bool sparse = top > 8 && g.end - g.first * Groups<T, P>::W < kThreads * Groups<T, P>::W;
  if (lane == 0) r.red[0][w] = edge_w, r.red[1][w] = part_w;
  if (sparse) {
    const float half = order_float(nth_key(bits, (top + 1) / 2)), third = order_float(nth_key(bits, (top + 2) / 3));
    if (lane == 0) r.red[2][w] = half, r.red[3][w] = third;
  }
  if (tid == 0) r.groups = 0, r.count = 0;
  __syncthreads();
  float edge = fmaxf(fmaxf(r.red[0][0], r.red[0][1]), fmaxf(r.red[0][2], r.red[0][3]));
  edge = fmaxf(edge, fminf(fminf(r.red[1][0], r.red[1][1]), fminf(r.red[1][2], r.red[1][3])));
  if (sparse) {
    auto inner = [&](const float (&v)[4], float& second, float& third) {
      const float h0 = fmaxf(v[0], v[1]), l0 = fminf(v[0], v[1]), h1 = fmaxf(v[2], v[3]), l1 = fminf(v[2], v[3]);
      second = fmaxf(fminf(h0, h1), fmaxf(l0, l1)), third = fminf(fmaxf(l0, l1), fminf(h0, h1));
    };
    float half, third, other;
    inner(r.red[2], half, other), inner(r.red[3], other, third);
    edge = fmaxf(edge, fmaxf(half, third));
  }
  auto add = [&](float x, uint32_t token) {
    const int at = atomicAdd(&r.count, 1);
    if (at < kRoom) r.keys[at] = key_of(x, token);
  };
  auto list = [&](auto wanted) {
    for (int s = 0; s < g.runs; ++s) {
      const float m = N::value(g.notes[s * kThreads + tid]);
      if (wanted(m) && m > -INFINITY) {
        const int at = atomicAdd(&r.groups, 1);
        if (at < kListed) r.listed[at] = (uint16_t)(s * kThreads + tid);
      }
    }
  };
  auto read = [&](int n, auto wanted) {
    for (int u = tid; u < n * P; u += kThreads) {
      const int at = r.listed[u / P];
      g.each(at / kThreads, u % P, at % kThreads, [&](float x, uint32_t token) {
        if (wanted(x) && x > -INFINITY) add(x, token);
      });
    }
  };
  int groups = 0;
  if (own) {
    if (__any(largest >= edge)) {
      held([&](float x, uint32_t token) {
        if (x >= edge && x > -INFINITY) add(x, token);
      });
    }
  } else {
    if (largest >= edge) list([&](float m) { return m >= edge; });
    __syncthreads();
    groups = r.groups;
    if (groups <= kListed) read(groups, [&](float x) { return x >= edge; });
  }
  __syncthreads();
  int n = r.count;
  if (groups > kListed || n > kRoom) {
    __syncthreads();
    if (tid < 32) r.above[tid] = 0;
    if (tid == 0) r.groups = 0, r.count = 0;
    __syncthreads();
    list([&](float m) { return m > edge; });
    __syncthreads();
    groups = r.groups;
    if (groups >= top) {
      // the edge is too low
      uint32_t u = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t v = u | 1u << bit;
        int many = 0;
        for (int s = 0; s < g.runs; ++s) many += __popcll(__ballot(order_bits(N::value(g.notes[s * kThreads + tid])) >= v));
        if (lane == 0) atomicAdd(&r.above[bit], many);
        __syncthreads();
        if (r.above[bit] >= top) u = v;
      }
      edge = order_float(u);
      if (tid == 0) r.groups = 0;
      __syncthreads();
      list([&](float m) { return m > edge; });
      __syncthreads();
      groups = r.groups;
    }
    read(groups, [&](float x) { return x > edge; });
    __syncthreads();
    n = r.count;
    __syncthreads();
    for (int s = 0; s < g.runs * P && n < top; ++s) {
      const int run = s / P, i = s % P;
      const bool mine = N::value(g.notes[run * kThreads + tid]) >= edge;
      int equal = 0;
      if (mine) g.each(run, i, tid, [&](float x, uint32_t) { equal += x == edge; });
      // how many there are before this thread's
      int before = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint64_t have = __ballot(equal >> b & 1);
        before += __popcll(have & ((1ull << lane) - 1)) << b;
        if (lane == 0) r.sums[w] = (b ? r.sums[w] : 0) + (__popcll(have) << b);
      }
      __syncthreads();
      for (int x = 0; x < w; ++x) before += r.sums[x];
      const int all = (r.sums[0] + r.sums[1]) + (r.sums[2] + r.sums[3]);
      if (equal) {
        g.each(run, i, tid, [&](float x, uint32_t token) {
          if (x == edge) {
            if (n + before < top) r.keys[n + before] = key_of(x, token);
            ++before;
          }
        });
      }
      n = n + all < top ? n + all : top;
      __syncthreads();
    }
  }
  rank_all(r.keys, n, r.best, top, r.above);
  __syncthreads();
}

// One work-group per part of a row.  A row is read in 16-byte pieces that
// begin at or before its first logit, so rows at odd places load as widely as
// others: piece i * 256 + tid of a slice is the thread's i-th.  H slices make
// a group, whose maxima the threads note in LDS: the best are found from those,
// and a few groups are read again.  (Candidates picked slice by slice, as beam
// selection has them, took 184 us where 1500 rows of 151936 take 104.)
//
// Memory and the vector instructions of the exponentials bound long rows: 1500
// rows of 151936 bf16 with ten alternatives 104 us (456 MB, 4.4 TB/s; 101 with
// none), 2047 of 32000 fp32 with none 45 us (262 MB, 5.8 TB/s).  Few rows are
// bound by the chain behind the loads: 48 of 151936 fp32 with 20, in 19 parts
// each, take 17 us and the join 7, for 29 MB; one row of bf16 with five 6 and 6.
template <typename T, int E, bool SELECT>
__global__ __launch_bounds__(kThreads) void score_kernel(ScoreArgs a) {
  constexpr int W = 16 / sizeof(T), P = E / W, H = kGroup / E;
  typedef Note<T> N;
  __shared__ typename std::conditional<SELECT, Room, int>::type room;
  __shared__ typename N::type notes[SELECT ? kRuns * kThreads : 1];
  __shared__ float red[4];
  __shared__ Stat stat[4];
  const LaneX lx = lane_x_init();
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, part = blockIdx.y, top = a.top;
  const int64_t row = blockIdx.x;
  const T* from = static_cast<const T*>(a.logits) + row * a.ld;
  const int lead = (int)((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
  const u32x4* pieces = reinterpret_cast<const u32x4*>(from - lead);
  const int64_t end = lead + a.vocab;  // elements from the first piece on
  const int first = part * a.per, last = first + a.per < a.slices ? first + a.per : a.slices;

  auto fetch = [&](int slice, u32x4 (&raw)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int64_t at = ((int64_t)slice * P + i) * kThreads + tid;
      raw[i] = at * W < end ? __builtin_nontemporal_load(pieces + at) : u32x4{};
    }
  };
  u32x4 raw[P];
  fetch(first, raw);
  const int64_t t = token_of(a, row);
  const float xt = t < 0 ? INFINITY : value_of(from, t);
  float x[E], m = -INFINITY, largest = -INFINITY, noted = -INFINITY;
  double sum = 0.0, weighted = 0.0;
  int ahead = 0;
  for (int slice = first; slice < last; ++slice) {
    const int64_t e0 = (int64_t)slice * (P * kThreads * W);  // the slice's first element
    auto token = [&](int i) { return e0 + ((int64_t)(i / W) * kThreads + tid) * W + i % W - lead; };
#pragma unroll
    for (int i = 0; i < P; ++i) unpack<T>(raw[i], x + i * W);
    if (e0 < lead || e0 + E * kThreads > end) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (token(i) < 0 || token(i) >= a.vocab) x[i] = -INFINITY;
    }
    if (slice + 1 < last) fetch(slice + 1, raw);
    float ms = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) ms = fmaxf(ms, x[i]);
    if (ms > m + 1.f) turn(sum, weighted, m, ms), m = ms;
    if (m > -INFINITY) {
#pragma unroll
      for (int i = 0; i < E; i += 8) {
        float s = 0.f, v = 0.f;
#pragma unroll
        for (int e = i; e < i + 8; ++e) {
          const float d = fmaxf(x[e] - m, -200.f), p = exp_of(d);
          s += p, v = __builtin_fmaf(p, d, v);
        }
        sum += s, weighted += v;
      }
    }
    // how many are ahead of the token: at or above it before its place, above it behind
    if (t >= 0) {
      const int64_t t0 = e0 - lead, t1 = t0 + E * kThreads;
      if (t1 <= t && xt > -INFINITY) {
#pragma unroll
        for (int i = 0; i < E; ++i) ahead += __popcll(__ballot(x[i] >= xt));
      } else if (t0 > t) {
#pragma unroll
        for (int i = 0; i < E; ++i) ahead += __popcll(__ballot(x[i] > xt));
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
          ahead += __popcll(__ballot(x[i] > xt || (x[i] == xt && token(i) >= 0 && token(i) < t)));
      }
    }
    if constexpr (SELECT) {
      largest = fmaxf(largest, ms);
      noted = fmaxf(noted, ms);
      const int k = slice - first;
      if (k % H == H - 1 || slice + 1 == last) notes[k / H * kThreads + tid] = N::of(noted), noted = -INFINITY;
    }
  }
  // the threads' sums below the highest level
  float all = wave_max(m, lx);
  if (lane == 0) red[w] = all;
  __syncthreads();
  all = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (all < INFINITY) turn(sum, weighted, m, all);
  sum = wave_sum64(sum, lx), weighted = wave_sum64(weighted, lx);
  if (lane == 0) stat[w] = Stat{sum, weighted, all, ahead, xt};
  if constexpr (SELECT) {
    const Groups<T, kGroup / W> g{pieces, (int64_t)first * P * kThreads, end, a.vocab, lead, (last - first + H - 1) / H, (last - first) * P, notes};
    select_best(g, largest, top, room, last - first == 1, [&](auto use) {
#pragma unroll
      for (int i = 0; i < E; ++i) use(x[i], (uint32_t)(((int64_t)first * P + i / W) * (kThreads * W) + tid * W + i % W - lead));
    });
  } else {
    __syncthreads();
  }
  const Stat s{(stat[0].sum + stat[1].sum) + (stat[2].sum + stat[3].sum),
               (stat[0].weighted + stat[1].weighted) + (stat[2].weighted + stat[3].weighted), all,
               t < 0 ? -1 : (stat[0].ahead + stat[1].ahead) + (stat[2].ahead + stat[3].ahead), xt};
  if (a.parts > 1) {
    if (tid == 0) a.stats[row * a.parts + part] = s;
    if constexpr (SELECT)
      if (tid < top) a.lists[(row * a.parts + part) * top + tid] = room.best[tid];
    return;
  }
  const double log_sum = log(s.sum);
  if (tid == 0) write_row(a, row, t < 0, s, log_sum);
  if constexpr (SELECT)
    if (tid < top) write_alternative(a, row, tid, room.best[tid], all, log_sum);
}

// The parts of a row together: one work-group per row.  LONG: lists of more than
// 32 (64 alternatives of 48 rows in 19 parts: 8 us, 21 without it; 20
// alternatives 6.9, with it 7.4).
template <bool LONG>
__global__ __launch_bounds__(kThreads) void score_join_kernel(ScoreArgs a) {
  __shared__ uint64_t room[kRoom];
  __shared__ uint64_t best[kMaxTop], tops[kThreads], line;
  __shared__ uint32_t edge[4], share[4];
  __shared__ Stat stat;
  __shared__ int count, above[kCounts];
  const LaneX lx = lane_x_init();
  const int tid = threadIdx.x, top = a.top;
  const int64_t row = blockIdx.x;
  const int n = a.parts * top;
  const uint64_t* lists = a.lists + row * n;
  uint64_t mine[kMaxParts * kMaxTop / kThreads];
  uint64_t high = 0;
  // Long lists: their first entries, then their second ones, and so on, dealt to
  // the waves in turn, or the threads' maxima would tell little.
  int part = 0, place = 0;
  if (LONG) {
    const int c = 4 * (tid & 63) + (tid >> 6);
    part = c % a.parts, place = c / a.parts;
  }
#pragma unroll
  for (int i = 0; i < kMaxParts * kMaxTop / kThreads; ++i) {
    int c = i * kThreads + tid;
    if (LONG) {
      c = place < top ? part * top + place : n;
      part += kThreads % a.parts, place += kThreads / a.parts;
      if (part >= a.parts) part -= a.parts, ++place;
    }
    mine[i] = c < n ? lists[c] : 0;
    high = mine[i] > high ? mine[i] : high;
  }
  tops[tid] = high;
  if (tid == 0) count = 0, line = 0;
  if (top > 0) {
    const uint32_t bits = (uint32_t)(high >> 32), e = nth_key(bits, top), s = LONG ? nth_key(bits, (top + 3) / 4) : 0;
    if ((tid & 63) == 0) edge[tid >> 6] = e, share[tid >> 6] = s;
  }
  if (tid < 64) {
    const Stat* st = a.stats + row * a.parts;
    const Stat none{0.0, 0.0, -INFINITY, 0, 0.f};
    Stat s = tid < a.parts ? st[tid] : none, s2 = tid + 64 < a.parts ? st[tid + 64] : none;
    // a part counts -1 where the token is none
    const float all = wave_max(fmaxf(s.top, s2.top), lx);
    if (all < INFINITY) turn(s.sum, s.weighted, s.top, all), turn(s2.sum, s2.weighted, s2.top, all);
    const double sum = wave_sum64(s.sum + s2.sum, lx), weighted = wave_sum64(s.weighted + s2.weighted, lx);
    const double ahead = wave_sum64((double)s.ahead + s2.ahead, lx);
    if (tid == 0) stat = Stat{sum, weighted, all, s.ahead < 0 ? -1 : (int)ahead, s.xt};
  }
  __syncthreads();
  if (top > 0) {
    // at least `top` threads of a wave, or a fourth of that in every wave, have a
    // candidate whose logit is not below the edge
    auto take = [&](uint64_t least) {
#pragma unroll
      for (int i = 0; i < kMaxParts * kMaxTop / kThreads; ++i)
        if (mine[i] && mine[i] >= least) {
          const int at = atomicAdd(&count, 1);
          if (at < kRoom) room[at] = mine[i];
        }
    };
    const uint32_t whole = max(max(edge[0], edge[1]), max(edge[2], edge[3])), fourths = min(min(share[0], share[1]), min(share[2], share[3]));
    if (high) take((uint64_t)max(whole, fourths) << 32);
    __syncthreads();
    int many = count;
    if (many > kRoom) {
      // equal logits: no two candidates are alike, so that at most `top` threads have one at or above this edge
      __syncthreads();
      if (tid == 0) count = 0;
      int higher = 0;
#pragma unroll 8
      for (int i = 0; i < kThreads; ++i) higher += tops[i] > high;
      if (higher == top - 1) line = high;
      __syncthreads();
      take(line);
      __syncthreads();
      many = count;
    }
    rank_all(room, many, best, top, above);
    __syncthreads();
  }
  const double log_sum = log(stat.sum);
  if (tid == 0) write_row(a, row, stat.ahead < 0, stat, log_sum);
  if (tid < top) write_alternative(a, row, tid, best[tid], stat.top, log_sum);
}

struct Layout {
  int each, slices, per, parts;
  size_t lists, bytes;
};

// Logits of a thread at a time: 32 where rows are long and there are many
// (1500 rows of 151936 bf16, ten alternatives: 104 us, with 16 108), 16 where
// they make fewer than eight slices of it (6000 rows of 32000, five: 108 us, with 32
// 115), 8 where there are few, for more work-groups.
Layout layout_of(int64_t rows, int64_t vocab, int top, int size) {
  Layout l;
  l.each = rows * ((vocab + 8191) / 8192) < 512 ? 8 : vocab < 8 * 8192 ? 16 : 32;
  const int64_t slice = (int64_t)kThreads * l.each;
  l.slices = (int)((vocab + 16 / size - 1 + slice - 1) / slice);  // wherever the row begins in its first piece
  int64_t parts = (1024 + rows - 1) / rows;
  const int64_t room = (int64_t)kRuns * (kGroup / l.each), least = (l.slices + room - 1) / room;
  parts = parts < l.slices ? parts : l.slices;
  parts = parts < kMaxParts ? parts : kMaxParts;
  parts = parts > least ? parts : least;
  l.per = (int)((l.slices + parts - 1) / parts);
  l.parts = (l.slices + l.per - 1) / l.per;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  l.lists = l.parts > 1 ? up((size_t)rows * l.parts * sizeof(Stat)) : 0;
  l.bytes = l.parts > 1 ? l.lists + up((size_t)rows * l.parts * top * sizeof(uint64_t)) : 0;
  return l;
}

template <typename T, bool SELECT>
auto score_kernel_of(int each) {
  return each == 32 ? score_kernel<T, 32, SELECT> : each == 16 ? score_kernel<T, 16, SELECT> : score_kernel<T, 8, SELECT>;
}
template <typename T>
auto score_kernel_of(int each, bool select) {
  return select ? score_kernel_of<T, true>(each) : score_kernel_of<T, false>(each);
}

// A grid has fewer than 2^32 threads along each side.
constexpr int64_t kMaxRows = (1ll << 32) / kThreads - 1;

bool sizes_fit(int64_t rows, int64_t vocab, int top) {
  return rows >= 1 && rows <= kMaxRows && vocab >= 1 && vocab <= (1 << 24) && top >= 0 && top <= kMaxTop && top <= vocab;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int dtype, int top) {
  if (!sizes_fit(rows, vocab, top)) return 0;
  return layout_of(rows, vocab, top, dtype == QS_DTYPE_F32 ? 4 : 2).bytes;
}

extern "C" size_t qs_token_logprobs_workspace_most(int64_t rows, int64_t vocab, int dtype, int top) {
  if (!sizes_fit(rows, vocab, top)) return 0;
  // from 1024 rows on a row has as many parts whatever their number
  const int size = dtype == QS_DTYPE_F32 ? 4 : 2;
  size_t most = layout_of(rows, vocab, top, size).bytes;
  for (int64_t r = 1; r < rows && r < 1024; ++r) {
    const size_t bytes = layout_of(r, vocab, top, size).bytes;
    most = bytes > most ? bytes : most;
  }
  return most;
}

extern "C" int qs_token_logprobs(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab, const void* tokens,
                                 int token_bytes, int top, float* logprobs, float* entropy, int32_t* ranks,
                                 float* top_logprobs, int32_t* top_tokens, void* workspace, size_t workspace_bytes,
                                 qs_stream_t stream) {
  const char* fn = "qs_token_logprobs";
  if (rows == 0) return QS_OK;
  QS_REQUIRE(logits && tokens && logprobs && entropy && ranks && (top == 0 || (top_logprobs && top_tokens)), "%s: null pointer", fn);
  QS_REQUIRE(dtype == QS_DTYPE_F32 || dtype == QS_DTYPE_F16 || dtype == QS_DTYPE_BF16, "%s: dtype %d", fn, dtype);
  QS_REQUIRE(token_bytes == 4 || token_bytes == 8, "%s: tokens of %d bytes", fn, token_bytes);
  QS_REQUIRE(rows >= 1 && vocab >= 1 && (rows == 1 || ld >= vocab), "%s: %lld rows of %lld tokens, %lld apart", fn,
             (long long)rows, (long long)vocab, (long long)ld);
  QS_REQUIRE(top >= 0 && top <= vocab, "%s: %d alternatives of %lld tokens", fn, top, (long long)vocab);
  QS_SUPPORTED(sizes_fit(rows, vocab, top), "%s: %lld rows of %lld tokens, %d alternatives (at most %d, of 2^24 tokens, of %lld rows)", fn,
               (long long)rows, (long long)vocab, top, kMaxTop, (long long)kMaxRows);
  const int size = dtype_bytes(dtype);
  QS_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0 && reinterpret_cast<uintptr_t>(tokens) % token_bytes == 0,
             "%s: logits and tokens must be aligned to their elements", fn);
  const Layout l = layout_of(rows, vocab, top, size);
  QS_REQUIRE(l.bytes == 0 || (workspace && workspace_bytes >= l.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
             "%s: workspace of %zu bytes (16-byte aligned), %zu needed", fn, workspace_bytes, l.bytes);
  char* ws = static_cast<char*>(workspace);
  const ScoreArgs a{logits, rows == 1 ? vocab : ld, vocab, tokens, token_bytes == 8, top, l.parts, l.slices, l.per,
                    reinterpret_cast<Stat*>(ws), reinterpret_cast<uint64_t*>(ws + l.lists), logprobs, entropy,
                    top_logprobs, ranks, top_tokens};
  const auto kernel = dtype == QS_DTYPE_F32   ? score_kernel_of<float>(l.each, top > 0)
                      : dtype == QS_DTYPE_F16 ? score_kernel_of<_Float16>(l.each, top > 0)
                                              : score_kernel_of<uint16_t>(l.each, top > 0);
  hipLaunchKernelGGL(kernel, dim3((unsigned)rows, (unsigned)l.parts), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("score_kernel");
  if (l.parts > 1) {
    const auto join = top > 32 ? score_join_kernel<true> : score_join_kernel<false>;
    hipLaunchKernelGGL(join, dim3((unsigned)rows), dim3(kThreads), 0, as_stream(stream), a);
    QS_LAUNCHED("score_join_kernel");
  }
  return QS_OK;
}
