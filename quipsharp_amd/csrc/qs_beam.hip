// Beam search: the best continuations over beams and vocabulary, and the
// states that follow them (qs_beam_select, qs_reorder_states).
//
// A continuation scores s_b + x_t - log sum_t' exp(x_t').  Within a beam the
// order is that of the logits, so one pass over them finds both what the sum
// needs (the running maximum and sum) and each slice's best `keep`; the
// second launch adds the slices' sums and chooses among the slices' bests by
// the score in fp64.
//
// Exponentials are fp32, sixteen of them are added by pairs in fp32, and all
// else is fp64.  With units of 2^-24: a term D below the largest logit is off
// by 2 D + 4 (twice a difference, a product with log2(e) and an exponential:
// to its slice's largest and from there to the beam's), which over a softmax
// of `vocab` terms, whose mean D is ln(vocab) at most, makes 2 ln(vocab) + 4,
// and the pairs 4: a log sum is right to 32 units (2e-6) for 151936 tokens.
#include <type_traits>

#include "qs_chunk_dev.h"

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kJoin = 256;  // threads of the join (selection of 32 requests of 8 beams: 35.4 us, with 512 38, with 1024 41)
constexpr int kMaxKeep = 128;
constexpr int kRoom = 2304;  // candidates of a slice (what lies above the edge, or 128 of it and a row of ties)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Order-preserving bits of a float; -0 counts as 0, NaN as -inf.
__device__ __forceinline__ uint32_t order_bits(float f) {
  f = f != f ? -INFINITY : f + 0.0f;
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_float(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ uint64_t order_bits64(double f) {
  f = f != f ? -INFINITY : f + 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, f);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double order_double(uint64_t u) {
  return __builtin_bit_cast(double, u >> 63 ? u & ~(1ull << 63) : ~u);
}

// Of a slice: its largest logit, and the sum of the exponentials below it.
struct Stat {
  double sum;
  float top;
};

struct SelectArgs {
  const void* logits;
  int64_t ld;
  const float* scores;
  const uint8_t* finished;
  Stat* stats;     // [rows][slices]
  uint64_t* best;  // [rows][slices][keep]: order bits << 32 | ~token, in descending order; 0 for none
  float* scores_out;
  int32_t *parents_out, *tokens_out;
  int64_t eos;
  int beams, vocab, keep, slices, dtype;
};

// exp(x - m) for x <= m, zero where there is nothing yet.  log2(e) in two
// parts: the rounding of one alone would be the same for all terms of a sum.
__device__ __forceinline__ float exp_below(float x, float m) {
  const float d = x - (m == -INFINITY ? 0.f : m);
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, 1.44269502f, d * 1.92596299e-8f));
}

__device__ __forceinline__ double wave_sum64(double v, LaneX lx) {
  auto add = [&](auto other) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(other(__uint_as_float((uint32_t)u))), hi = __float_as_uint(other(__uint_as_float((uint32_t)(u >> 32))));
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  add([&](float x) { return lane_xor<32>(x, lx); });
  add([&](float x) { return lane_xor<16>(x, lx); });
  add([&](float x) { return lane_xor<8>(x, lx); });
  add([&](float x) { return lane_xor<4>(x, lx); });
  add([&](float x) { return lane_xor<2>(x, lx); });
  add([&](float x) { return lane_xor<1>(x, lx); });
  return v;
}

// The largest u such that at least n lanes (1 .. 64) have a key of u or more.
__device__ __forceinline__ uint32_t nth_key(uint32_t key, int n) {
  uint32_t u = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t v = u | 1u << bit;
    if (__popcll(__ballot(key >= v)) >= n) u = v;
  }
  return u;
}

// The logits of a thread: number (i * 256 + tid) * W + e of the slice, which
// begins at t0, is x[i * W + e].
template <typename T, bool WIDE, int E>
struct Slice {
  static constexpr int W = WIDE ? 16 / sizeof(T) : 1;
  float x[E];
  __device__ __forceinline__ static int token(int t0, int i) { return t0 + (i / W * kThreads + (int)threadIdx.x) * W + i % W; }
  __device__ __forceinline__ void load(const T* row, int t0, int vocab) {
    if (WIDE && t0 + E * kThreads <= vocab) {
      u32x4 v[E / W];
#pragma unroll
      for (int i = 0; i < E / W; ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + token(t0, i * W)));
#pragma unroll
      for (int i = 0; i < E / W; ++i) {
        const u32x4 u = v[i];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if constexpr (sizeof(T) == 4) x[i * W + e] = __uint_as_float(u[e]);
          else if constexpr (std::is_same<T, _Float16>::value) x[i * W + e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[e / 2] >> 16 * (e & 1)));
          else x[i * W + e] = __uint_as_float(e & 1 ? u[e / 2] & 0xFFFF0000u : u[e / 2] << 16);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int t = token(t0, i);
        float f = -INFINITY;
        if (t < vocab) {
          if constexpr (sizeof(T) == 4) f = row[t];
          else if constexpr (std::is_same<T, _Float16>::value) f = (float)row[t];
          else f = __uint_as_float((uint32_t)row[t] << 16);
        }
        x[i] = f;
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = fmaxf(x[i], -INFINITY);  // NaN counts as -inf
  }
};

// One work-group per slice of 256 E logits, which stay in registers.
//
// A logit is among the slice's best only if it is not below the edge, the
// keep-th largest of the threads' largest, or something lower that is found
// without an exchange: up to 32, the largest of the waves' keep-th largest
// and, from 9 on, the least of their keep / 4-th (256 rows of 151936 bf16,
// keep 32: 59 us for the selection with both instead of 70, 48 with longer
// slices).  Few logits lie above it in most cases; where they and those at it
// are more than kRoom, the edge is taken from the threads, above which lie
// (keep - 1) E at most, which slice_size keeps below kRoom, and of those at it
// the lowest tokens are taken.
//
// Bound by the logits' way from memory: 26 us for 155 MB (256 rows of 151936
// fp32).
template <typename T, bool WIDE, int E>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(SelectArgs a) {
  typedef Slice<T, WIDE, E> S;
  __shared__ uint64_t room[kRoom];
  __shared__ float tops[kThreads];
  __shared__ float red[3][4];
  __shared__ double sums[4];
  __shared__ float line;
  __shared__ int count;
  const LaneX lx = lane_x_init();
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, slice = blockIdx.x;
  const int64_t row = blockIdx.y;
  if (a.finished && a.finished[row]) return;  // its one continuation needs no logits
  const int t0 = slice * (E * kThreads), keep = a.keep;
  S s;
  s.load(static_cast<const T*>(a.logits) + row * a.ld, t0, a.vocab);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < E; ++i) m = fmaxf(m, s.x[i]);
  float top = m;
  top = fmaxf(top, lane_xor<32>(top, lx));
  top = fmaxf(top, lane_xor<16>(top, lx));
  top = fmaxf(top, lane_xor<8>(top, lx));
  top = fmaxf(top, lane_xor<4>(top, lx));
  top = fmaxf(top, lane_xor<2>(top, lx));
  top = fmaxf(top, lane_xor<1>(top, lx));
  const float edge_w = keep <= 32 ? order_float(nth_key(order_bits(m), keep)) : -INFINITY;
  const float part_w = keep <= 32 && keep > 8 ? order_float(nth_key(order_bits(m), (keep + 3) / 4)) : -INFINITY;
  tops[tid] = m;
  if (lane == 0) red[0][w] = top, red[1][w] = edge_w, red[2][w] = part_w;
  if (tid == 0) count = 0;
  __syncthreads();
  const float all = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float edge = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
  edge = fmaxf(edge, fminf(fminf(red[2][0], red[2][1]), fminf(red[2][2], red[2][3])));
  auto threads_edge = [&]() {
    int above = 0, same = 0;
    for (int i = 0; i < kThreads; ++i) above += tops[i] > m, same += tops[i] == m;
    if (above < keep && keep <= above + same) line = m;  // all that write it write the same
    __syncthreads();
    return line;
  };
  if (keep > 32) edge = threads_edge();
  double sum = 0.0;
  if (all < INFINITY) {
#pragma unroll
    for (int p = 0; p < E; p += 16) {
      float part[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) part[i] = exp_below(s.x[p + i], all);
#pragma unroll
      for (int n = 8; n > 0; n /= 2)
#pragma unroll
        for (int i = 0; i < n; ++i) part[i] += part[i + n];
      sum += part[0];
    }
  }
  sum = wave_sum64(sum, lx);
  if (lane == 0) sums[w] = sum;
  auto add = [&](int i) {
    const int at = atomicAdd(&count, 1);
    if (at < kRoom) room[at] = (uint64_t)order_bits(s.x[i]) << 32 | (uint32_t)~S::token(t0, i);
  };
  if (__any(m >= edge)) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (s.x[i] >= edge && S::token(t0, i) < a.vocab) add(i);
  }
  __syncthreads();
  int n = count;
  if (n > kRoom) {
    // too many at the edge: those above it, then the others by rising tokens until there are enough
    if (keep <= 32) edge = threads_edge();
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (s.x[i] > edge) add(i);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; i += S::W) {
      const bool enough = count >= keep;
      __syncthreads();
      if (enough) continue;
#pragma unroll
      for (int e = i; e < i + S::W; ++e)
        if (s.x[e] == edge && S::token(t0, e) < a.vocab) add(e);
      __syncthreads();
    }
    n = count;
  }
  uint64_t* best = a.best + (row * a.slices + slice) * keep;
  for (int c = tid; c < n; c += kThreads) {
    const uint64_t me = room[c];
    int place = 0;
    for (int i = 0; i < n; ++i) place += room[i] > me;
    if (place < keep) best[place] = me;
  }
  for (int c = n + tid; c < keep; c += kThreads) best[c] = 0;
  if (tid == 0) {
    a.stats[row * a.slices + slice] = Stat{(sums[0] + sums[1]) + (sums[2] + sums[3]), all};
  }
}

struct Candidate {
  uint64_t score;  // order bits of the fp64 score
  uint32_t at;     // ~(beam * vocab + token)
};
__device__ __forceinline__ bool over(const Candidate& x, const Candidate& y) {
  return x.score > y.score || (x.score == y.score && x.at > y.at);
}

// One work-group per request.
__global__ __launch_bounds__(kJoin) void beam_join_kernel(SelectArgs a, Candidate* spill) {
  constexpr int kList = 512, kAhead = 4, kMore = 4;
  __shared__ double base[1024];    // the sum; then the log sum, of a finished beam its score
  __shared__ float largest[1024];  // the largest logit; then the score
  __shared__ uint8_t state[1024];
  __shared__ Candidate list[kList];
  __shared__ Candidate tops[kJoin], line;
  __shared__ uint32_t edge;
  __shared__ int count;
  const LaneX lx = lane_x_init();
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t b = blockIdx.x;
  // A thread's k-th candidate.  The lists that they come from are in order, so
  // each row of them is turned against the one before: a thread that had only
  // the lists' first entries, where keep divides the threads, would leave the
  // edge below to the others' (one request of 16 beams, 151936 tokens, keep 32:
  // 1530 us, turned 66).
  auto place = [&](int k) { return k * kJoin + ((tid + 37 * k) & (kJoin - 1)); };
  const int some = a.slices * a.keep, per = some > a.keep + 1 ? some : a.keep + 1, all = a.beams * per;
  // More candidates than the threads have at hand at first, and lists enough for
  // a close edge: by lists (the request above 22 us, 300 beams of 20000 tokens,
  // keep 128, 97 instead of 540, 32 x 8 beams, keep 8, 35.4 instead of 37.8;
  // 4 beams of 151936, keep 4, of 592 candidates, 11.0 by lists, 10.7 without).
  const bool lists = all > kAhead * kJoin && a.beams * a.slices >= 64 && a.beams * a.slices >= 2 * a.keep;
  // a thread's first candidates are on their way while the sums are made
  uint64_t ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int e = place(i), j = e / per;
    ahead[i] = !lists && e < all && e - j * per < some ? a.best[(b * a.beams + j) * some + e - j * per] : 0;
  }
  for (int j = w; j < a.beams; j += kJoin / 64) {
    // lane i: slices i, i + 64 ..
    const Stat* st = a.stats + (b * a.beams + j) * a.slices;
    const Stat own = lane < a.slices ? st[lane] : Stat{0.0, -INFINITY};
    float top = own.top;
    for (int i = lane + 64; i < a.slices; i += 64) top = fmaxf(top, st[i].top);
    top = fmaxf(top, lane_xor<32>(top, lx));
    top = fmaxf(top, lane_xor<16>(top, lx));
    top = fmaxf(top, lane_xor<8>(top, lx));
    top = fmaxf(top, lane_xor<4>(top, lx));
    top = fmaxf(top, lane_xor<2>(top, lx));
    top = fmaxf(top, lane_xor<1>(top, lx));
    double l = 0.0;
    if (fabsf(top) < INFINITY) {
      l = own.sum * exp_below(own.top, top);
      for (int i = lane + 64; i < a.slices; i += 64) l += st[i].sum * exp_below(st[i].top, top);
    }
    l = wave_sum64(l, lx);
    if (lane == 0) base[j] = l, largest[j] = top;
  }
  if (tid == 0) count = 0, edge = 0;
  __syncthreads();
  for (int j = tid; j < a.beams; j += kJoin) {
    const int64_t row = b * a.beams + j;
    const bool done = a.finished && a.finished[row];
    const float s = a.scores[row], top = largest[j];
    const bool fine = fabsf(s) < INFINITY, runs = !done && fine && fabsf(top) < INFINITY;
    base[j] = runs ? (double)top + log(base[j]) : fine ? s : -INFINITY;
    largest[j] = s, state[j] = runs ? 0 : done ? 1 : 2;
  }
  __syncthreads();
  // a beam offers slices * keep candidates; one that is finished or has none keep + 1: eos and the first tokens
  auto get = [&](int j, int i, uint64_t k) {
    int64_t t = -1;
    double v = -INFINITY;
    if (state[j] == 0) {
      if (!k) return Candidate{0, 0};
      t = (uint32_t)~k;
      v = largest[j] + ((double)order_float((uint32_t)(k >> 32)) - base[j]);  // in this order: equal continuations tie
    } else {
      const bool has = state[j] == 1 && a.eos >= 0 && a.eos < a.vocab;
      if (i > a.keep || (i == a.keep && !has)) return Candidate{0, 0};
      if (i == a.keep) t = a.eos, v = base[j];
      else t = i < a.vocab && !(has && i == a.eos) ? i : -1;
      if (t < 0) return Candidate{0, 0};
    }
    return Candidate{order_bits64(v), ~(uint32_t)(j * (int64_t)a.vocab + t)};
  };
  auto each = [&](auto use) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (!lists && place(i) < all) use(get(place(i) / per, place(i) % per, ahead[i]));
    // the others, four loads on their way together
    for (int i = lists ? 0 : kAhead; i * kJoin < all; i += kMore) {
      uint64_t k[kMore];
#pragma unroll
      for (int x = 0; x < kMore; ++x) {
        const int e = place(i + x), j = e / per;
        k[x] = e < all && e - j * per < some ? a.best[(b * a.beams + j) * some + e - j * per] : 0;
      }
#pragma unroll
      for (int x = 0; x < kMore; ++x)
        if (place(i + x) < all) use(get(place(i + x) / per, place(i + x) % per, k[x]));
    }
  };
  // `lists`: only the first entry of each slice's list is looked at for the
  // edge, and of each list what is not below it.
  auto list_of = [&](int u, auto use) {
    const int j = u / a.slices, s = u - j * a.slices;
    use(j, s * a.keep, a.best + ((b * a.beams + j) * a.slices + s) * a.keep);
  };
  auto firsts = [&](auto use) {
    for (int u = tid; u < a.beams * a.slices; u += kJoin)
      list_of(u, [&](int j, int i, const uint64_t* from) {
        if (state[j] == 0) use(get(j, i, from[0]));
        else if (i == 0) use(get(j, 0, 0)), use(get(j, a.keep, 0));
      });
  };
  auto down_to = [&](uint32_t least, auto use) {
    auto reaches = [&](const Candidate& c) { return c.score && (uint32_t)(c.score >> 32) >= least; };
    if (!lists) {
      each([&](const Candidate& c) {
        if (reaches(c)) use(c);
      });
      return;
    }
    for (int u = tid; u < a.beams * a.slices; u += kJoin)
      list_of(u, [&](int j, int i0, const uint64_t* from) {
        if (state[j] != 0) {
          if (i0 == 0)
            for (int i = 0; i <= a.keep; ++i) {
              const Candidate c = get(j, i, 0);
              if (reaches(c)) use(c);
            }
          return;
        }
        bool on = true;
        for (int i = 0; on && i < a.keep; i += kMore) {
          uint64_t k[kMore];
#pragma unroll
          for (int x = 0; x < kMore; ++x) k[x] = i + x < a.keep ? from[i + x] : 0;
#pragma unroll
          for (int x = 0; x < kMore; ++x) {
            const Candidate c = get(j, i0 + i + x, k[x]);
            on = on && reaches(c);
            if (on) use(c);
          }
        }
      });
  };
  // The upper half of a score's order bits is enough to leave most out: at
  // least `keep` candidates have the edge's or more, and so have the best.
  uint32_t top = 0;
  auto highest = [&](const Candidate& c) {
    const uint32_t hi = (uint32_t)(c.score >> 32);
    top = hi > top ? hi : top;
  };
  if (lists) firsts(highest);
  else each(highest);
  // Of a wave's threads, or of all (one request of 40 beams, keep 64: 66 us and
  // 32; 8 of 10 beams, keep 40: 28.5 and 31.6).
  if (a.keep <= 48) {
    const uint32_t u = nth_key(top, a.keep);
    if (lane == 0) atomicMax(&edge, u);
  } else {
    tops[tid].at = top;
    __syncthreads();
    int above = 0, same = 0;
    for (int i = 0; i < kJoin; ++i) above += tops[i].at > top, same += tops[i].at == top && i < tid;
    if (above + same == a.keep - 1) edge = top;
  }
  __syncthreads();
  const uint32_t least = edge;
  Candidate* more = spill + b * (int64_t)all;
  auto add = [&](const Candidate& c) {
    const int at = atomicAdd(&count, 1);
    (at < kList ? list[at] : more[at]) = c;
  };
  down_to(least, add);
  __threadfence();
  __syncthreads();
  int n = count;
  if (n > kList) {
    // Many scores that agree in the upper half, equal ones perhaps: the same
    // once more with the whole order, in which no two are alike (128 of 115000
    // equal ones: 0.8 ms; the ranks of all would take 70 ms).
    Candidate mine{0, 0};
    each([&](const Candidate& c) {
      if (over(c, mine)) mine = c;
    });
    __syncthreads();
    tops[tid] = mine;
    if (tid == 0) count = 0, line = Candidate{0, 0};
    __syncthreads();
    int above = 0;
    for (int i = 0; i < kJoin; ++i) above += over(tops[i], mine);
    if (above == a.keep - 1 && mine.score) line = mine;
    __syncthreads();
    const Candidate low = line;
    down_to(least, [&](const Candidate& c) {
      if (!over(low, c)) add(c);
    });
    __threadfence();
    __syncthreads();
    n = count;
  }
  for (int c = tid; c < n; c += kJoin) {
    const Candidate x = c < kList ? list[c] : more[c];
    int rank = 0;
    const int near = n < kList ? n : kList;
    for (int i = 0; i < near; ++i) rank += over(list[i], x);
    for (int i = kList; i < n; ++i) rank += over(more[i], x);
    if (rank < a.keep) {
      const uint32_t at = ~x.at;
      a.scores_out[b * a.keep + rank] = (float)order_double(x.score);
      a.parents_out[b * a.keep + rank] = (int32_t)(b * a.beams + at / a.vocab);
      a.tokens_out[b * a.keep + rank] = (int32_t)(at % a.vocab);
    }
  }
}

// Logits per thread: 32 where that leaves work-groups enough to fill the chip
// (256 rows of 151936 fp32, keep 8: 35.4 us for the whole selection, with 16 42;
// bf16, keep 32: 48 and 59), 16 otherwise and where what lies above the edge
// would not fit (beam_slice_kernel).
int slice_size(int64_t rows, int64_t vocab, int keep) {
  return keep <= 64 && rows * ((vocab + 32 * kThreads - 1) / (32 * kThreads)) >= 512 ? 32 : 16;
}

struct Layout {
  int slices, each;
  size_t stats, best, spill, bytes;
};

Layout layout_of(int64_t batch, int beams, int64_t vocab, int keep) {
  Layout l;
  const int64_t rows = batch * beams;
  l.each = slice_size(rows, vocab, keep);
  const int64_t slice = (int64_t)kThreads * l.each;
  l.slices = (int)((vocab + slice - 1) / slice);
  const int64_t per = (int64_t)l.slices * keep > keep + 1 ? (int64_t)l.slices * keep : keep + 1;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  l.stats = 0;
  l.best = up((size_t)rows * l.slices * sizeof(Stat));
  l.spill = l.best + up((size_t)rows * l.slices * keep * sizeof(uint64_t));
  l.bytes = l.spill + up((size_t)rows * per * sizeof(Candidate));
  return l;
}

template <typename T>
auto slice_kernel(bool wide, int each) {
  if (wide) return each == 32 ? beam_slice_kernel<T, true, 32> : beam_slice_kernel<T, true, 16>;
  return each == 32 ? beam_slice_kernel<T, false, 32> : beam_slice_kernel<T, false, 16>;
}

// ---------------------------------------------------------------------------
// states
// ---------------------------------------------------------------------------

struct ReorderArgs {
  const char* src[QS_MAX_STATES];
  char* dst[QS_MAX_STATES];
  int64_t bytes[QS_MAX_STATES], stride[QS_MAX_STATES];
  int width[QS_MAX_STATES];  // of one access
  const int32_t* parents;
  int64_t rows_in;
};

template <typename T>
__device__ __forceinline__ void row_copy(const char* from, char* to, int64_t bytes) {
  const int64_t n = bytes / sizeof(T);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    T x{};
    if (from) x = reinterpret_cast<const T*>(from)[i];
    reinterpret_cast<T*>(to)[i] = x;
  }
}

__global__ __launch_bounds__(256) void reorder_kernel(ReorderArgs a) {
  const int64_t i = blockIdx.y;
  const int s = blockIdx.z;
  const int64_t p = a.parents[i];
  const char* from = p >= 0 && p < a.rows_in ? a.src[s] + p * a.stride[s] : nullptr;
  char* to = a.dst[s] + i * a.bytes[s];
  if (a.width[s] == 16) row_copy<uint4>(from, to, a.bytes[s]);
  else if (a.width[s] == 4) row_copy<uint32_t>(from, to, a.bytes[s]);
  else row_copy<uint8_t>(from, to, a.bytes[s]);
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" size_t qs_beam_select_workspace_bytes(int64_t batch, int beams, int64_t vocab, int keep) {
  if (batch < 1 || beams < 1 || vocab < 1 || keep < 1) return 0;
  return layout_of(batch, beams, vocab, keep).bytes;
}

extern "C" int qs_beam_select(const void* logits, int dtype, int64_t ld, int64_t batch, int beams, int64_t vocab,
                              const float* scores, const uint8_t* finished, int64_t eos, int keep, float* scores_out,
                              int32_t* parents_out, int32_t* tokens_out, void* workspace, size_t workspace_bytes,
                              qs_stream_t stream) {
  if (batch == 0) return QS_OK;
  QS_REQUIRE(logits && scores && scores_out && parents_out && tokens_out, "qs_beam_select: null pointer");
  QS_REQUIRE(dtype == QS_DTYPE_F32 || dtype == QS_DTYPE_F16 || dtype == QS_DTYPE_BF16, "qs_beam_select: dtype %d", dtype);
  QS_REQUIRE(batch >= 1 && beams >= 1 && vocab >= 1 && ld >= vocab && keep >= 1, "qs_beam_select: %lld x %d beams of %lld tokens (row stride %lld), keep %d",
             (long long)batch, beams, (long long)vocab, (long long)ld, keep);
  QS_SUPPORTED(beams <= 1024 && keep <= kMaxKeep && vocab <= (1 << 24) && beams * vocab <= INT32_MAX && batch * beams <= 65535,
               "qs_beam_select: %lld x %d beams of %lld tokens, keep %d (at most 1024 beams, 65535 rows, keep %d)",
               (long long)batch, beams, (long long)vocab, keep, kMaxKeep);
  QS_REQUIRE(keep <= beams * vocab, "qs_beam_select: keep %d of %lld continuations", keep, (long long)(beams * vocab));
  const Layout l = layout_of(batch, beams, vocab, keep);
  QS_REQUIRE(workspace && workspace_bytes >= l.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "qs_beam_select: workspace of %zu bytes (16-byte aligned), %zu needed", workspace_bytes, l.bytes);
  char* ws = static_cast<char*>(workspace);
  const SelectArgs a{logits, ld, scores, finished, reinterpret_cast<Stat*>(ws + l.stats),
                     reinterpret_cast<uint64_t*>(ws + l.best), scores_out, parents_out, tokens_out, eos, beams,
                     (int)vocab, keep, l.slices, dtype};
  const size_t size = dtype == QS_DTYPE_F32 ? 4 : 2;
  const bool wide = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && ld * size % 16 == 0;
  const dim3 grid((unsigned)l.slices, (unsigned)(batch * beams));
  const auto slice = dtype == QS_DTYPE_F32   ? slice_kernel<float>(wide, l.each)
                     : dtype == QS_DTYPE_F16 ? slice_kernel<_Float16>(wide, l.each)
                                             : slice_kernel<uint16_t>(wide, l.each);
  hipLaunchKernelGGL(slice, grid, dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("beam_slice_kernel");
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)batch), dim3(kJoin), 0, as_stream(stream), a,
                     reinterpret_cast<Candidate*>(ws + l.spill));
  QS_LAUNCHED("beam_join_kernel");
  return QS_OK;
}

extern "C" int qs_reorder_states(int count, const void* const* src, void* const* dst, const int64_t* row_bytes,
                                 const int64_t* src_stride, const int32_t* parents, int64_t rows_out, int64_t rows_in,
                                 qs_stream_t stream) {
  if (count == 0 || rows_out == 0) return QS_OK;
  QS_REQUIRE(count >= 1 && count <= QS_MAX_STATES && src && dst && row_bytes && src_stride && parents && rows_out >= 1 &&
                 rows_out <= 65535 && rows_in >= 0,
             "qs_reorder_states: %d states (at most %d), %lld of %lld rows", count, QS_MAX_STATES, (long long)rows_out, (long long)rows_in);
  ReorderArgs a{};
  int64_t most = 0;
  for (int s = 0; s < count; ++s) {
    QS_REQUIRE(row_bytes[s] >= 0 && src_stride[s] >= row_bytes[s] && (((src[s] || rows_in == 0) && dst[s]) || row_bytes[s] == 0),
               "qs_reorder_states: state %d: rows of %lld bytes, %lld apart", s, (long long)row_bytes[s], (long long)src_stride[s]);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(src[s]) | reinterpret_cast<uintptr_t>(dst[s]) | (uintptr_t)row_bytes[s] | (uintptr_t)src_stride[s];
    a.src[s] = static_cast<const char*>(src[s]), a.dst[s] = static_cast<char*>(dst[s]);
    a.bytes[s] = row_bytes[s], a.stride[s] = src_stride[s];
    a.width[s] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    const int64_t n = row_bytes[s] / a.width[s];
    most = n > most ? n : most;
  }
  if (most == 0) return QS_OK;
  a.parents = parents, a.rows_in = rows_in;
  const int64_t wide = (most + 255) / 256, gx = wide < 256 ? wide : 256;
  hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)gx, (unsigned)rows_out, (unsigned)count), dim3(256), 0, as_stream(stream), a);
  QS_LAUNCHED("reorder_kernel");
  return QS_OK;
}
