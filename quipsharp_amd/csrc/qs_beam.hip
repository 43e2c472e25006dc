// Beam search: the best continuations over beams and vocabulary, and the
// states that follow them (qs_beam_select, qs_reorder_states).
//
// A continuation scores s_b + x_t - log sum_t' exp(x_t').  Within a beam the
// order is that of the logits, so one pass over them finds both what the sum
// needs (the running maximum and sum) and each slice's best `keep`; the
// second launch adds the slices' sums and chooses among the slices' bests by
// the score in fp64.
#include "qs_common.h"

namespace qs {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxKeep = 128;
constexpr int kPer = 16;                  // logits per thread
constexpr int kSlice = kThreads * kPer;   // logits per work-group

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

struct SelectArgs {
  const void* logits;
  int64_t ld;
  const float* scores;
  const uint8_t* finished;
  float *stats;    // [rows][slices][2]: maximum, sum
  uint64_t* best;  // [rows][slices][keep]: order bits << 32 | ~token, in descending order; 0 for none
  float* scores_out;
  int32_t *parents_out, *tokens_out;
  int64_t eos;
  int beams, vocab, keep, slices, dtype;
};

// One work-group per slice of a row of logits.
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(SelectArgs a) {
  __shared__ uint64_t tops[kThreads];
  __shared__ uint64_t cand[kMaxKeep * kPer];
  __shared__ float red[kThreads / 64];
  __shared__ uint64_t edge;
  __shared__ int count;
  const int tid = threadIdx.x, slice = blockIdx.x;
  const int64_t row = blockIdx.y;
  if (a.finished && a.finished[row]) return;  // its one continuation needs no logits
  float x[kPer];
  uint64_t key[kPer], top = 0;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int t = slice * kSlice + i * kThreads + tid;
    x[i] = t < a.vocab ? load_as_float(a.logits, a.dtype, row * a.ld + t) : -INFINITY;
    x[i] = x[i] != x[i] ? -INFINITY : x[i];
    key[i] = t < a.vocab ? (uint64_t)order_bits(x[i]) << 32 | (uint32_t)~t : 0;
    top = key[i] > top ? key[i] : top;
    m = fmaxf(m, x[i]);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  tops[tid] = top;
  if ((tid & 63) == 0) red[tid >> 6] = m;
  if (tid == 0) count = 0, edge = 0;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float sum = 0.f;
  if (fabsf(m) != INFINITY) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += expf(x[i] - m);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
  // the keep-th largest of the threads' largest: at least `keep` keys are not below it, and only `keep` threads hold
  // such keys, kPer each at most
  int above = 0;
  for (int i = 0; i < kThreads; ++i) above += tops[i] > top;
  if (above == a.keep - 1 && top) edge = top;
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = sum;
  const uint64_t least = edge ? edge : 1;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (key[i] >= least) cand[atomicAdd(&count, 1)] = key[i];
  __syncthreads();
  const int n = count;
  uint64_t* best = a.best + (row * a.slices + slice) * a.keep;
  for (int c = tid; c < n; c += kThreads) {
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += cand[i] > cand[c];
    if (rank < a.keep) best[rank] = cand[c];
  }
  for (int c = n + tid; c < a.keep; c += kThreads) best[c] = 0;
  if (tid == 0) {
    float* st = a.stats + 2 * (row * a.slices + slice);
    st[0] = m, st[1] = (red[0] + red[1]) + (red[2] + red[3]);
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
__global__ __launch_bounds__(kThreads) void beam_join_kernel(SelectArgs a, Candidate* spill) {
  __shared__ Candidate tops[kThreads];
  __shared__ double base[1024];  // score - log sum; of a beam without continuations -inf
  __shared__ uint8_t state[1024];
  __shared__ Candidate edge;
  __shared__ int count;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t b = blockIdx.x;
  for (int j = w; j < a.beams; j += kThreads / 64) {
    const int64_t row = b * a.beams + j;
    const bool done = a.finished && a.finished[row];
    const float s = a.scores[row];
    double c = -INFINITY;
    if (fabsf(s) < INFINITY) {
      if (done) {
        c = s;
      } else {
        const float* st = a.stats + 2 * row * a.slices;
        float m = -INFINITY;
        for (int i = lane; i < a.slices; i += 64) m = fmaxf(m, st[2 * i]);
#pragma unroll
        for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        double sum = 0;
        if (fabsf(m) < INFINITY)
          for (int i = lane; i < a.slices; i += 64) sum += exp((double)st[2 * i] - m) * st[2 * i + 1];
#pragma unroll
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if (fabsf(m) < INFINITY) c = (double)s - ((double)m + log(sum));
      }
    }
    if (lane == 0) base[j] = c, state[j] = done ? 1 : c == -INFINITY ? 2 : 0;
  }
  if (tid == 0) count = 0, edge = Candidate{0, 0};
  __syncthreads();
  // a beam offers slices * keep candidates; one that is finished or has none keep + 1: eos and the first tokens
  const int per = a.slices * a.keep > a.keep + 1 ? a.slices * a.keep : a.keep + 1, all = a.beams * per;
  auto get = [&](int e) {
    const int j = e / per, i = e % per;
    const int64_t row = b * a.beams + j;
    int64_t t = -1;
    double v = -INFINITY;
    if (state[j] == 0) {
      if (i >= a.slices * a.keep) return Candidate{0, 0};
      const uint64_t k = a.best[row * a.slices * a.keep + i];
      if (!k) return Candidate{0, 0};
      t = (uint32_t)~k;
      v = base[j] + (double)order_float((uint32_t)(k >> 32));
    } else {
      const bool has = state[j] == 1 && a.eos >= 0 && a.eos < a.vocab;
      if (i > a.keep || (i == a.keep && !has)) return Candidate{0, 0};
      if (i == a.keep) t = a.eos, v = base[j];
      else t = i < a.vocab && !(has && i == a.eos) ? i : -1;
      if (t < 0) return Candidate{0, 0};
    }
    return Candidate{order_bits64(v), ~(uint32_t)(j * (int64_t)a.vocab + t)};
  };
  Candidate top{0, 0};
  for (int e = tid; e < all; e += kThreads) {
    const Candidate c = get(e);
    if (over(c, top)) top = c;
  }
  tops[tid] = top;
  __syncthreads();
  int above = 0;
  for (int i = 0; i < kThreads; ++i) above += over(tops[i], top);
  if (above == a.keep - 1 && top.score) edge = top;
  __syncthreads();
  const Candidate least = edge;
  Candidate* cand = spill + b * (int64_t)all;
  for (int e = tid; e < all; e += kThreads) {
    const Candidate c = get(e);
    if (c.score && !over(least, c)) cand[atomicAdd(&count, 1)] = c;
  }
  __threadfence();
  __syncthreads();
  const int n = count;
  for (int c = tid; c < n; c += kThreads) {
    const Candidate x = cand[c];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += over(cand[i], x);
    if (rank < a.keep) {
      const uint32_t at = ~x.at;
      a.scores_out[b * a.keep + rank] = (float)order_double(x.score);
      a.parents_out[b * a.keep + rank] = (int32_t)(b * a.beams + at / a.vocab);
      a.tokens_out[b * a.keep + rank] = (int32_t)(at % a.vocab);
    }
  }
}

struct Layout {
  int slices;
  size_t stats, best, spill, bytes;
};

Layout layout_of(int64_t batch, int beams, int64_t vocab, int keep) {
  Layout l;
  l.slices = (int)((vocab + kSlice - 1) / kSlice);
  const int64_t rows = batch * beams, per = (int64_t)l.slices * keep > keep + 1 ? (int64_t)l.slices * keep : keep + 1;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  l.stats = 0;
  l.best = up((size_t)rows * l.slices * 2 * sizeof(float));
  l.spill = l.best + up((size_t)rows * l.slices * keep * sizeof(uint64_t));
  l.bytes = l.spill + up((size_t)rows * per * sizeof(Candidate));
  return l;
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
  const SelectArgs a{logits, ld, scores, finished, reinterpret_cast<float*>(ws + l.stats),
                     reinterpret_cast<uint64_t*>(ws + l.best), scores_out, parents_out, tokens_out, eos, beams,
                     (int)vocab, keep, l.slices, dtype};
  hipLaunchKernelGGL(beam_slice_kernel, dim3((unsigned)l.slices, (unsigned)(batch * beams)), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("beam_slice_kernel");
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)batch), dim3(kThreads), 0, as_stream(stream), a,
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
    QS_REQUIRE(row_bytes[s] >= 0 && src_stride[s] >= row_bytes[s] && ((src[s] && dst[s]) || row_bytes[s] == 0),
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
