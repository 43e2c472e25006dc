// The work on a paged key-value cache's pages: storing new tokens, copying,
// forking rows (beams), giving pages out and back, and moving the pages in
// use together.  The tables are small and their work is a chain of short
// steps, so one work-group does all of it (no step waits for another
// work-group); it leaves a list of copies, and a second launch, as wide as
// the chip, moves the bytes.  Each step over global memory costs a round trip
// of about a microsecond, so tables and counts that fit are kept in LDS
// meanwhile (`NEAR`; 7 us against 14 for a fork of 32 rows).
#include "qs_rope_dev.h"

namespace qs {
namespace {

constexpr int kMaxRows = 1024;
constexpr int kThreads = 1024;
// Loops over pages and copies count in int: a step beyond the last stays below 2^31.
constexpr int kPageStep = 8 * kThreads;  // the longest step (ref_copy)
constexpr int kCopyStep = 64;            // work-groups that deal copies

struct Store {
  char* data;
  int64_t planes, pages, row_bytes;
  int kv_heads, page;
};

// A copy of the first `used` positions of every head of a page.
struct Copy {
  int32_t src, dst, used;
};

// plan[0]: the number of copies; the copies from plan + 4.
__device__ __host__ __forceinline__ int32_t* plan_copies(int32_t* plan) { return plan + 4; }

// Reference counts are changed with atomics, which act in the L2: they are
// read with atomic loads too, which do not take a line that the L1 still has.
__device__ __forceinline__ int ref_load(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void ref_add(int32_t* p, int v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void ref_store(int32_t* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The counts of all pages, for a kernel's own work on them: loads of eight
// pages of a thread are on their way together (the stores, which may be to the
// same place, would have each wait for the one before).
__device__ __forceinline__ void ref_copy(const int32_t* from, int32_t* to, int pages) {
  constexpr int kN = kPageStep / kThreads;
  for (int p0 = threadIdx.x; p0 < pages; p0 += kN * blockDim.x) {
    int n[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) n[i] = p0 + i * (int)blockDim.x < pages ? from[p0 + i * blockDim.x] : 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (p0 + i * (int)blockDim.x < pages) ref_store(to + p0 + i * blockDim.x, n[i]);
  }
}

// Every global access of the work-group before the barrier is done when a
// thread goes on after it (loads and atomics of another wave see it in the L2).
__device__ __forceinline__ void group_sync() {
  __threadfence();
  __syncthreads();
}

// Exclusive prefix sum over the 1024 threads; *total gets the sum.  `part` is
// 16 ints of LDS; a barrier stands before and after.
__device__ __forceinline__ int scan1024(int v, int* part, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) part[w] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const int y = part[i];
    before += i < w ? y : 0;
    all += y;
  }
  *total = all;
  return before + x - v;
}

// ---------------------------------------------------------------------------
// copies
// ---------------------------------------------------------------------------

// Pieces of 16 KB of (copy, plane, head), dealt over the grid; a thread's four
// loads are on their way together.  Stores go past the caches, which would
// only hand the lines on: 266 MB moved in 98 us instead of 119 (with the loads
// past them too 103).
constexpr int kPiece = 16384;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void copy_piece(const Store& st, unsigned rest, unsigned pieces, int64_t src, int64_t dst, int64_t bytes) {
  const int64_t head_bytes = st.page * st.row_bytes, page_bytes = head_bytes * st.kv_heads;
  const unsigned plane_head = rest / pieces, piece = rest - plane_head * pieces;
  const unsigned plane = plane_head / (unsigned)st.kv_heads, head = plane_head - plane * (unsigned)st.kv_heads;
  const int64_t at = (int64_t)piece * kPiece + threadIdx.x * 16;
  char* base = st.data + (int64_t)plane * st.pages * page_bytes + head * head_bytes + at;
  const char* from = base + src * page_bytes;
  char* to = base + dst * page_bytes;
  u32x4 x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + 4096 * j < bytes) x[j] = *reinterpret_cast<const u32x4*>(from + 4096 * j);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + 4096 * j < bytes) __builtin_nontemporal_store(x[j], reinterpret_cast<u32x4*>(to + 4096 * j));
}

// blockIdx.y deals the planes and heads of a copy, blockIdx.x the copies.
__global__ __launch_bounds__(256) void page_copy_kernel(Store st, const int32_t* plan) {
  const int count = plan[0];
  const Copy* copies = reinterpret_cast<const Copy*>(plan + 4);
  const unsigned pieces = (unsigned)((st.page * st.row_bytes + kPiece - 1) / kPiece);
  const unsigned per = (unsigned)(st.planes * st.kv_heads) * pieces;
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const Copy c = copies[i];
    for (unsigned r = blockIdx.y; r < per; r += gridDim.y) copy_piece(st, r, pieces, c.src, c.dst, c.used * st.row_bytes);
  }
}

// The caller's pairs; those outside the pool have nothing to copy.
__global__ __launch_bounds__(256) void page_list_kernel(Store st, const int32_t* src, const int32_t* dst, int count) {
  const unsigned pieces = (unsigned)((st.page * st.row_bytes + kPiece - 1) / kPiece);
  const unsigned per = (unsigned)(st.planes * st.kv_heads) * pieces;
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const int64_t s = src[i], d = dst[i];
    if (s < 0 || d < 0 || s >= st.pages || d >= st.pages) continue;
    for (unsigned r = blockIdx.y; r < per; r += gridDim.y) copy_piece(st, r, pieces, s, d, st.page * st.row_bytes);
  }
}

// Work-groups for up to `count` copies: 4096 in all, each with a few pieces.
dim3 copy_grid(const Store& st, int64_t count) {
  const int64_t pieces = (st.page * st.row_bytes + kPiece - 1) / kPiece, per = st.planes * st.kv_heads * pieces;
  int64_t x = count < kCopyStep ? count : kCopyStep;
  int64_t y = 4096 / x;
  y = y < per ? y : per;
  return dim3((unsigned)x, (unsigned)y);
}

// ---------------------------------------------------------------------------
// advance: fork, give back, give out
// ---------------------------------------------------------------------------

struct AdvanceArgs {
  const int32_t *table, *lengths, *refs, *parents;
  const int32_t* row_tokens;  // per row, or null: `tokens` for all
  int32_t *table_out, *lengths_out, *refs_out, *short_pages, *plan;
  int32_t* over;     // per row, or null: lengths go on beyond the table
  int32_t* missing;  // the sum of short_pages over the steps, or null
  int rows, cols, pages, page, tokens;
};

constexpr int kTileInts = 8192;  // table entries staged at a time
constexpr int kNearPages = 8192;

template <bool NEAR>
__global__ __launch_bounds__(kThreads) void page_advance_kernel(AdvanceArgs a) {
  __shared__ int32_t tile[kTileInts];
  __shared__ int32_t near_refs[NEAR ? kNearPages : 1], near_table[NEAR ? kTileInts : 1];
  __shared__ int32_t len[kMaxRows], from[kMaxRows], need[kMaxRows + 1], mine[kMaxRows];
  __shared__ uint8_t shared_page[kMaxRows];
  __shared__ int part[kThreads / 64];
  __shared__ int copies;
  __shared__ unsigned long long lost;  // pages in columns that the table does not have, and those missing since an earlier step
  const int tid = threadIdx.x;
  const int64_t room = (int64_t)a.cols * a.page;
  auto sync = [&]() {
    if (NEAR) __syncthreads();
    else group_sync();
  };
  auto ref_at = [&](int p) { return NEAR ? near_refs[p] : ref_load(a.refs_out + p); };
  auto change = [&](int p, int v) {
    if (NEAR) atomicAdd(near_refs + p, v);
    else ref_add(a.refs_out + p, v);
  };
  auto entry = [&](int64_t e) { return NEAR ? near_table[e] : a.table_out[e]; };
  auto set_entry = [&](int64_t e, int p) {
    if (NEAR) near_table[e] = p;
    else a.table_out[e] = p;
  };
  if (NEAR)
    for (int p = tid; p < a.pages; p += kThreads) near_refs[p] = a.refs[p];
  else if (a.refs_out != a.refs)
    ref_copy(a.refs, a.refs_out, a.pages);
  int old_len = 0, tokens = a.tokens;
  int64_t start = 0;  // where the new tokens begin: at old_len, or beyond the table
  if (tid < a.rows) {
    if (a.row_tokens) {
      const int n = a.row_tokens[tid];
      tokens = n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : n;
    }
    int par = a.parents ? a.parents[tid] : tid;
    par = par >= 0 && par < a.rows ? par : -1;
    from[tid] = par;
    const int n = par >= 0 ? a.lengths[par] : 0;
    old_len = n < 0 ? 0 : n > room ? (int)room : n;
    start = a.over || n < old_len ? old_len : n;
    len[tid] = old_len;
    shared_page[tid] = 0;
  }
  if (tid == 0) copies = 0, lost = 0;
  sync();
  // rows take their parents' pages up to the parents' lengths, a block of
  // columns of every row at a time (outputs may be the inputs)
  const int width = kTileInts / a.rows < a.cols ? kTileInts / a.rows : a.cols;
  for (int c0 = 0; c0 < a.cols; c0 += width) {
    const int n = a.cols - c0 < width ? a.cols - c0 : width, all = a.rows * n;
    for (int e = tid; e < all; e += kThreads) tile[e] = a.table[(int64_t)(e / n) * a.cols + c0 + e % n];
    __syncthreads();
    for (int e = tid; e < all; e += kThreads) {
      const int i = e / n, c = e % n, par = from[i];
      int old = tile[e], now = par >= 0 && (int64_t)(c0 + c) * a.page < len[i] ? tile[par * n + c] : -1;
      old = old >= 0 && old < a.pages ? old : -1;
      now = now >= 0 && now < a.pages ? now : -1;
      if (now != old) {
        if (now >= 0) change(now, 1);
        if (old >= 0) change(old, -1);
      }
      set_entry((int64_t)i * a.cols + c0 + c, now);
    }
    __syncthreads();
  }
  sync();
  // the page that a row writes next, where it is partly filled and another row holds it too
  int c0 = 0, used = 0;
  if (tid < a.rows) {
    c0 = old_len / a.page, used = old_len % a.page;
    int p = -1;
    if (tokens > 0 && used > 0) {
      p = entry((int64_t)tid * a.cols + c0);
      // the positions before are lost, and a page now would have their places hold anything
      if (p < 0) atomicAdd(&lost, 1ull);
    }
    mine[tid] = p >= 0 && ref_at(p) > 1 ? p : -1;
  }
  __syncthreads();
  // a wave for a row, against all others (1024 rows and no new page: 54 us; with
  // a thread for every pair 212)
  for (int i = tid >> 6; i < a.rows; i += kThreads / 64) {
    const int p = mine[i], n = len[i];
    if (p < 0) continue;
    const int c = n / a.page;
    for (int j = tid & 63; j < a.rows; j += 64)
      if (len[j] > n || (len[j] == n && j < i))
        if (entry((int64_t)j * a.cols + c) == p) shared_page[i] = 1;
  }
  __syncthreads();
  // pages that a row needs: a copy's, then those of columns first .. last
  int wants = 0, first = 0;
  bool copy = false;
  if (tid < a.rows) {
    copy = shared_page[tid];
    first = c0 + (used > 0);
    const int64_t end = start + tokens;
    int64_t last = tokens > 0 ? (end - 1) / a.page : -1;
    if (last >= a.cols) {
      const int64_t from_col = start / a.page;
      atomicAdd(&lost, (unsigned long long)(last - (from_col < a.cols ? a.cols : from_col) + 1));
      last = a.cols - 1;
    }
    wants = copy + (last >= first ? (int)(last - first + 1) : 0);
    const int64_t cut = a.over ? room : INT32_MAX;
    a.lengths_out[tid] = (int)(end < cut ? end : cut);
    if (a.over) a.over[tid] = end <= room ? 0 : (int)(end < INT32_MAX ? end - room : INT32_MAX - room);
  }
  int total;
  const int mark = scan1024(wants, part, &total);
  if (tid < a.rows) need[tid] = mark, from[tid] = copy;
  if (tid == 0) need[a.rows] = total;
  __syncthreads();
  // free pages in ascending order; the page of rank k goes to the row whose
  // share of the ranks holds k
  int found = 0;
  auto give = [&](int p, int k) {
    int lo = 0, hi = a.rows;  // need[lo] <= k < need[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (need[mid] <= k) lo = mid; else hi = mid;
    }
    const int n0 = len[lo] / a.page, u = len[lo] % a.page;
    int nth = k - need[lo], col;
    if (from[lo] && nth == 0) {
      col = n0;
      const int at = atomicAdd(&copies, 1);
      Copy* c = reinterpret_cast<Copy*>(plan_copies(a.plan)) + at;
      c->src = mine[lo], c->dst = p, c->used = u;
      change(mine[lo], -1);
    } else {
      col = n0 + (u > 0) + nth - from[lo];
    }
    set_entry((int64_t)lo * a.cols + col, p);
    if (NEAR) near_refs[p] = 1;
    else ref_store(a.refs_out + p, 1);
  };
  constexpr int kEach = NEAR ? 1 : 4;  // pages of a thread at a time, next to each other (70000 to look through: 33 us, one by one 65)
  for (int p0 = 0; p0 < a.pages && found < total; p0 += kEach * kThreads) {
    const int p = p0 + kEach * tid;
    bool is_free[kEach];
    int mine_free = 0, n;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine_free += is_free[i] = p + i < a.pages && ref_at(p + i) <= 0;
    int k = found + scan1024(mine_free, part, &n);
    found += n;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (is_free[i]) {
        if (k < total) give(p + i, k);
        ++k;
      }
  }
  // a copy that got no page: the row loses its hold
  if (tid < a.rows && copy && mark >= found) {
    set_entry((int64_t)tid * a.cols + c0, -1);
    change(mine[tid], -1);
  }
  __syncthreads();
  if (NEAR) {
    for (int e = tid; e < a.rows * a.cols; e += kThreads) a.table_out[e] = near_table[e];
    for (int p = tid; p < a.pages; p += kThreads) a.refs_out[p] = near_refs[p];
  }
  if (tid == 0) {
    a.plan[0] = copies;
    const unsigned long long missing = lost + (total > found ? total - found : 0);
    a.short_pages[0] = missing < INT32_MAX ? (int)missing : INT32_MAX;
    if (a.missing) {
      const unsigned long long sum = missing + (a.missing[0] < 0 ? 0 : a.missing[0]);
      a.missing[0] = sum < INT32_MAX ? (int)sum : INT32_MAX;
    }
  }
}

// ---------------------------------------------------------------------------
// give back
// ---------------------------------------------------------------------------

struct FreeArgs {
  const int32_t *table, *lengths, *refs;
  const uint8_t* keep;
  int32_t *table_out, *lengths_out, *refs_out;
  int rows, cols, pages, page, window, sinks;
};

template <bool NEAR>
__global__ __launch_bounds__(kThreads) void page_free_kernel(FreeArgs a) {
  __shared__ int32_t near_refs[NEAR ? kNearPages : 1];
  const int tid = threadIdx.x;
  if (NEAR) {
    for (int p = tid; p < a.pages; p += kThreads) near_refs[p] = a.refs[p];
    __syncthreads();
  } else {
    if (a.refs_out != a.refs) ref_copy(a.refs, a.refs_out, a.pages);
    group_sync();
  }
  const int64_t all = (int64_t)a.rows * a.cols;
  for (int64_t e = tid; e < all; e += kThreads) {
    const int i = NEAR ? (int)((unsigned)e / (unsigned)a.cols) : (int)(e / a.cols), c = (int)(e - (int64_t)i * a.cols);
    const int old = a.table[e];
    const bool valid = old >= 0 && old < a.pages;
    bool drop = a.keep && !a.keep[i];
    if (!drop && a.window > 0)
      drop = (int64_t)c * a.page >= a.sinks && (int64_t)(c + 1) * a.page <= (int64_t)a.lengths[i] - a.window + 1;
    if (drop && valid) {
      if (NEAR) atomicAdd(near_refs + old, -1);
      else ref_add(a.refs_out + old, -1);
    }
    a.table_out[e] = valid && !drop ? old : -1;
  }
  __syncthreads();  // lengths_out may be lengths, which all of a row's threads read above
  if (NEAR)
    for (int p = tid; p < a.pages; p += kThreads) a.refs_out[p] = near_refs[p];
  for (int i = tid; i < a.rows; i += kThreads) {
    const int n = a.lengths[i];
    a.lengths_out[i] = a.keep && !a.keep[i] ? 0 : n;
  }
}

// ---------------------------------------------------------------------------
// move together
// ---------------------------------------------------------------------------

struct CompactArgs {
  const int32_t *refs, *table;
  int32_t *refs_out, *table_out, *plan, *map;
  int64_t entries;
  int pages, page;
};

constexpr int64_t kNearEntries = 1 << 15;  // of a table that the same work-group writes anew

// Counts, moves and map in LDS, the table too: no second launch for it.
__global__ __launch_bounds__(kThreads) void page_compact_near_kernel(CompactArgs a) {
  __shared__ int32_t refs[kNearPages], map[kNearPages], from[kNearPages / 2], to[kNearPages / 2];
  __shared__ int part[kThreads / 64];
  const int tid = threadIdx.x;
  int mine = 0, live;
  for (int p = tid; p < a.pages; p += kThreads) {
    const int n = a.refs[p];
    refs[p] = n;
    mine += n > 0;
  }
  scan1024(mine, part, &live);
  // the k-th free place below `live` takes the k-th page in use beyond it
  int free_before = 0, high_before = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kThreads) {
    const int p = p0 + tid;
    const bool used = p < a.pages && refs[p] > 0;
    const bool hole = p < live && !used, high = used && p >= live;
    int n;
    const int k = scan1024(hole ? 1 : high ? 1 << 16 : 0, part, &n);
    if (hole) to[free_before + (k & 0xFFFF)] = p;
    if (high) from[high_before + (k >> 16)] = p;
    if (p < a.pages) map[p] = p;
    free_before += n & 0xFFFF, high_before += n >> 16;
  }
  __syncthreads();
  Copy* copies = reinterpret_cast<Copy*>(plan_copies(a.plan));
  for (int k = tid; k < high_before; k += kThreads) {
    const int s = from[k], d = to[k];
    copies[k] = Copy{s, d, a.page};
    map[s] = d;
    refs[d] = refs[s], refs[s] = 0;  // no page is in two moves
  }
  __syncthreads();
  for (int p = tid; p < a.pages; p += kThreads) a.refs_out[p] = refs[p];
  for (int e = tid; e < a.entries; e += kThreads) {
    const int p = a.table[e];
    a.table_out[e] = p >= 0 && p < a.pages ? map[p] : -1;
  }
  if (tid == 0) a.plan[0] = high_before;
}

__global__ __launch_bounds__(kThreads) void page_compact_kernel(CompactArgs a) {
  __shared__ int part[kThreads / 64];
  const int tid = threadIdx.x;
  int mine = 0, live;
  for (int p = tid; p < a.pages; p += kThreads) mine += a.refs[p] > 0;
  scan1024(mine, part, &live);
  // the k-th free place below `live` takes the k-th page in use beyond it
  Copy* copies = reinterpret_cast<Copy*>(plan_copies(a.plan));
  int free_before = 0, high_before = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kThreads) {
    const int p = p0 + tid;
    const bool used = p < a.pages && a.refs[p] > 0;
    const bool hole = p < live && !used, high = used && p >= live;
    int n;
    const int k = scan1024(hole ? 1 : high ? 1 << 16 : 0, part, &n);
    if (hole) copies[free_before + (k & 0xFFFF)].dst = p;
    if (high) copies[high_before + (k >> 16)].src = p;
    if (p < a.pages) a.map[p] = p;
    free_before += n & 0xFFFF, high_before += n >> 16;
  }
  group_sync();
  if (a.refs_out != a.refs) ref_copy(a.refs, a.refs_out, a.pages);
  group_sync();
  for (int k = tid; k < high_before; k += kThreads) {
    const int s = copies[k].src, d = copies[k].dst;
    copies[k].used = a.page;
    a.map[s] = d;
    const int n = a.refs[s];
    a.refs_out[d] = n;
    a.refs_out[s] = 0;
  }
  if (tid == 0) a.plan[0] = high_before;
}

__global__ __launch_bounds__(256) void page_remap_kernel(const int32_t* table, int32_t* table_out, const int32_t* map,
                                                         int64_t entries, int pages) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= entries) return;
  const int p = table[e];
  table_out[e] = p >= 0 && p < pages ? map[p] : -1;
}

// ---------------------------------------------------------------------------
// new tokens
// ---------------------------------------------------------------------------

// Where a row's tokens end, as the attention has it.
__device__ __forceinline__ int64_t row_end(const qs_page_pool& pool, const int32_t* over, int64_t row) {
  const int64_t n = pool.lengths[row];
  return over && n == pool.cols * pool.page && over[row] > 0 ? n + over[row] : n;
}

struct AppendArgs {
  const uint16_t *k, *v;
  int64_t k_token, k_head, v_token, v_head, tokens;
  const int32_t *starts, *over;
  int rows, kv_heads, head_dim;
};

// Element address of position p of a row's page, or null.
__device__ __forceinline__ uint16_t* place(void* base, int64_t s_page, int64_t s_head, int64_t s_pos, const qs_page_pool& pool,
                                           int row, int64_t p, int head) {
  if (p < 0 || p >= pool.cols * pool.page) return nullptr;
  const int id = pool.table[row * pool.table_ld + p / pool.page];
  if (id < 0 || id >= pool.pages) return nullptr;
  return static_cast<uint16_t*>(base) + id * s_page + head * s_head + (p % pool.page) * s_pos;
}

// One thread per 8 elements of a head.  A token of 48 rows and 8 heads of 128:
// 3.1 us, a launch's time; 8192 tokens of one row 13.0 us, bound by memory (67
// MB, 5.2 TB/s).
__global__ __launch_bounds__(256) void page_append_kernel(qs_page_pool pool, AppendArgs a) {
  const int per = a.head_dim / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / (per * a.kv_heads);
  if (t >= a.tokens) return;
  const int rest = (int)(i % (per * a.kv_heads)), head = rest / per, d = rest % per * 8;
  int row = (int)t;
  int64_t back = 1;
  if (a.starts) {
    int lo = 0, hi = a.rows;  // the last row that starts at t or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid] <= t) lo = mid; else hi = mid;
    }
    row = lo;
    back = a.starts[row + 1] - t;
    if (a.starts[row] > t || back <= 0) return;
  }
  const int64_t p = row_end(pool, a.over, row) - back;
  if (uint16_t* to = place(pool.k, pool.k_page, pool.k_head, pool.k_pos, pool, row, p, head))
    *reinterpret_cast<uint4*>(to + d) = *reinterpret_cast<const uint4*>(a.k + t * a.k_token + head * a.k_head + d);
  if (uint16_t* to = place(pool.v, pool.v_page, pool.v_head, pool.v_pos, pool, row, p, head))
    *reinterpret_cast<uint4*>(to + d) = *reinterpret_cast<const uint4*>(a.v + t * a.v_token + head * a.v_head + d);
}

// One wave per head of one row, as qk_norm_rope_kernel: 3.1 us, a launch's
// time, for 48 rows of 64 and 8 heads.
__global__ __launch_bounds__(256) void page_append_rope_kernel(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                                               const uint16_t* qw, const uint16_t* kw,
                                                               const uint16_t* cos_t, const uint16_t* sin_t,
                                                               int64_t table_rows, uint16_t* q_out, qs_page_pool pool,
                                                               const int32_t* over, int nh, int nkv, float eps) {
  const LaneX lx = lane_x_init();
  const int b = blockIdx.x, hh = blockIdx.y * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
  if (hh >= nh + 2 * nkv) return;
  const int64_t pos = row_end(pool, over, b) - 1;
  // a row without tokens, or a position beyond the tables, has no rotation: its queries are zeros and nothing is stored
  const bool inside = pos >= 0 && pos < table_rows, isq = hh < nh;
  if (hh >= nh + nkv) {
    if (!inside) return;
    const int g = hh - nh - nkv;
    const uint16_t* src = v + ((int64_t)b * nkv + g) * 128;
    if (uint16_t* to = place(pool.v, pool.v_page, pool.v_head, pool.v_pos, pool, b, pos, g)) to[l] = src[l], to[l + 64] = src[l + 64];
    return;
  }
  const int g = isq ? hh : hh - nh;
  uint16_t o0 = 0, o1 = 0;
  if (inside) {
    const uint16_t* src = isq ? q + ((int64_t)b * nh + g) * 128 : k + ((int64_t)b * nkv + g) * 128;
    const uint16_t* w = isq ? qw : kw;
    norm_rope(bf(src[l]), bf(src[l + 64]), bf(w[l]), bf(w[l + 64]), load_rot(cos_t + pos * 128, sin_t + pos * 128, l), eps, lx, o0, o1);
  }
  uint16_t* to = isq ? q_out + ((int64_t)b * nh + g) * 128
                     : inside ? place(pool.k, pool.k_page, pool.k_head, pool.k_pos, pool, b, pos, g) : nullptr;
  if (to) to[l] = o0, to[l + 64] = o1;
}

int store_checks(const char* fn, const qs_page_store* s, Store& out) {
  QS_REQUIRE(s && s->data, "%s: null pointer", fn);
  QS_REQUIRE(s->planes >= 1 && s->pages >= 1 && s->pages <= INT32_MAX && s->kv_heads >= 1 && s->page >= 1 &&
                 s->page <= 4096 && s->row_bytes >= 16 && s->row_bytes % 16 == 0 && s->row_bytes <= 65536,
             "%s: %lld planes of %lld pages, %d heads, %d positions of %lld bytes (a multiple of 16)", fn,
             (long long)s->planes, (long long)s->pages, s->kv_heads, s->page, (long long)s->row_bytes);
  QS_SUPPORTED(s->planes * s->kv_heads * ((s->page * s->row_bytes + kPiece - 1) / kPiece) <= INT32_MAX,
               "%s: %lld planes of %d heads", fn, (long long)s->planes, s->kv_heads);
  QS_REQUIRE((reinterpret_cast<uintptr_t>(s->data) & 15) == 0, "%s: the store must be 16-byte aligned", fn);
  out = Store{static_cast<char*>(s->data), s->planes, s->pages, s->row_bytes, s->kv_heads, s->page};
  return QS_OK;
}

int table_checks(const char* fn, int64_t rows, int64_t cols, int64_t pages, int page) {
  QS_REQUIRE(rows >= 1 && cols >= 1 && cols <= (1 << 24) && pages >= 1 && pages <= INT32_MAX - kPageStep && page >= 1 &&
                 cols * page <= INT32_MAX - 65536,
             "%s: table of %lld x %lld, %lld pages of %d", fn, (long long)rows, (long long)cols, (long long)pages, page);
  return QS_OK;
}

int launch_copies(const Store& st, const int32_t* plan, int64_t most, hipStream_t stream) {
  hipLaunchKernelGGL(page_copy_kernel, copy_grid(st, most), dim3(256), 0, stream, st, plan);
  QS_LAUNCHED("page_copy_kernel");
  return QS_OK;
}

int pool_checks(const char* fn, const qs_page_pool* p, int64_t rows, int kv_heads, int head_dim) {
  QS_REQUIRE(p && p->k && p->v && p->table && p->lengths, "%s: null pointer", fn);
  QS_REQUIRE(rows >= 1 && rows <= (1 << 20) && kv_heads >= 1 && kv_heads <= 65535 && head_dim >= 8 && head_dim % 8 == 0 &&
                 head_dim <= 4096 && p->pages >= 1 && p->pages <= INT32_MAX && p->page >= 1 && p->cols >= 1 &&
                 p->table_ld >= p->cols && p->cols * p->page <= INT32_MAX,
             "%s: rows %lld, %d heads of %d, %lld pages of %d, table of %lld columns", fn, (long long)rows, kv_heads,
             head_dim, (long long)p->pages, p->page, (long long)p->cols);
  const int64_t st[6] = {p->k_page, p->k_head, p->k_pos, p->v_page, p->v_head, p->v_pos};
  for (int64_t x : st) QS_REQUIRE(x >= 0 && x % 8 == 0, "%s: pool strides must be multiples of 8 elements, got %lld", fn, (long long)x);
  QS_REQUIRE(((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15) == 0,
             "%s: the pools must be 16-byte aligned", fn);
  return QS_OK;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" int qs_page_append(const void* k, const void* v, int64_t tokens, int64_t rows, int kv_heads, int head_dim,
                              int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, const int32_t* starts,
                              const qs_page_pool* pool, qs_stream_t stream) {
  return qs_page_append_over(k, v, tokens, rows, kv_heads, head_dim, k_token, k_head, v_token, v_head, starts, pool,
                             nullptr, stream);
}

extern "C" int qs_page_append_over(const void* k, const void* v, int64_t tokens, int64_t rows, int kv_heads, int head_dim,
                                   int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                   const int32_t* starts, const qs_page_pool* pool, const int32_t* over,
                                   qs_stream_t stream) {
  if (tokens == 0 || rows == 0) return QS_OK;
  if (const int rc = pool_checks("qs_page_append", pool, rows, kv_heads, head_dim)) return rc;
  QS_REQUIRE(k && v && tokens >= 1 && (starts || tokens == rows), "qs_page_append: %lld tokens of %lld rows",
             (long long)tokens, (long long)rows);
  const int64_t st[4] = {k_token, k_head, v_token, v_head};
  for (int64_t x : st) QS_REQUIRE(x >= 0 && x % 8 == 0, "qs_page_append: strides must be multiples of 8 elements, got %lld", (long long)x);
  QS_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
             "qs_page_append: keys and values must be 16-byte aligned");
  const int64_t threads = tokens * kv_heads * (head_dim / 8);
  QS_REQUIRE(threads <= ((int64_t)INT32_MAX << 8), "qs_page_append: %lld tokens", (long long)tokens);
  const AppendArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_token, k_head, v_token, v_head,
                     tokens, starts, over, (int)rows, kv_heads, head_dim};
  hipLaunchKernelGGL(page_append_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, as_stream(stream), *pool, a);
  QS_LAUNCHED("page_append_kernel");
  return QS_OK;
}

extern "C" int qs_page_append_rope(const void* q, const void* k, const void* v, const void* q_norm_w,
                                   const void* k_norm_w, const void* cos_table, const void* sin_table,
                                   int64_t table_rows, void* q_out, int64_t rows, int nh, int nkv, int head_dim,
                                   const qs_page_pool* pool, float eps, qs_stream_t stream) {
  return qs_page_append_rope_over(q, k, v, q_norm_w, k_norm_w, cos_table, sin_table, table_rows, q_out, rows, nh, nkv,
                                  head_dim, pool, nullptr, eps, stream);
}

extern "C" int qs_page_append_rope_over(const void* q, const void* k, const void* v, const void* q_norm_w,
                                        const void* k_norm_w, const void* cos_table, const void* sin_table,
                                        int64_t table_rows, void* q_out, int64_t rows, int nh, int nkv, int head_dim,
                                        const qs_page_pool* pool, const int32_t* over, float eps, qs_stream_t stream) {
  if (rows == 0) return QS_OK;
  QS_REQUIRE(q && k && v && q_norm_w && k_norm_w && cos_table && sin_table && q_out, "qs_page_append_rope: null pointer");
  QS_SUPPORTED(head_dim == 128, "qs_page_append_rope: head_dim %d (128 only)", head_dim);
  if (const int rc = pool_checks("qs_page_append_rope", pool, rows, nkv, head_dim)) return rc;
  QS_REQUIRE(nh >= 1 && nh % nkv == 0 && nh <= 65535 && rows <= INT32_MAX && table_rows >= 1,
             "qs_page_append_rope: heads %d / %d, tables of %lld rows", nh, nkv, (long long)table_rows);
  hipLaunchKernelGGL(page_append_rope_kernel, dim3((unsigned)rows, (unsigned)((nh + 2 * nkv + 3) / 4)), dim3(256), 0,
                     as_stream(stream), static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                     static_cast<const uint16_t*>(v), static_cast<const uint16_t*>(q_norm_w),
                     static_cast<const uint16_t*>(k_norm_w), static_cast<const uint16_t*>(cos_table),
                     static_cast<const uint16_t*>(sin_table), table_rows, static_cast<uint16_t*>(q_out), *pool, over, nh, nkv, eps);
  QS_LAUNCHED("page_append_rope_kernel");
  return QS_OK;
}

extern "C" size_t qs_page_advance_workspace_bytes(int64_t rows) {
  return rows < 1 ? 0 : 16 + (size_t)rows * sizeof(Copy);
}

extern "C" int qs_page_advance(const qs_page_store* store, const int32_t* table, const int32_t* lengths,
                               const int32_t* refs, const int32_t* parents, int64_t rows, int64_t cols, int tokens,
                               int32_t* table_out, int32_t* lengths_out, int32_t* refs_out, int32_t* short_pages,
                               void* workspace, size_t workspace_bytes, qs_stream_t stream) {
  return qs_page_advance_rows(store, table, lengths, refs, parents, rows, cols, tokens, nullptr, table_out, lengths_out,
                              refs_out, short_pages, workspace, workspace_bytes, stream);
}

extern "C" int qs_page_advance_rows(const qs_page_store* store, const int32_t* table, const int32_t* lengths,
                                    const int32_t* refs, const int32_t* parents, int64_t rows, int64_t cols, int tokens,
                                    const int32_t* row_tokens, int32_t* table_out, int32_t* lengths_out,
                                    int32_t* refs_out, int32_t* short_pages, void* workspace, size_t workspace_bytes,
                                    qs_stream_t stream) {
  return qs_page_advance_over(store, table, lengths, refs, parents, rows, cols, tokens, row_tokens, table_out, lengths_out,
                              refs_out, short_pages, nullptr, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int qs_page_advance_over(const qs_page_store* store, const int32_t* table, const int32_t* lengths,
                                    const int32_t* refs, const int32_t* parents, int64_t rows, int64_t cols, int tokens,
                                    const int32_t* row_tokens, int32_t* table_out, int32_t* lengths_out,
                                    int32_t* refs_out, int32_t* short_pages, int32_t* over, int32_t* missing,
                                    void* workspace, size_t workspace_bytes, qs_stream_t stream) {
  Store st;
  if (const int rc = store_checks("qs_page_advance", store, st)) return rc;
  if (const int rc = table_checks("qs_page_advance", rows, cols, st.pages, st.page)) return rc;
  QS_SUPPORTED(rows <= kMaxRows && rows * cols <= INT32_MAX, "qs_page_advance: %lld rows of %lld columns (at most %d, 2^31 entries)",
               (long long)rows, (long long)cols, kMaxRows);
  QS_REQUIRE(table && lengths && refs && table_out && lengths_out && refs_out && short_pages, "qs_page_advance: null pointer");
  QS_REQUIRE(tokens >= 0 && tokens <= (1 << 30), "qs_page_advance: %d tokens", tokens);
  QS_REQUIRE(workspace && workspace_bytes >= qs_page_advance_workspace_bytes(rows) && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "qs_page_advance: workspace of %zu bytes (16-byte aligned), %zu needed", workspace_bytes,
             qs_page_advance_workspace_bytes(rows));
  int32_t* plan = static_cast<int32_t*>(workspace);
  const AdvanceArgs a{table, lengths, refs, parents, row_tokens, table_out, lengths_out, refs_out, short_pages, plan,
                      over, missing, (int)rows, (int)cols, (int)st.pages, st.page, tokens};
  if (st.pages <= kNearPages && rows * cols <= kTileInts) hipLaunchKernelGGL(page_advance_kernel<true>, dim3(1), dim3(kThreads), 0, as_stream(stream), a);
  else hipLaunchKernelGGL(page_advance_kernel<false>, dim3(1), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("page_advance_kernel");
  return launch_copies(st, plan, rows, as_stream(stream));
}

extern "C" int qs_page_free(const int32_t* table, const int32_t* lengths, const int32_t* refs, const uint8_t* keep,
                            int64_t rows, int64_t cols, int64_t pages, int page, int window, int sinks,
                            int32_t* table_out, int32_t* lengths_out, int32_t* refs_out, qs_stream_t stream) {
  if (const int rc = table_checks("qs_page_free", rows, cols, pages, page)) return rc;
  QS_REQUIRE(rows <= (1 << 20) && table && lengths && refs && table_out && lengths_out && refs_out, "qs_page_free: null pointer or %lld rows", (long long)rows);
  QS_REQUIRE(window >= 0 && sinks >= 0 && (sinks == 0 || window > 0), "qs_page_free: window %d, sinks %d", window, sinks);
  const FreeArgs a{table, lengths, refs, keep, table_out, lengths_out, refs_out, (int)rows, (int)cols, (int)pages, page, window, sinks};
  if (pages <= kNearPages && rows * cols <= INT32_MAX) hipLaunchKernelGGL(page_free_kernel<true>, dim3(1), dim3(kThreads), 0, as_stream(stream), a);
  else hipLaunchKernelGGL(page_free_kernel<false>, dim3(1), dim3(kThreads), 0, as_stream(stream), a);
  QS_LAUNCHED("page_free_kernel");
  return QS_OK;
}

extern "C" size_t qs_page_compact_workspace_bytes(int64_t pages) {
  return pages < 1 ? 0 : 16 + (size_t)pages * (sizeof(Copy) + sizeof(int32_t));
}

extern "C" int qs_page_compact(const qs_page_store* store, const int32_t* table, const int32_t* refs, int64_t rows,
                               int64_t cols, int32_t* table_out, int32_t* refs_out, void* workspace,
                               size_t workspace_bytes, qs_stream_t stream) {
  Store st;
  if (const int rc = store_checks("qs_page_compact", store, st)) return rc;
  if (const int rc = table_checks("qs_page_compact", rows, cols, st.pages, st.page)) return rc;
  QS_REQUIRE(rows <= (1 << 20) && table && refs && table_out && refs_out, "qs_page_compact: null pointer or %lld rows", (long long)rows);
  const size_t need = qs_page_compact_workspace_bytes(st.pages);
  QS_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "qs_page_compact: workspace of %zu bytes (16-byte aligned), %zu needed", workspace_bytes, need);
  int32_t* plan = static_cast<int32_t*>(workspace);
  int32_t* map = plan + 4 + 3 * st.pages;
  const int64_t entries = rows * cols;
  const CompactArgs a{refs, table, refs_out, table_out, plan, map, entries, (int)st.pages, st.page};
  if (st.pages <= kNearPages && entries <= kNearEntries) {
    hipLaunchKernelGGL(page_compact_near_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), a);
    QS_LAUNCHED("page_compact_near_kernel");
  } else {
    hipLaunchKernelGGL(page_compact_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), a);
    QS_LAUNCHED("page_compact_kernel");
    hipLaunchKernelGGL(page_remap_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, as_stream(stream), table,
                       table_out, map, entries, (int)st.pages);
    QS_LAUNCHED("page_remap_kernel");
  }
  return launch_copies(st, plan, st.pages, as_stream(stream));
}

extern "C" int qs_page_copy(const qs_page_store* store, const int32_t* src, const int32_t* dst, int64_t count,
                            qs_stream_t stream) {
  if (count == 0) return QS_OK;
  Store st;
  if (const int rc = store_checks("qs_page_copy", store, st)) return rc;
  QS_REQUIRE(src && dst && count >= 1 && count <= INT32_MAX - kCopyStep, "qs_page_copy: null pointer or %lld pairs", (long long)count);
  hipLaunchKernelGGL(page_list_kernel, copy_grid(st, count), dim3(256), 0, as_stream(stream), st, src, dst, (int)count);
  QS_LAUNCHED("page_list_kernel");
  return QS_OK;
}
