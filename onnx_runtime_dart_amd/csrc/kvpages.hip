// Pages of the quantised KV cache: copied, their rows moved together, shared between sequences
// and handed out.
//
// A page's codes of keys, of values and its scales are three runs of memory, so a copy is one read
// and one write of them.  Rows that move within a sequence only ever move down, in order: a
// workgroup per head takes them 32 or 128 at a time, reads all before it writes any, and nothing
// that it writes is read later (row j comes from kept[j] >= j, later rows from beyond it).  Long
// lists go through the workspace, twice the traffic but all workgroups at once.
//
// Bound by bytes where there are many: pages of 4 sequences of 7001 to 8192 e4m3 tokens of 8 heads of
// 128 copied in 28 us (4.9 TB/s, read and written), half of their tokens moved in 15 + 13 us and 5 for
// the lists (in order, without the workspace: 118); else by chains of loads: 25 rows of 64 sequences
// 6.4 us, a fork 2.3 to 2.8, 64 copies of pages 4.4.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_common.h"

namespace {

// -------------------------------------------------------------------- copies

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Units of 16 bytes of a page: its codes of keys (as many of values), its scales.
struct PageUnits {
  int64_t codes, all;
};
__host__ __device__ inline PageUnits page_units(const mg_kv_cache &c) {
  const int64_t codes = ((int64_t)c.kv_heads * c.dp * kv_bits(c.fmt) / 8 << c.plog) / 16;
  return PageUnits{codes, 2 * codes + ((int64_t)c.kv_heads * kv_scales(c.fmt) * 4 << c.plog) / 16};
}
constexpr int kPiece = 1024;  // units that a workgroup copies: four a thread
__host__ __device__ inline int page_pieces(const mg_kv_cache &c) {
  return (int)((page_units(c).all + kPiece - 1) / kPiece);
}
// A workgroup's piece of a page's copy.
__device__ inline void copy_piece(const mg_kv_cache &c, int64_t src, int64_t dst, int piece) {
  const PageUnits n = page_units(c);
  auto unit = [&](int64_t page, int64_t i) {
    void *p = i < n.codes ? (void *)c.k : i < 2 * n.codes ? (void *)c.v : (void *)c.sc;
    const int64_t size = i < 2 * n.codes ? n.codes : n.all - 2 * n.codes;
    const int64_t at = i < n.codes ? i : i < 2 * n.codes ? i - n.codes : i - 2 * n.codes;
    return static_cast<u32x4 *>(p) + page * size + at;
  };
  const int64_t first = (int64_t)piece * kPiece + threadIdx.x;
  u32x4 x[4];
#pragma unroll
  for (int u = 0; u < 4; u++) x[u] = *unit(src, std::min(first + 256 * u, n.all - 1));
#pragma unroll
  for (int u = 0; u < 4; u++)
    if (first + 256 * u < n.all) *unit(dst, first + 256 * u) = x[u];
}

struct Pairs {
  mg_kv_cache c;
  const int32_t *src, *dst;
  int64_t n;
  int pieces;
  uint32_t *marks;  // [pages], or null (up to 1024 pairs): each workgroup looks through them
};
// Of a page: a pair's src (its dst another page), a pair's dst (its src another), and how many pairs'
// dst in all.
constexpr uint32_t kIsSrc = 1, kIsDst = 2, kOneDst = 4;
// Whether pair i is to be copied, by the whole workgroup; *bad: it is refused.
__device__ inline bool pair_ok(const Pairs &a, int64_t i, bool *bad) {
  const int s = a.src[i], d = a.dst[i];
  *bad = false;
  if ((s < 0 && d < 0) || s == d) return false;
  bool clash = s < 0 || d < 0 || s >= a.c.pages || d >= a.c.pages;
  if (a.marks) {
    if (!clash) {
      const uint32_t on = a.marks[d];
      clash = on / kOneDst > 1 || (on & kIsSrc) || (a.marks[s] & kIsDst);
    }
    *bad = clash;
    return !clash;
  }
  for (int64_t j = threadIdx.x; j < a.n; j += 256) {
    const int sj = a.src[j], dj = a.dst[j];
    if (j != i && !(sj < 0 && dj < 0)) clash |= dj == d || (sj != dj && (sj == d || dj == s));
  }
  *bad = __syncthreads_or(clash);
  return !*bad;
}

__global__ __launch_bounds__(256) void k_clear_marks(const Pairs a) {
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p < a.c.pages) a.marks[p] = 0;
}
__global__ __launch_bounds__(256) void k_mark(const Pairs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n) return;
  const int s = a.src[i], d = a.dst[i];
  if (s < 0 && d < 0) return;
  if (s != d && s >= 0 && s < a.c.pages) atomicOr(a.marks + s, kIsSrc);
  if (s != d && d >= 0 && d < a.c.pages) atomicOr(a.marks + d, kIsDst);
  if (d >= 0 && d < a.c.pages) atomicAdd(a.marks + d, kOneDst);
}
__global__ __launch_bounds__(256) void k_copy_pages(const Pairs a) {
  const int64_t i = blockIdx.x / a.pieces;
  const int piece = blockIdx.x % a.pieces;
  bool bad;
  const bool ok = pair_ok(a, i, &bad);
  if (bad && piece == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
  if (ok) copy_piece(a.c, a.src[i], a.dst[i], piece);
}

// ------------------------------------------------------------------- compact

// A sequence's rows to move: j0 .. count - 1 (rows before j0 stay where they are).
struct Moves {
  int j0, count;
  int bad, unused;  // bad: the sequence is refused (count is 0)
};
struct Compact {
  mg_kv_cache c;
  mg_seq_batch s;
  const int32_t *kept, *count;
  int32_t *past_out;
  // Staged (long lists): the sequences' moves, and rows on their way [sequence][head][keys or
  // values][chunk], then their scales.
  Moves *moves;
  uint8_t *rows;
  float *scales;
  int chunks;
};

// By the whole workgroup.
__device__ inline Moves moves_of(const Compact &a, const kv_seq &q, int64_t b) {
  const int count = a.count[b];
  bool bad = q.bad || count < 0 || count > q.n;
  int same = 0;
  if (!bad) {
    const int32_t *kept = a.kept + q.start;
#pragma unroll 4
    for (int j = threadIdx.x; j < count; j += 256) {
      const int k = kept[j], before = kept[max(j - 1, 0)];
      bad |= k < 0 || k >= q.n || (j > 0 && k <= before);
      same += k == j;
    }
  }
  // (Rising numbers from 0 on: once one is beyond its place, all are.)
  __shared__ int sum;
  if (threadIdx.x == 0) sum = 0;
  bad = __syncthreads_or(bad);
  if (same) atomicAdd(&sum, same);
  __syncthreads();
  return bad ? Moves{0, 0, 1, 0} : Moves{sum, count, 0, 0};
}

// Nibbles of a token's values in the dword of a pair of dims (see kv_common.h).
__device__ inline int v4_shift(int t) { return 4 * (4 * (t & 1) + (t >> 1)); }
template <bool INT4>
__device__ inline uint32_t token_of(uint32_t w, int t) {
  return INT4 ? w >> v4_shift(t) & 0x0f0fu : w >> 8 * t & 0xffu;
}
template <bool INT4>
__device__ inline uint32_t token_to(uint32_t x, int t) {
  return INT4 ? x << v4_shift(t) : x << 8 * t;
}

// IN_ORDER: a workgroup takes all of a sequence's rows of a head, ROWS at a time.  GATHER and
// SCATTER: one such chunk a workgroup, through the workspace.  blockIdx: head, sequence, keys or
// values (and twice the chunk).
enum { IN_ORDER, GATHER, SCATTER };
template <bool INT4, int ROWS, int PHASE>
__global__ __launch_bounds__(256) void k_compact(const Compact a) {
  constexpr int kUnits = ROWS / 16;  // vectors of 16 bytes a thread: rows are at most 256 bytes
  __shared__ int64_t from[ROWS], to[ROWS];  // places in the cache, -1: none
  const int64_t b = blockIdx.y;
  const int h = blockIdx.x, kind = blockIdx.z & 1, chunk = blockIdx.z >> 1;
  const kv_seq q = kv_sequence(a.s, b);
  const Moves m = PHASE == IN_ORDER ? moves_of(a, q, b) : a.moves[b];
  if (PHASE == IN_ORDER && h == 0 && kind == 0 && threadIdx.x == 0) {
    if (m.bad) atomicOr(a.c.refused, 1);
    if (a.past_out) a.past_out[b] = a.s.past[b] + m.count;
  }
  if (m.j0 >= m.count) return;
  const int page = 1 << a.c.plog, mask = page - 1, heads = a.c.kv_heads;
  const int rb = a.c.dp * (INT4 ? 4 : 8) / 8;  // bytes of a vector's codes
  auto place = [&](int64_t pos) {
    const int64_t id = kv_page(a.s, b, pos, a.c.plog, a.c.pages);
    return id < 0 ? (int64_t)-1 : ((id * heads + h) << a.c.plog) + (pos & mask);
  };
  // Groups of four places, from the first that changes on.
  const int64_t g1 = ((int64_t)q.past + m.count + 3) >> 2;
  int64_t g = ((q.past + m.j0) >> 2) + (PHASE == IN_ORDER ? 0 : (int64_t)chunk * (ROWS / 4));
  const int64_t staged = ((b * heads + h) * 2 + kind) * a.chunks + chunk;
  for (; g < g1; g += ROWS / 4) {
    if (PHASE == IN_ORDER) __syncthreads();
    if (threadIdx.x < ROWS) {
      const int64_t pos = 4 * g + threadIdx.x, j = pos - q.past;
      int64_t t = -1, f = -1;
      if (j >= m.j0 && j < m.count) {
        t = place(pos);
        f = place((int64_t)q.past + a.kept[q.start + j]);
        if (t < 0 || f < 0) {
          t = f = -1;
          atomicOr(a.c.refused, 1);
        }
      }
      to[threadIdx.x] = t;
      from[threadIdx.x] = f;
    }
    __syncthreads();
    const int rows = (int)std::min<int64_t>(ROWS, 4 * (g1 - g)), units = rows * rb / 16;
    // Scales: (page, head) block, kind, token.
    const int sc = kind + 2 * ((int)threadIdx.x / ROWS), row = threadIdx.x % ROWS;
    const bool scaled = (int)threadIdx.x < (INT4 ? 2 * ROWS : ROWS) && to[row] >= 0;
    auto scale = [&](int64_t at) {
      return a.c.sc + ((at >> a.c.plog) * kv_scales(a.c.fmt) + sc) * page + (at & mask);
    };
    float *scale_ws = a.scales + staged * 2 * ROWS + threadIdx.x;
    u32x4 *row_ws = reinterpret_cast<u32x4 *>(a.rows + staged * ROWS * rb) + threadIdx.x;
    float s = 0.f;
    if (scaled) s = PHASE == SCATTER ? *scale_ws : *scale(from[row]);
    u32x4 x[kUnits];
    if (PHASE == SCATTER) {
#pragma unroll
      for (int u = 0; u < kUnits; u++)
        if (256 * u < units) x[u] = row_ws[256 * u];
    } else if (kind == 0) {
      const int vec = rb / 16;
#pragma unroll
      for (int u = 0; u < kUnits; u++) {
        if (256 * u >= units) break;
        const int i = 256 * u + threadIdx.x, r = min(i / vec, ROWS - 1);
        // (Rows that do not move read the cache's first.)
        const int64_t at = to[r] >= 0 ? from[r] * rb + 16 * (i % vec) : 0;
        x[u] = *reinterpret_cast<const u32x4 *>(a.c.k + at);
      }
    }
    // Values: dwords of four tokens, those of rows that move from where they are, the others kept.
    const int vec = rb / 4;  // vectors of four dwords of a group
    // The group (four places lie together) that gets rows in this call, -1: none.
    auto group = [&](int k) {
      int64_t g4 = -1;
#pragma unroll
      for (int t = 0; t < 4; t++) g4 = std::max(g4, to[4 * k + t] >> 2);
      return g4;
    };
    if (PHASE != SCATTER && kind == 1) {
#pragma unroll
      for (int u = 0; u < kUnits; u++) {
        if (256 * u >= units) break;
        const int i = 256 * u + threadIdx.x, k = min(i / vec, ROWS / 4 - 1), o = i % vec;
        const int64_t own = std::max<int64_t>(group(k), 0);
        x[u] = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const int64_t at = to[4 * k + t] >= 0 ? from[4 * k + t] : 4 * own + t;
          const u32x4 w = *reinterpret_cast<const u32x4 *>(a.c.v + (at >> 2) * 4 * rb + 16 * o);
          const int n = (int)(at & 3);
#pragma unroll
          for (int e = 0; e < 4; e++) x[u][e] |= token_to<INT4>(token_of<INT4>(w[e], n), t);
        }
      }
    }
    if (PHASE == GATHER) {
      if (scaled) *scale_ws = s;
#pragma unroll
      for (int u = 0; u < kUnits; u++)
        if (256 * u < units) row_ws[256 * u] = x[u];
      return;
    }
    if (PHASE == IN_ORDER) {  // all read before any is written
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
      if (256 * u >= units) break;
      const int i = 256 * u + threadIdx.x;
      if (i >= units) break;
      if (kind == 0) {
        const int r = i / (rb / 16);
        if (to[r] >= 0) *reinterpret_cast<u32x4 *>(a.c.k + to[r] * rb + 16 * (i % (rb / 16))) = x[u];
      } else {
        const int64_t own = group(i / vec);
        if (own >= 0) *reinterpret_cast<u32x4 *>(a.c.v + own * 4 * rb + 16 * (i % vec)) = x[u];
      }
    }
    if (scaled) *scale(to[row]) = s;
    if (PHASE == SCATTER) return;
  }
}

// The sequences' moves for the staged form, and their new lengths.
__global__ __launch_bounds__(256) void k_moves(const Compact a) {
  const int64_t b = blockIdx.x;
  const Moves m = moves_of(a, kv_sequence(a.s, b), b);
  if (threadIdx.x) return;
  if (m.bad) atomicOr(a.c.refused, 1);
  if (a.moves) a.moves[b] = m;
  if (a.past_out) a.past_out[b] = a.s.past[b] + m.count;
}

// ---------------------------------------------------------- shared and free pages

struct Fork {
  mg_kv_cache c;
  mg_seq_batch s;
  const int32_t *parent;
  int64_t out_batch, out_stride;
  int32_t *past_out, *table_out, *refs;
};
// The first out_batch workgroups: a new sequence each; the others: an old one's entries.
__global__ __launch_bounds__(256) void k_fork(const Fork a) {
  const int64_t i = blockIdx.x;
  if (i >= a.out_batch) {
    const int32_t *row = a.s.page_table + (i - a.out_batch) * a.s.table_stride;
    for (int64_t e = threadIdx.x; e < a.s.table_stride; e += 256) {
      const int id = row[e];
      if (id >= 0 && id < a.c.pages) atomicSub(a.refs + id, 1);
    }
    return;
  }
  const int p = a.parent[i];
  int64_t past = 0;
  bool bad = p >= a.s.batch;
  if (p >= 0 && !bad) {
    past = a.s.past[p];
    bad = past < 0 || past > a.s.max_len;
  }
  int64_t pages = (past + (1 << a.c.plog) - 1) >> a.c.plog;
  bad = bad || pages > a.s.table_stride || pages > a.out_stride;
  if (bad) past = pages = 0;
  if (threadIdx.x == 0) a.past_out[i] = (int32_t)past;
  for (int64_t e = threadIdx.x; e < a.out_stride; e += 256) {
    int id = -1;
    if (e < pages) {
      id = a.s.page_table[p * a.s.table_stride + e];
      if (id < 0 || id >= a.c.pages) {
        id = -1;
        bad = true;
      } else {
        atomicAdd(a.refs + id, 1);
      }
    }
    a.table_out[i * a.out_stride + e] = id;
  }
  if (bad) atomicOr(a.c.refused, 1);
}

constexpr int kRun = 4096;  // pages of a run
struct Fit {
  mg_kv_cache c;
  mg_seq_batch s;
  int32_t *table, *refs, *granted;
  int64_t nrun;
  // Workspace: a sequence's held pages (-1: refused), whether it takes a copy (1) or keeps a page that
  // earlier ones are to leave (2: not granted where free pages end before it), its first page among
  // those handed out, its copy's pages; the runs' free pages, then those before them.
  int32_t *held, *copy, *first, *need, *old, *own;
  int32_t *free;
};
// The pages that sequence b needs.
__device__ inline int64_t wanted(const Fit &a, const kv_seq &q) {
  return ((int64_t)q.past + q.n + (1 << a.c.plog) - 1) >> a.c.plog;
}

// The pages that a sequence keeps: those of its past and, of the ones behind, those that it needs
// and holds alone, up to the first that is not so.
__global__ __launch_bounds__(256) void k_fit_held(const Fit a) {
  const int64_t b = blockIdx.x;
  const kv_seq q = kv_sequence(a.s, b);
  const int64_t want = wanted(a, q), stride = a.s.table_stride;
  const int64_t full = ((int64_t)q.past + (1 << a.c.plog) - 1) >> a.c.plog;
  const int32_t *row = a.table + b * stride;
  __shared__ int held, alone;
  if (threadIdx.x == 0) held = alone = (int)want;
  __syncthreads();
  bool bad = q.bad || want > stride;
  if (!bad) {
    for (int64_t e = threadIdx.x; e < want; e += 256) {
      const int id = row[e];
      if (id < 0)
        atomicMin(&held, (int)e);
      else if (id >= a.c.pages)
        bad = true;
      else if (e >= full && a.refs[id] > 1)
        atomicMin(&alone, (int)e);
    }
  }
  bad = __syncthreads_or(bad);
  if (!bad) {
    // All pages of the past, and none behind a gap.
    bad = held < full;
    for (int64_t e = held + (int)threadIdx.x; e < want; e += 256) bad |= row[e] >= 0;
    bad = __syncthreads_or(bad);
  }
  if (threadIdx.x == 0) {
    a.held[b] = bad ? -1 : min(held, alone);
    if (bad) atomicOr(a.c.refused, 1);
  }
}
// Lets the others go.
__global__ __launch_bounds__(256) void k_fit_release(const Fit a) {
  const int64_t b = blockIdx.x, stride = a.s.table_stride;
  const int held = a.held[b];
  if (held < 0) return;
  int32_t *row = a.table + b * stride;
  for (int64_t e = held + (int)threadIdx.x; e < stride; e += 256) {
    const int id = row[e];
    if (id >= 0 && id < a.c.pages) atomicSub(a.refs + id, 1);
    row[e] = -1;
  }
}

// The page that sequence b writes into the middle of, -1: none.
__device__ inline int middle(const Fit &a, int64_t b) {
  const kv_seq q = kv_sequence(a.s, b);
  if (a.held[b] < 0 || q.n == 0 || (q.past & ((1 << a.c.plog) - 1)) == 0) return -1;
  return a.table[b * a.s.table_stride + (q.past >> a.c.plog)];
}
// A sequence's need of pages (the first workgroups), and the free ones of each run.
__global__ __launch_bounds__(256) void k_fit_need(const Fit a) {
  if (blockIdx.x >= a.s.batch) {
    const int64_t run = blockIdx.x - a.s.batch;
    int n = 0;
    for (int64_t i = run * kRun + threadIdx.x; i < std::min((run + 1) * kRun, a.c.pages); i += 256)
      n += a.refs[i] == 0;
    __shared__ int sum;
    if (threadIdx.x == 0) sum = 0;
    __syncthreads();
    if (n) atomicAdd(&sum, n);
    __syncthreads();
    if (threadIdx.x == 0) a.free[run] = sum;
    return;
  }
  const int64_t b = blockIdx.x;
  const int page = middle(a, b);
  int before = 0;
  if (page >= 0)
    for (int64_t o = threadIdx.x; o < b; o += 256) before += middle(a, o) == page;
  __shared__ int earlier;
  if (threadIdx.x == 0) earlier = 0;
  __syncthreads();
  if (before) atomicAdd(&earlier, before);
  __syncthreads();
  if (threadIdx.x) return;
  const int refs = page >= 0 ? a.refs[page] : 0;
  const bool copy = page >= 0 && earlier + 1 < refs;
  a.copy[b] = copy ? 1 : refs > 1 ? 2 : 0;
  a.need[b] = a.held[b] < 0 ? 0 : (int)(wanted(a, kv_sequence(a.s, b)) - a.held[b]) + copy;
  a.old[b] = copy ? page : -1;
  a.own[b] = -1;
}

// The running sum of n numbers in place (each: what is before it), by 1024 threads.
__device__ inline int64_t scan_all(const int32_t *in, int32_t *out, int64_t n, int64_t *part) {
  int64_t base = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i0 = 0; i0 < n; i0 += 1024) {
    const int64_t i = i0 + threadIdx.x;
    const int64_t own = i < n ? in[i] : 0;
    int64_t x = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int64_t before = base;
    for (int k = 0; k < wave; k++) before += part[k];
    for (int k = 0; k < 16; k++) base += part[k];
    if (i < n) out[i] = (int32_t)std::min<int64_t>(before + x - own, 0x7fffffff);
  }
  return base;
}
// Which sequences get their pages, in order.
__global__ __launch_bounds__(1024) void k_fit_share(const Fit a) {
  __shared__ int64_t part[16];
  const int64_t all = scan_all(a.free, a.free, a.nrun, part);
  scan_all(a.need, a.first, a.s.batch, part);
  for (int64_t b = threadIdx.x; b < a.s.batch; b += 1024) {
    const int need = a.need[b];
    const bool fits = (int64_t)a.first[b] + need <= all;
    const bool given = a.held[b] >= 0 && ((need == 0 && a.copy[b] == 0) || fits);
    a.granted[b] = given;
  }
}

// Hands a run's free pages out.
__global__ __launch_bounds__(256) void k_fit_give(const Fit a) {
  const int64_t run = blockIdx.x, batch = a.s.batch;
  __shared__ int part[4];
  int base = a.free[run];
  const int64_t last = batch - 1;
  const int64_t all = (int64_t)a.first[last] + a.need[last];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i0 = run * kRun; i0 < std::min((run + 1) * kRun, a.c.pages) && base < all; i0 += 256) {
    const int64_t i = i0 + threadIdx.x;
    const bool is = i < a.c.pages && a.refs[i] == 0;
    const uint64_t mask = __ballot(is);
    __syncthreads();
    if (lane == 0) part[wave] = __popcll(mask);
    __syncthreads();
    int g = base + __popcll(mask & ((1ull << lane) - 1));
    for (int k = 0; k < wave; k++) g += part[k];
    base += part[0] + part[1] + part[2] + part[3];
    if (!is || g >= all) continue;
    // The last sequence whose pages begin at g or before, among those that need any.
    int64_t lo = 0, hi = batch;
    while (hi - lo > 1) {
      const int64_t at = (lo + hi) / 2;
      if (a.first[at] <= g) lo = at;
      else hi = at;
    }
    if (!a.granted[lo] || g - a.first[lo] >= a.need[lo]) continue;
    const bool copy = a.copy[lo] == 1;
    int at = g - a.first[lo];
    int32_t *row = a.table + lo * a.s.table_stride;
    if (copy && at == 0) {
      row[kv_sequence(a.s, lo).past >> a.c.plog] = (int32_t)i;
      a.own[lo] = (int32_t)i;
      atomicSub(a.refs + a.old[lo], 1);
    } else {
      row[a.held[lo] + at - copy] = (int32_t)i;
    }
    a.refs[i] = 1;
  }
}

// All of it but the copies by one workgroup: what few sequences and pages need, without the waits
// between launches, every table entry in a register of its own (64 sequences of 64 pages: 13
// us, 21 in the kernels of their own and as many waits; 4 sequences: 9 and 17).  What it holds sets the
// border: with the copies 64 sequences of 126 entries take 20 us here, of 128 entries 45 in the other
// form, 512 of 128 67.  Many sequences of few pages are slower here, by the search for earlier ones
// of the same page: 1024 of 6 entries 95, 1040 80 in the other form.  A chain: the entries, their
// counts, what is let go, what is free, the entries written: 7 us of waits.
constexpr int kOneBatch = 1024, kOnePages = 65536, kOneNeed = 8192, kOneEach = kOneNeed / 1024;
// A count that other waves change in this launch.
__device__ inline int count_of(const int32_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ __launch_bounds__(1024) void k_fit_one(const Fit a) {
  // Of each sequence: its page of the first new row, if that falls into the middle, else -1; pages
  // wanted, full of the past (the last one too), held; the first gap and the first shared page.
  __shared__ int mid[kOneBatch], want[kOneBatch], full[kOneBatch], gap[kOneBatch], other[kOneBatch];
  __shared__ int need[kOneBatch], first[kOneBatch], free[kOneNeed];
  __shared__ uint8_t bad[kOneBatch], copies[kOneBatch];  // copies: as Fit's copy
  __shared__ int64_t part[16];
  __shared__ int count[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, me = threadIdx.x;
  const int batch = (int)a.s.batch, stride = (int)a.s.table_stride;
  // The table's entries, eight a thread.
  int id[kOneEach], refs[kOneEach];
#pragma unroll
  for (int i = 0; i < kOneEach; i++) {
    const int at = me + 1024 * i;
    id[i] = at < batch * stride ? a.table[at] : -1;
  }
  // A sequence a thread.
  kv_seq q = {};
  if (me < batch) {
    q = kv_sequence(a.s, me);
    const int64_t w = wanted(a, q);
    bad[me] = q.bad || w > stride;
    want[me] = bad[me] ? 0 : (int)w;
    full[me] = bad[me] ? 0 : (int)(((int64_t)q.past + (1 << a.c.plog) - 1) >> a.c.plog);
    gap[me] = other[me] = want[me];
    // (For now the entry, which a sequence that is not refused keeps.)
    mid[me] = q.n > 0 && (q.past & ((1 << a.c.plog) - 1)) != 0 ? q.past >> a.c.plog : -1;
  }
#pragma unroll
  for (int i = 0; i < kOneEach; i++) refs[i] = id[i] >= 0 && id[i] < a.c.pages ? a.refs[id[i]] : 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOneEach; i++) {
    const int at = me + 1024 * i;
    if (at >= batch * stride) break;
    const int b = at / stride, e = at - b * stride;
    if (e >= want[b]) continue;
    if (id[i] < 0) atomicMin(gap + b, e);
    if (id[i] >= a.c.pages) bad[b] = 1;
    if (e >= full[b] && refs[i] > 1) atomicMin(other + b, e);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOneEach; i++) {  // (nothing behind a gap)
    const int at = me + 1024 * i;
    if (at >= batch * stride) break;
    const int b = at / stride, e = at - b * stride;
    if (e < want[b] && e > gap[b] && id[i] >= 0) bad[b] = 1;
  }
  __syncthreads();
  if (me < batch) {
    if (gap[me] < full[me]) bad[me] = 1;
    if (bad[me]) atomicOr(a.c.refused, 1);
    gap[me] = bad[me] ? -1 : min(gap[me], other[me]);  // what it keeps
    need[me] = -1;
  }
  __syncthreads();
  const int *held = gap;
  // What is let go; the pages in whose middle rows begin.
#pragma unroll
  for (int i = 0; i < kOneEach; i++) {
    const int at = me + 1024 * i;
    if (at >= batch * stride) break;
    const int b = at / stride, e = at - b * stride;
    if (held[b] < 0) continue;
    if (e < held[b]) {
      if (e == mid[b]) need[b] = id[i];
      continue;
    }
    if (id[i] >= 0 && id[i] < a.c.pages) atomicSub(a.refs + id[i], 1);
    a.table[at] = -1;
  }
  // (The counts are kept by the L2 that this workgroup's atomics and count_of go to: waiting is enough.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  // The first pages' counts, on their way while the need is added up.
  int c[4];
  auto counts = [&](int64_t p0) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int64_t p = p0 + 4 * me + k;
      c[k] = p < a.c.pages ? count_of(a.refs + p) : 1;
    }
  };
  counts(0);
  if (me < batch) mid[me] = need[me];  // the page
  __syncthreads();
  // What is needed, in all and before each.
  for (int b = wave; b < batch; b += 16) {
    const int page = mid[b];
    int earlier = 0;
    for (int o0 = 0; page >= 0 && o0 < b; o0 += 64)
      earlier += __popcll(__ballot(o0 + lane < b && mid[min(o0 + lane, b)] == page));
    if (lane == 0) need[b] = earlier;
  }
  __syncthreads();
  if (me < batch) {
    const int r = mid[me] >= 0 ? count_of(a.refs + mid[me]) : 0;
    const bool copy = mid[me] >= 0 && need[me] + 1 < r;
    copies[me] = copy ? 1 : r > 1 ? 2 : 0;
    need[me] = held[me] < 0 ? 0 : want[me] - held[me] + copy;
  }
  __syncthreads();
  const int total = (int)scan_all(need, first, batch, part);
  // The free pages that are needed, lowest first: four a thread.
  int found = 0;
  for (int64_t p0 = 0; p0 < a.c.pages && found < total; p0 += 4096) {
    int is = 0, n = 0;
    if (p0) counts(p0);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (c[k] == 0) is |= 1 << k, n++;
    int x = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) count[wave] = x;
    __syncthreads();
    int at = found + x - n;
    for (int k = 0; k < 16; k++) {
      if (k < wave) at += count[k];
      found += count[k];
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (is >> k & 1) {
        if (at < total) free[at] = (int)(p0 + 4 * me + k);
        at++;
      }
  }
  __syncthreads();
  if (me < batch) {
    const bool copy = copies[me] == 1;
    const bool given = held[me] >= 0 && ((need[me] == 0 && copies[me] == 0) || first[me] + need[me] <= found);
    a.granted[me] = given;
    a.own[me] = given && copy ? free[first[me]] : -1;
    a.old[me] = mid[me];
    bad[me] = !given;
    if (given && copy) atomicSub(a.refs + mid[me], 1);
  }
  __syncthreads();
  for (int g = me; g < min(total, found); g += 1024) {
    // The last sequence whose pages begin at g or before.
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
      const int at = (lo + hi) / 2;
      if (first[at] <= g) lo = at;
      else hi = at;
    }
    const int at = g - first[lo];
    if (bad[lo] || at >= need[lo]) continue;
    const bool copy = copies[lo] == 1;
    const int e = copy && at == 0 ? full[lo] - 1 : held[lo] + at - copy;
    a.table[(int64_t)lo * stride + e] = free[g];
    a.refs[free[g]] = 1;
  }
}

__global__ __launch_bounds__(256) void k_fit_copy(const Fit a) {
  const int64_t b = blockIdx.y;
  const int own = a.own[b];
  if (own >= 0) copy_piece(a.c, a.old[b], own, blockIdx.x);
}

}  // namespace

size_t mg_kv_copy_ws(const mg_kv_cache &c, int64_t n) {
  return n > 1024 ? mg_align((size_t)c.pages * 4) : 0;
}

mg_status mg_kv_copy_run(mg_ctx *ctx, const mg_kv_cache &c, const int32_t *src, const int32_t *dst,
                         int64_t n, void *ws) {
  Pairs a{c, src, dst, n, page_pieces(c), nullptr};
  // Each workgroup reads the whole list for its pair; long ones leave their marks at the pages first.
  if (n > 1024) {
    a.marks = static_cast<uint32_t *>(ws);
    k_clear_marks<<<dim3((unsigned)((c.pages + 255) / 256)), dim3(256), 0, ctx->stream>>>(a);
    k_mark<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, ctx->stream>>>(a);
  }
  k_copy_pages<<<dim3((unsigned)(n * a.pieces)), dim3(256), 0, ctx->stream>>>(a);
  return mg_launch_check("KV cache copy");
}
int64_t mg_kv_copy_groups(const mg_kv_cache &c, int64_t n) { return n * page_pieces(c); }

// Chunks of a sequence in the staged form.
constexpr int kLong = 128;
static int64_t compact_chunks(const mg_seq_batch &s) { return (s.max_new + 3 + kLong - 1) / kLong + 1; }
size_t mg_kv_compact_ws(const mg_kv_cache &c, const mg_seq_batch &s) {
  // Lists of up to 256 rows move in order, and what is beyond a launch.
  const int64_t chunks = compact_chunks(s);
  if (s.max_new <= 2 * kLong || chunks > 32767 || s.batch * c.kv_heads * 2 > MG_MOST_GROUPS / chunks) return 0;
  const size_t parts = (size_t)s.batch * c.kv_heads * 2 * chunks;
  return mg_align((size_t)s.batch * sizeof(Moves)) + parts * kLong * (c.dp * kv_bits(c.fmt) / 8 + 8);
}

template <bool INT4>
static void compact(mg_ctx *ctx, Compact a, void *ws) {
  const unsigned heads = (unsigned)a.c.kv_heads, batch = (unsigned)a.s.batch;
  hipStream_t st = ctx->stream;
  int32_t *past_out = a.past_out;
  const bool alias = past_out == a.s.past;  // (written once nothing reads the past any more)
  if (alias) a.past_out = nullptr;
  if (a.s.max_new == 0) {
    // No rows: the lengths alone.
  } else if (!ws) {
    const dim3 grid(heads, batch, 2);
    if (a.s.max_new <= 32)
      k_compact<INT4, 32, IN_ORDER><<<grid, dim3(256), 0, st>>>(a);
    else
      k_compact<INT4, kLong, IN_ORDER><<<grid, dim3(256), 0, st>>>(a);
  } else {
    a.chunks = (int)compact_chunks(a.s);
    char *p = static_cast<char *>(ws);
    a.moves = reinterpret_cast<Moves *>(p);
    p += mg_align((size_t)a.s.batch * sizeof(Moves));
    a.scales = reinterpret_cast<float *>(p);
    p += (size_t)a.s.batch * heads * 2 * a.chunks * kLong * 8;
    a.rows = reinterpret_cast<uint8_t *>(p);
    const dim3 grid(heads, batch, 2 * (unsigned)a.chunks);
    k_moves<<<dim3(batch), dim3(256), 0, st>>>(a);
    k_compact<INT4, kLong, GATHER><<<grid, dim3(256), 0, st>>>(a);
    k_compact<INT4, kLong, SCATTER><<<grid, dim3(256), 0, st>>>(a);
  }
  if (past_out && (alias || a.s.max_new == 0)) {
    a.past_out = past_out;
    k_moves<<<dim3(batch), dim3(256), 0, st>>>(a);
  }
}

mg_status mg_kv_compact_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s,
                            const int32_t *kept, const int32_t *count, int32_t *past_out, void *ws) {
  const Compact a{c, s, kept, count, past_out, nullptr, nullptr, nullptr, 1};
  if (c.fmt == MG_KV_INT4)
    compact<true>(ctx, a, ws);
  else
    compact<false>(ctx, a, ws);
  return mg_launch_check("KV cache compact");
}

mg_status mg_kv_fork_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s,
                         const int32_t *parent, int64_t out_batch, int32_t *past_out,
                         int32_t *table_out, int64_t out_stride, int32_t *refs) {
  const Fork a{c, s, parent, out_batch, out_stride, past_out, table_out, refs};
  k_fork<<<dim3((unsigned)(out_batch + s.batch)), dim3(256), 0, ctx->stream>>>(a);
  return mg_launch_check("KV cache fork");
}

size_t mg_kv_fit_ws(const mg_kv_cache &c, int64_t batch) {
  return 6 * mg_align((size_t)batch * 4) + mg_align((size_t)((c.pages + kRun - 1) / kRun) * 4);
}

mg_status mg_kv_fit_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s, int32_t *refs,
                        int32_t *granted, void *ws) {
  Fit a{c, s, const_cast<int32_t *>(s.page_table), refs, granted};
  a.nrun = (c.pages + kRun - 1) / kRun;
  char *p = static_cast<char *>(ws);
  const size_t one = mg_align((size_t)s.batch * 4);
  int32_t **parts[] = {&a.held, &a.copy, &a.first, &a.need, &a.old, &a.own, &a.free};
  for (int32_t **x : parts) {
    *x = reinterpret_cast<int32_t *>(p);
    p += one;
  }
  const unsigned batch = (unsigned)s.batch;
  hipStream_t st = ctx->stream;
  if (s.batch <= kOneBatch && c.pages <= kOnePages && s.batch * (s.table_stride + 1) <= kOneNeed) {
    k_fit_one<<<dim3(1), dim3(1024), 0, st>>>(a);
    k_fit_copy<<<dim3((unsigned)page_pieces(c), batch), dim3(256), 0, st>>>(a);
    return mg_launch_check("KV cache fit");
  }
  k_fit_held<<<dim3(batch), dim3(256), 0, st>>>(a);
  k_fit_release<<<dim3(batch), dim3(256), 0, st>>>(a);
  k_fit_need<<<dim3(batch + (unsigned)a.nrun), dim3(256), 0, st>>>(a);
  k_fit_share<<<dim3(1), dim3(1024), 0, st>>>(a);
  k_fit_give<<<dim3((unsigned)a.nrun), dim3(256), 0, st>>>(a);
  k_fit_copy<<<dim3((unsigned)page_pieces(c), batch), dim3(256), 0, st>>>(a);
  return mg_launch_check("KV cache fit");
}
