// Pages of the quantised KV cache: copied, their rows moved together, shared between sequences
// and handed out.
//
// A page's codes of keys, of values and its scales are three runs of memory, so a copy is one read
// and one write of them.  Rows that move within a sequence only ever move down, in order: a
// workgroup per head takes them 128 at a time, reads all before it writes any, and nothing that
// it writes is read later (row j comes from kept[j] >= j, later rows from beyond it).
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
  uint8_t *ok;  // [n], or null: each workgroup sees for itself
};
// Whether pair i is to be copied, by the whole workgroup; *bad: it is refused.
__device__ inline bool pair_ok(const Pairs &a, int64_t i, bool *bad) {
  const int s = a.src[i], d = a.dst[i];
  *bad = false;
  if ((s < 0 && d < 0) || s == d) return false;
  bool clash = s < 0 || d < 0 || s >= a.c.pages || d >= a.c.pages;
  for (int64_t j = threadIdx.x; j < a.n; j += 256) {
    const int sj = a.src[j], dj = a.dst[j];
    if (j != i && !(sj < 0 && dj < 0)) clash |= dj == d || (sj != dj && (sj == d || dj == s));
  }
  *bad = __syncthreads_or(clash);
  return !*bad;
}

__global__ __launch_bounds__(256) void k_check_pairs(const Pairs a) {
  bool bad;
  const bool ok = pair_ok(a, blockIdx.x, &bad);
  if (threadIdx.x == 0) {
    a.ok[blockIdx.x] = ok;
    if (bad) atomicOr(a.c.refused, 1);
  }
}
__global__ __launch_bounds__(256) void k_copy_pages(const Pairs a) {
  const int64_t i = blockIdx.x / a.pieces;
  const int piece = blockIdx.x % a.pieces;
  if (a.ok) {
    if (!a.ok[i]) return;
  } else {
    bool bad;
    const bool ok = pair_ok(a, i, &bad);
    if (bad && piece == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
    if (!ok) return;
  }
  copy_piece(a.c, a.src[i], a.dst[i], piece);
}

// ------------------------------------------------------------------- compact

struct Compact {
  mg_kv_cache c;
  mg_seq_batch s;
  const int32_t *kept, *count;
  int32_t *past_out;
};

constexpr int kRows = 128;  // rows moved at a time

// A sequence's rows to move: j0 .. count - 1 (rows before j0 stay where they are).
struct Moves {
  kv_seq q;
  int j0, count;
};
// By the whole workgroup; false: nothing to move.  *bad: the sequence is refused.
__device__ inline bool moves_of(const Compact &a, int64_t b, Moves *o, bool *bad) {
  o->q = kv_sequence(a.s, b);
  o->count = a.count[b];
  *bad = o->q.bad || o->count < 0 || o->count > o->q.n;
  if (*bad) return false;
  const int32_t *kept = a.kept + o->q.start;
  int same = 0;
  bool wrong = false;
  for (int j = threadIdx.x; j < o->count; j += 256) {
    const int k = kept[j];
    wrong |= k < 0 || k >= o->q.n || (j > 0 && k <= kept[j - 1]);
    same += k == j;
  }
  *bad = __syncthreads_or(wrong);
  if (*bad) return false;
  // (Rising numbers from 0 on: once one is beyond its place, all are.)
  __shared__ int sum;
  if (threadIdx.x == 0) sum = 0;
  __syncthreads();
  if (same) atomicAdd(&sum, same);
  __syncthreads();
  o->j0 = sum;
  return o->j0 < o->count;
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

// blockIdx: head, sequence, keys or values.
template <bool INT4>
__global__ __launch_bounds__(256) void k_compact(const Compact a) {
  __shared__ int64_t from[kRows + 4], to[kRows + 4];  // places in the cache, -1: none
  const int64_t b = blockIdx.y;
  const int h = blockIdx.x;
  Moves m;
  bool bad;
  const bool any = moves_of(a, b, &m, &bad);
  const bool first = threadIdx.x == 0 && h == 0 && blockIdx.z == 0;
  if (bad && first) atomicOr(a.c.refused, 1);
  if (!any) return;
  const int page = 1 << a.c.plog, mask = page - 1, heads = a.c.kv_heads;
  const int rb = a.c.dp * (INT4 ? 4 : 8) / 8;  // bytes of a vector's codes
  auto place = [&](int64_t pos) {
    const int64_t id = kv_page(a.s, b, pos, a.c.plog, a.c.pages);
    return id < 0 ? (int64_t)-1 : ((id * heads + h) << a.c.plog) + (pos & mask);
  };
  // Groups of four places, from the first that changes on.
  const int64_t g0 = (m.q.past + m.j0) >> 2, g1 = ((int64_t)m.q.past + m.count + 3) >> 2;
  for (int64_t g = g0; g < g1; g += kRows / 4) {
    __syncthreads();
    bool missing = false;
    if (threadIdx.x < kRows) {
      const int64_t pos = 4 * g + threadIdx.x, j = pos - m.q.past;
      int64_t t = -1, f = -1;
      if (j >= m.j0 && j < m.count) {
        t = place(pos);
        f = place((int64_t)m.q.past + a.kept[m.q.start + j]);
        missing = t < 0 || f < 0;
      }
      to[threadIdx.x] = missing ? -1 : t;
      from[threadIdx.x] = missing ? -1 : f;
    }
    if (missing) atomicOr(a.c.refused, 1);
    __syncthreads();
    // Scales, read now and written behind the barrier.
    const int sc = (int)blockIdx.z + 2 * ((int)threadIdx.x / kRows), row = threadIdx.x % kRows;
    const bool scaled = (INT4 || threadIdx.x < kRows) && to[row] >= 0;
    // The scale of a place: (page, head) block, kind, token.
    auto scale = [&](int64_t at) {
      return a.c.sc + ((at >> a.c.plog) * kv_scales(a.c.fmt) + sc) * page + (at & mask);
    };
    float s = 0.f;
    if (scaled) s = *scale(from[row]);
    if (blockIdx.z == 0) {
      const int vec = rb / 16;  // 2 .. 16
      u32x4 x[8];
      // (At most 2048 vectors of 16 bytes; rows that do not move read the cache's first.)
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int i = 256 * u + threadIdx.x, r = i / vec;
        const int64_t at = r < kRows && to[r] >= 0 ? from[r] * rb + 16 * (i - r * vec) : 0;
        x[u] = *reinterpret_cast<const u32x4 *>(a.c.k + at);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int i = 256 * u + threadIdx.x, r = i / vec;
        if (r < kRows && to[r] >= 0)
          *reinterpret_cast<u32x4 *>(a.c.k + to[r] * rb + 16 * (i - r * vec)) = x[u];
      }
    } else {
      // Dwords of four tokens: those of rows that move from where they are, the others kept.
      const int vec = rb / 4;  // vectors of four dwords of a group: 8 .. 64
      u32x4 x[8];
      // The group (four places lie together) that gets rows in this call, -1: none.
      auto group = [&](int q) {
        int64_t g4 = -1;
#pragma unroll
        for (int t = 0; t < 4; t++) g4 = std::max(g4, to[4 * q + t] >> 2);
        return g4;
      };
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int i = 256 * u + threadIdx.x, q = std::min(i / vec, kRows / 4 - 1), o = i % vec;
        const int64_t own = std::max<int64_t>(group(q), 0);
        x[u] = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const int64_t at = to[4 * q + t] >= 0 ? from[4 * q + t] : 4 * own + t;
          const u32x4 w = *reinterpret_cast<const u32x4 *>(a.c.v + (at >> 2) * 4 * rb + 16 * o);
          const int k = (int)(at & 3);
#pragma unroll
          for (int e = 0; e < 4; e++) x[u][e] |= token_to<INT4>(token_of<INT4>(w[e], k), t);
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int i = 256 * u + threadIdx.x, q = i / vec, o = i % vec;
        const int64_t own = q < kRows / 4 ? group(q) : -1;
        if (own >= 0) *reinterpret_cast<u32x4 *>(a.c.v + own * 4 * rb + 16 * o) = x[u];
      }
    }
    if (scaled) *scale(to[row]) = s;
  }
}

// (Its own launch: past_out may be the past that the moves read.)
__global__ __launch_bounds__(256) void k_past(const Compact a) {
  Moves m;
  bool bad;
  moves_of(a, blockIdx.x, &m, &bad);
  if (threadIdx.x == 0)
    a.past_out[blockIdx.x] = a.s.past[blockIdx.x] + (bad ? 0 : m.count);
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
  // Workspace: a sequence's held pages (-1: refused), whether it takes a copy (1) or waits for
  // those that share its page (2), its first page among those handed out, its copy's pages; the
  // runs' free pages, then those before them.
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

__global__ __launch_bounds__(256) void k_fit_copy(const Fit a) {
  const int64_t b = blockIdx.y;
  const int own = a.own[b];
  if (own >= 0) copy_piece(a.c, a.old[b], own, blockIdx.x);
}

}  // namespace

size_t mg_kv_copy_ws(int64_t n) { return n > 1024 ? mg_align((size_t)n) : 0; }

mg_status mg_kv_copy_run(mg_ctx *ctx, const mg_kv_cache &c, const int32_t *src, const int32_t *dst,
                         int64_t n, void *ws) {
  Pairs a{c, src, dst, n, page_pieces(c), nullptr};
  // Each workgroup reads the whole list for its pair: for long ones once, not for every piece.
  if (n > 1024) {
    a.ok = static_cast<uint8_t *>(ws);
    k_check_pairs<<<dim3((unsigned)n), dim3(256), 0, ctx->stream>>>(a);
  }
  k_copy_pages<<<dim3((unsigned)(n * a.pieces)), dim3(256), 0, ctx->stream>>>(a);
  return mg_launch_check("KV cache copy");
}
int64_t mg_kv_copy_groups(const mg_kv_cache &c, int64_t n) { return n * page_pieces(c); }

mg_status mg_kv_compact_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s,
                            const int32_t *kept, const int32_t *count, int32_t *past_out) {
  const Compact a{c, s, kept, count, past_out};
  const dim3 grid((unsigned)c.kv_heads, (unsigned)s.batch, 2);
  if (s.max_new > 0) {
    if (c.fmt == MG_KV_INT4)
      k_compact<true><<<grid, dim3(256), 0, ctx->stream>>>(a);
    else
      k_compact<false><<<grid, dim3(256), 0, ctx->stream>>>(a);
  }
  if (past_out) k_past<<<dim3((unsigned)s.batch), dim3(256), 0, ctx->stream>>>(a);
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
  k_fit_held<<<dim3(batch), dim3(256), 0, st>>>(a);
  k_fit_release<<<dim3(batch), dim3(256), 0, st>>>(a);
  k_fit_need<<<dim3(batch + (unsigned)a.nrun), dim3(256), 0, st>>>(a);
  k_fit_share<<<dim3(1), dim3(1024), 0, st>>>(a);
  k_fit_give<<<dim3((unsigned)a.nrun), dim3(256), 0, st>>>(a);
  k_fit_copy<<<dim3((unsigned)page_pieces(c), batch), dim3(256), 0, st>>>(a);
  return mg_launch_check("KV cache fit");
}
