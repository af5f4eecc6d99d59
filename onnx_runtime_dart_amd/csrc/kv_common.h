// The quantised KV cache: its memory, and where a batch's rows lie in it.  Shared by the
// kernels that write, read and attend (kvcache.hip, kvattn.hip) and by the host-side
// location check (api.hip).
#pragma once

#include "mg_internal.h"

// A cache of `pages` pages of 2^plog tokens.  Every (page, head) holds
//   K codes  [token][dim]: INT8 q + 128, E4M3 its bits, INT4 two dims a byte (even dim low);
//   V codes  [token / 4][dim][token % 4], so that the four tokens of one dim are one dword
//            (the matrix instruction's order for the values); INT4: the dword of a dim pair
//            (a, a + 1) holds nibbles {t0 a, t2 a, t0 b, t2 b, t1 a, t3 a, t1 b, t3 b};
//   scales   fp32 [S][token]: K scale, V scale, and for INT4 K middle, V middle.
// dims are padded to a multiple of 64 with codes of any value (never NaN): the query is zero there,
// and what the values give there is not stored.
struct mg_kv_cache {
  int device = 0;
  int fmt = 0;
  int plog = 0;
  int kv_heads = 0, d = 0, dp = 0;
  int64_t pages = 0;
  uint8_t *k = nullptr, *v = nullptr;
  float *sc = nullptr;
  int32_t *refused = nullptr;
  int64_t bytes = 0;
};

__host__ __device__ inline int kv_bits(int fmt) { return fmt == MG_KV_INT4 ? 4 : 8; }
__host__ __device__ inline int kv_scales(int fmt) { return fmt == MG_KV_INT4 ? 4 : 2; }

// What all lanes read alike and no kernel that reads it so writes: a scalar load, which other
// loads in flight need not be waited for with.
template <class T>
__device__ inline T kv_scalar(const T *p) {
  return *(const __attribute__((address_space(4))) T *)p;
}

// Sequence b's rows [start, start + n) at positions past ..; n = 0 with bad set when a
// number breaks the batch's bounds.
struct kv_seq {
  int start, n, past;
  bool bad;
};
__host__ __device__ inline kv_seq kv_sequence(const mg_seq_batch &s, int64_t b) {
  const int64_t r0 = s.row_start[b], r1 = s.row_start[b + 1], p = s.past[b];
  kv_seq q;
  q.bad = r0 < 0 || r1 < r0 || r1 > s.rows || r1 - r0 > s.max_new || p < 0 ||
          p + (r1 - r0) > s.max_len;
  q.start = q.bad ? 0 : (int)r0;
  q.n = q.bad ? 0 : (int)(r1 - r0);
  q.past = q.bad ? 0 : (int)p;
  return q;
}
// The page of a position of sequence b, -1 when the table or the cache has none.
__host__ __device__ inline int64_t kv_page(const mg_seq_batch &s, int64_t b, int64_t pos, int plog,
                                           int64_t pages) {
  const int64_t at = pos >> plog;
  if (at >= s.table_stride) return -1;
  const int64_t id = s.page_table[b * s.table_stride + at];
  return id < 0 || id >= pages ? -1 : id;
}

// Launches (kvcache.hip, kvattn.hip); batch bounds and pointers checked by the caller.
mg_status mg_kv_clear(mg_ctx *ctx, mg_kv_cache *c);
mg_status mg_kv_append_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s,
                           const float *k, int64_t ks, const float *v, int64_t vs,
                           const mg_rope *rope);
mg_status mg_kv_read_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s, float *k,
                         int64_t ks, float *v, int64_t vs);
struct mg_kv_attn {
  mg_kv_cache c;
  mg_seq_batch s;
  const float *q;
  float *y;
  int64_t q_stride, y_stride;
  int group;  // query heads of a KV head
  mg_rope rope;  // half_rot 0: none
  const uint64_t *tree;
  int tree_words;
  float scale2;  // scale * log2(e)
  bool vec;  // q, y and the tables take 16-byte accesses
  // The plan: rows (query, head of the group) a workgroup takes, whether its waves split the
  // keys of 16 rows (else rows), row blocks a sequence, key splits.
  bool keys;
  int rows_wg, nblk, nsplit;
  float share;  // 1 / nsplit
  // Partial results of (row, split): outputs, then (maximum, sum).
  int64_t parts;
  float *part;
  float2 *part_ml;
};
// Fills the plan (split: keys may be split) and returns the workspace of its partials.
size_t mg_kv_attn_plan(const mg_ctx *ctx, mg_kv_attn *a, bool split);
mg_status mg_kv_attn_run(mg_ctx *ctx, mg_kv_attn a, void *ws);
