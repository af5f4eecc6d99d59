// Rotary positions, shared by the rotation, the cache's append and its attention.
#pragma once

#include "mg_internal.h"

constexpr int MG_ROPE_MAX_HALF = 128;

struct mg_rotate_problem {
  const float *x;
  float *y;
  int64_t batch, seq, heads, d;
  int64_t xs[3], ys[3];
  mg_rope rope;
};

// Element d of vector x turned at position pos: in 64 bits, rounded once (the products of
// two fp32 values are exact there).  NaN where the tables have no such position.
__device__ inline float rope_at(const float *x, int64_t d, int64_t pos, const mg_rope &r) {
  const int64_t half = r.half_rot;
  if (d >= 2 * half) return x[d];
  if ((uint64_t)pos >= (uint64_t)r.max_pos) return __builtin_nanf("");
  const int64_t i = r.interleaved ? d >> 1 : d < half ? d : d - half;
  const bool second = r.interleaved ? d & 1 : d >= half;
  const int64_t o = r.interleaved ? d ^ 1 : second ? d - half : d + half;
  const double c = r.cos_table[pos * half + i], s = r.sin_table[pos * half + i];
  const double a = x[d], z = x[o];
  return (float)(second ? a * c + z * s : a * c - z * s);
}

mg_status mg_rope_tables_run(mg_ctx *ctx, int64_t first, int64_t count, int64_t half,
                             const double *freq, double a, float *c, float *s);
mg_status mg_rotate_run(mg_ctx *ctx, const mg_rotate_problem &p);
