// Rotary positions: the tables, scaled for long contexts, and the rotation of packed or
// strided vectors.
//
// Tables: entry (p, i) is value_factor * cos / sin of p f_i.  The angle in turns, p f_i /
// 2 pi, is formed in 64 bits and its whole part dropped there, so an entry at position
// 10^6 is as exact as one at 0; what is left, at most half a turn, goes through the fp32
// sincospi.  One pass of writes bounds it.
//
// Rotation: y = (x c - z s, z c + x s) per pair in 64 bits, rounded once, as the
// rotation inside GroupQueryAttention.  One pass of reads and writes bounds it.
#include <hip/hip_runtime.h>

#include <cmath>

#include "mg_internal.h"
#include "rope_common.h"

namespace {

struct Freq {
  double turns[MG_ROPE_MAX_HALF];  // f_i / 2 pi
};

__global__ __launch_bounds__(256) void k_rope_tables(const Freq f, int64_t first, int64_t n,
                                                     int half, float a, float *__restrict__ c,
                                                     float *__restrict__ s) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  const int64_t p = e / half;
  const double t = (double)(first + p) * f.turns[e - p * half];
  const float r = (float)(2.0 * (t - rint(t)));  // in half turns, [-1, 1]
  float sv, cv;
  sincospif(r, &sv, &cv);
  c[e] = a * cv;
  s[e] = a * sv;
}

// One thread a pair, or one element that passes through (so y may be x).
__global__ __launch_bounds__(256) void k_rotate(mg_rotate_problem p) {
  const int64_t half = p.rope.half_rot, units = p.d - half;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= p.batch * p.seq * p.heads * units) return;
  const int64_t u = e % units, h = e / units % p.heads, r = e / (units * p.heads);
  const int64_t b = r / p.seq, s = r % p.seq;
  const int64_t pos = p.rope.positions ? p.rope.positions[r] : s;
  const float *x = p.x + b * p.xs[0] + s * p.xs[1] + h * p.xs[2];
  float *y = p.y + b * p.ys[0] + s * p.ys[1] + h * p.ys[2];
  if (u >= half) {
    y[half + u] = x[half + u];
    return;
  }
  const int64_t d = p.rope.interleaved ? 2 * u : u, o = p.rope.interleaved ? d + 1 : d + half;
  const float yd = rope_at(x, d, pos, p.rope), yo = rope_at(x, o, pos, p.rope);
  y[d] = yd;
  y[o] = yo;
}

}  // namespace

mg_status mg_rope_tables_run(mg_ctx *ctx, int64_t first, int64_t count, int64_t half,
                             const double *freq, double a, float *c, float *s) {
  Freq f;
  for (int i = 0; i < MG_ROPE_MAX_HALF; i++)
    f.turns[i] = i < half ? freq[i] * 0.15915494309189533577 : 0.0;
  const int64_t n = count * half;
  k_rope_tables<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, ctx->stream>>>(
      f, first, n, (int)half, (float)a, c, s);
  return mg_launch_check("rotary tables");
}

mg_status mg_rotate_run(mg_ctx *ctx, const mg_rotate_problem &p) {
  const int64_t n = p.batch * p.seq * p.heads * (p.d - p.rope.half_rot);
  k_rotate<<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, ctx->stream>>>(p);
  return mg_launch_check("rotary embedding");
}
