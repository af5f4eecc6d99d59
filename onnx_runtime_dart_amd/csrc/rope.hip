// Rotary positions: the tables, scaled for long contexts, and the rotation of packed or
// strided vectors.
//
// Tables: entry (p, i) is value_factor * cos / sin of p f_i.  The angle in turns, p f_i /
// 2 pi, is formed in 64 bits and its whole part dropped there, so an entry at position
// 10^6 is as exact as one at 0; what is left, at most half a turn, is rounded to fp32 and goes
// through the fp32 sincospi, then times value_factor in fp32: three roundings, where cosines in
// 64 bits would round once, for twice the error (4e-8 of the entries' size on average).  One pass
// of writes bounds it: a thread makes four adjacent entries (one 16-byte store a table) where
// half_rot is a multiple of four.
//
// Rotation: y = (x c - z s, z c + x s) per pair in 64 bits, rounded once, as the
// rotation inside GroupQueryAttention.  One pass of reads and writes bounds it: a thread
// turns four adjacent pairs of up to four heads of one row, so that it reads its table
// entries once for them (8191 rows of 32 heads of 128: 55 us, 4.9 TB/s).
#include <hip/hip_runtime.h>

#include <cmath>

#include "mg_internal.h"
#include "rope_common.h"

namespace {

struct Freq {
  double turns[MG_ROPE_MAX_HALF];  // f_i / 2 pi
};

// W adjacent entries a thread; IX: an index type that holds every entry.
template <int W, class IX>
__global__ __launch_bounds__(256) void k_rope_tables(const Freq f, int64_t first, IX n, IX half,
                                                     float a, float *__restrict__ c,
                                                     float *__restrict__ s) {
  const IX e = ((IX)blockIdx.x * 256 + threadIdx.x) * W;
  if (e >= n) return;
  const IX p = e / half;
  const int i = (int)(e - p * half);
  const double pos = (double)(first + (int64_t)p);
  float cv[W], sv[W];
#pragma unroll
  for (int j = 0; j < W; j++) {
    const double t = pos * f.turns[i + j];
    sincospif((float)(2.0 * (t - rint(t))), &sv[j], &cv[j]);  // in half turns, [-1, 1]
  }
  if constexpr (W == 4) {
    *reinterpret_cast<float4 *>(c + e) = make_float4(a * cv[0], a * cv[1], a * cv[2], a * cv[3]);
    *reinterpret_cast<float4 *>(s + e) = make_float4(a * sv[0], a * sv[1], a * sv[2], a * sv[3]);
  } else {
    c[e] = a * cv[0];
    s[e] = a * sv[0];
  }
}

// Adjacent elements moved at a time: 16 bytes or one element.
template <int W>
struct Part {
  float v[W];
};
template <int W>
__device__ inline Part<W> get(const float *p) {
  Part<W> r;
  if constexpr (W == 4) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    r.v[0] = x.x, r.v[1] = x.y, r.v[2] = x.z, r.v[3] = x.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <int W>
__device__ inline void put(float *p, const Part<W> &x) {
  if constexpr (W == 4)
    *reinterpret_cast<float4 *>(p) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
  else
    *p = x.v[0];
}

constexpr int kHeads = 4;  // heads a thread turns

// A thread: W pairs, or W elements that pass through, of kHeads heads of a row.  Units of a
// vector: half / W of pairs, then the rest.  Reads of a pair precede its writes (y may be x).
template <int W, class IX>
__global__ __launch_bounds__(256) void k_rotate(const mg_rotate_problem p, IX total, IX units,
                                                IX groups) {
  const IX e = (IX)blockIdx.x * 256 + threadIdx.x;
  if (e >= total) return;
  const IX rg = e / units, u = (e - rg * units) * W;
  const IX r = rg / groups;
  const int h0 = (int)(rg - r * groups) * kHeads;
  const int half = (int)p.rope.half_rot;
  const IX b = r / (IX)p.seq;
  const int64_t s = r - b * (IX)p.seq;
  const int64_t xo = (int64_t)b * p.xs[0] + s * p.xs[1], yo = (int64_t)b * p.ys[0] + s * p.ys[1];
  const int n = (int)min((int64_t)kHeads, p.heads - h0);
  if (u >= (IX)half) {
    const int64_t d = (int64_t)u + half;
    for (int h = h0; h < h0 + n; h++)
      put<W>(p.y + yo + h * p.ys[2] + d, get<W>(p.x + xo + h * p.xs[2] + d));
    return;
  }
  const int64_t pos = p.rope.positions ? p.rope.positions[r] : s;
  const bool in = (uint64_t)pos < (uint64_t)p.rope.max_pos;
  const int64_t t = (in ? pos : 0) * half + (int64_t)u;
  const Part<W> ct = get<W>(p.rope.cos_table + t), st = get<W>(p.rope.sin_table + t);
  double c[W], sn[W];
#pragma unroll
  for (int j = 0; j < W; j++) {
    c[j] = in ? (double)ct.v[j] : __builtin_nan("");
    sn[j] = st.v[j];
  }
  const bool il = p.rope.interleaved;
  const int64_t d0 = il ? 2 * (int64_t)u : (int64_t)u, d1 = il ? d0 + W : d0 + half;
#pragma unroll
  for (int k = 0; k < kHeads; k++) {
    if (k >= n) break;
    const float *x = p.x + xo + (h0 + k) * p.xs[2];
    float *y = p.y + yo + (h0 + k) * p.ys[2];
    const Part<W> x0 = get<W>(x + d0), x1 = get<W>(x + d1);
    Part<W> y0, y1;
#pragma unroll
    for (int j = 0; j < W; j++) {
      // (A pair interleaved in the two quads: elements 2 j and 2 j + 1 of the eight.)
      const int a = 2 * j, z = 2 * j + 1;
      const float xa = !il ? x0.v[j] : a < W ? x0.v[a % W] : x1.v[a % W];
      const float xz = !il ? x1.v[j] : z < W ? x0.v[z % W] : x1.v[z % W];
      const float ya = (float)((double)xa * c[j] - (double)xz * sn[j]);
      const float yz = (float)((double)xz * c[j] + (double)xa * sn[j]);
      if (!il) {
        y0.v[j] = ya;
        y1.v[j] = yz;
      } else {
        (a < W ? y0 : y1).v[a % W] = ya;
        (z < W ? y0 : y1).v[z % W] = yz;
      }
    }
    put<W>(y + d0, y0);
    put<W>(y + d1, y1);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int W>
mg_status rotate(mg_ctx *ctx, const mg_rotate_problem &p) {
  const int64_t units = (p.d - p.rope.half_rot) / W, groups = (p.heads + kHeads - 1) / kHeads;
  const int64_t n = p.batch * p.seq * groups * units;
  if (n > 256 * MG_MOST_GROUPS) return mg_fail(MG_UNSUPPORTED, "RotaryEmbedding: too many elements");
  const dim3 grid((unsigned)((n + 255) / 256));
  // 32-bit indices where they suffice: their divisions cost a fraction of the 64-bit ones
  // (8191 rows of 32 heads: 166 us with 64-bit indices and an element a thread).
  if (n < 0x7fffff00)
    k_rotate<W, uint32_t><<<grid, dim3(256), 0, ctx->stream>>>(p, (uint32_t)n, (uint32_t)units,
                                                               (uint32_t)groups);
  else
    k_rotate<W, uint64_t><<<grid, dim3(256), 0, ctx->stream>>>(p, (uint64_t)n, (uint64_t)units,
                                                               (uint64_t)groups);
  return mg_launch_check("rotary embedding");
}

}  // namespace

mg_status mg_rope_tables_run(mg_ctx *ctx, int64_t first, int64_t count, int64_t half,
                             const double *freq, double a, float *c, float *s) {
  Freq f;
  for (int i = 0; i < MG_ROPE_MAX_HALF; i++)
    f.turns[i] = i < half ? freq[i] * 0.15915494309189533577 : 0.0;
  const int64_t n = count * half;
  const bool quad = half % 4 == 0 && aligned16(c) && aligned16(s);
  const int64_t groups = (n + (quad ? 1023 : 255)) / (quad ? 1024 : 256);
  if (groups > MG_MOST_GROUPS) return mg_fail(MG_UNSUPPORTED, "RotaryTables: too many entries");
  const dim3 grid((unsigned)groups);
  hipStream_t st = ctx->stream;
  if (quad && n < 0x7ffffc00)
    k_rope_tables<4, uint32_t><<<grid, dim3(256), 0, st>>>(f, first, (uint32_t)n, (uint32_t)half,
                                                           (float)a, c, s);
  else if (quad)
    k_rope_tables<4, uint64_t><<<grid, dim3(256), 0, st>>>(f, first, (uint64_t)n, (uint64_t)half,
                                                           (float)a, c, s);
  else if (n < 0x7fffff00)
    k_rope_tables<1, uint32_t><<<grid, dim3(256), 0, st>>>(f, first, (uint32_t)n, (uint32_t)half,
                                                           (float)a, c, s);
  else
    k_rope_tables<1, uint64_t><<<grid, dim3(256), 0, st>>>(f, first, (uint64_t)n, (uint64_t)half,
                                                           (float)a, c, s);
  return mg_launch_check("rotary tables");
}

mg_status mg_rotate_run(mg_ctx *ctx, const mg_rotate_problem &p) {
  bool quad = aligned16(p.x) && aligned16(p.y) && aligned16(p.rope.cos_table) &&
              aligned16(p.rope.sin_table) && p.d % 4 == 0 && p.rope.half_rot % 4 == 0;
  for (int i = 0; i < 3; i++) quad = quad && p.xs[i] % 4 == 0 && p.ys[i] % 4 == 0;
  return quad ? rotate<4>(ctx, p) : rotate<1>(ctx, p);
}
