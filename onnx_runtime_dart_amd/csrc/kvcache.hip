// Writing rows of keys and values to the quantised cache, and reading them back.
//
// A wave takes the up to four rows of one aligned group of four positions and one head: the
// values of four tokens interleave in the cache, so one wave alone writes every byte of
// such a group.  Lane l owns E adjacent dims.  Each vector's extreme values are joined
// across the wave, its codes formed in 64 bits (so that they are those of the exact
// quotient, whatever the order of the arithmetic) and packed in the lane.
// One pass of reads and writes bounds both directions.
#include <hip/hip_runtime.h>

#include <cmath>

#include "kv_common.h"
#include "rope_common.h"

namespace {

constexpr int kTok = 4;

struct KvRows {
  mg_kv_cache c;
  mg_seq_batch s;
  const float *k, *v;
  float *ko, *vo;
  int64_t ks, vs;
  mg_rope rope;
};

// The group of four positions of a wave: g-th of sequence b.
struct Group {
  kv_seq q;
  int64_t page;  // -1: none
  int pos;       // of its first place
  int slot;      // that place in the page
  bool in[kTok];
};
__device__ inline bool group_of(const KvRows &a, int64_t b, int g, Group *o) {
  o->q = kv_sequence(a.s, b);
  if (o->q.bad) {
    if (g == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
    return false;
  }
  o->pos = (o->q.past & ~3) + 4 * g;
  if (o->pos >= o->q.past + o->q.n) return false;
  o->page = kv_page(a.s, b, o->pos, a.c.plog, a.c.pages);
  o->slot = o->pos & ((1 << a.c.plog) - 1);
#pragma unroll
  for (int t = 0; t < kTok; t++)
    o->in[t] = o->pos + t >= o->q.past && o->pos + t < o->q.past + o->q.n;
  return true;
}

__device__ inline float wave_max(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ inline bool finite(float x) { return __builtin_fabsf(x) < __builtin_inff(); }

// The codes of one vector: E elements of it a lane, of which n belong to the vector.
template <int FMT, int E>
__device__ inline void quantise(const float (&x)[E], int n, uint32_t (&code)[E], float &s,
                                float &m) {
  float hi = -__builtin_inff(), lo = __builtin_inff();
  bool ok = true;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (e < n) {
      hi = fmaxf(hi, x[e]);
      lo = fminf(lo, x[e]);
      ok &= finite(x[e]);
    }
  }
  ok = __all(ok);
  hi = wave_max(hi);
  lo = -wave_max(-lo);
  if (FMT == MG_KV_INT4) {
    m = (float)(((double)hi + (double)lo) * 0.5);
    s = (float)(((double)hi - (double)lo) / 30.0);
  } else {
    m = 0.f;
    s = (float)((double)fmaxf(hi, -lo) / (FMT == MG_KV_INT8 ? 127.0 : 448.0));
  }
#pragma unroll
  for (int e = 0; e < E; e++) {
    const double u = ok && s > 0.f ? ((double)x[e] - (double)m) / (double)s : 0.0;
    if (FMT == MG_KV_INT8) {
      code[e] = (uint32_t)((int)fmin(fmax(rint(u), -127.0), 127.0) + 128);
    } else if (FMT == MG_KV_INT4) {
      code[e] = (uint32_t)(int)fmin(fmax(rint((u + 15.0) * 0.5), 0.0), 15.0);
    } else {
      // Steps of 2^(e - 3) with e the exponent, -6 at least.
      int ex;
      (void)frexp(u, &ex);
      ex = max(ex - 1, -6) - 3;
      const double r = fmin(fabs(rint(ldexp(u, -ex))), ldexp(448.0, -ex));  // 0 .. 16
      // r in [8, 16): mantissa r - 8 of exponent ex + 3; below: subnormal (ex = -9).
      const int q = (int)r;
      const int bits = q >= 16 ? (ex + 4 + 7) << 3 : q >= 8 ? ((ex + 3 + 7) << 3) + q - 8 : q;
      code[e] = (uint32_t)bits | (__builtin_signbit(u) ? 0x80u : 0u);
    }
  }
  if (!ok) {
    s = __builtin_nanf("");
    m = s;
  }
}

template <int FMT>
__device__ inline float value_of(uint32_t code, float s, float m) {
  if (FMT == MG_KV_INT8) return (float)((int)code - 128) * s;
  if (FMT == MG_KV_INT4) return fmaf((float)(2 * (int)code - 15), s, m);
  // e4m3 as fp16 bits with a bias lower by 8.
  const uint32_t h = (code & 0x80u) << 8 | (code & 0x7fu) << 7;
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h) * 256.f * s;
}

// Nibble of token t of the pair's first (0) or second (1) dim in its dword.
__device__ __host__ constexpr int v4_nibble(int t, int second) {
  return 4 * (t & 1) + 2 * second + (t >> 1);
}

template <int FMT, int E>
__global__ __launch_bounds__(256) void k_append(const KvRows a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = blockIdx.y * 4 + wave;
  Group g;
  if (!group_of(a, blockIdx.z, blockIdx.x, &g)) return;
  if (g.page < 0) {
    if (threadIdx.x == 0) atomicOr(a.c.refused, 1);
    return;
  }
  if (h >= a.c.kv_heads) return;
  const int d0 = lane * E, page = 1 << a.c.plog;
  const bool mine = d0 < a.c.dp;
  const int64_t ph = g.page * a.c.kv_heads + h;
  float *sc = a.c.sc + ph * kv_scales(FMT) * page + g.slot;
  uint8_t *kc = a.c.k + ph * page * (a.c.dp * kv_bits(FMT) / 8);
  uint8_t *vc = a.c.v + ph * page * (a.c.dp * kv_bits(FMT) / 8);
  uint32_t vcode[kTok][E];
#pragma unroll
  for (int t = 0; t < kTok; t++) {
    if (!g.in[t]) continue;
    const int64_t row = g.q.start + (g.pos + t - g.q.past);
    float x[E];
    uint32_t code[E];
    float s, m;
    const float *src = a.k + row * a.ks + (int64_t)h * a.c.d;
    const int64_t pos = a.rope.half_rot && a.rope.positions ? a.rope.positions[row] : g.pos + t;
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = d0 + e < a.c.d ? rope_at(src, d0 + e, pos, a.rope) : 0.f;
    quantise<FMT, E>(x, a.c.d - d0, code, s, m);
    if (lane == 0) {
      sc[t] = s;
      if (FMT == MG_KV_INT4) sc[2 * page + t] = m;
    }
    if (mine) {
      const int64_t at = (int64_t)(g.slot + t) * a.c.dp + d0;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if (FMT == MG_KV_INT4)
          kc[(at + e) / 2] = (uint8_t)(code[e] | code[e + 1] << 4);
        else
          *reinterpret_cast<uint16_t *>(kc + at + e) = (uint16_t)(code[e] | code[e + 1] << 8);
      }
    }
    src = a.v + row * a.vs + (int64_t)h * a.c.d;
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = d0 + e < a.c.d ? src[d0 + e] : 0.f;
    quantise<FMT, E>(x, a.c.d - d0, vcode[t], s, m);
    if (lane == 0) {
      sc[page + t] = s;
      if (FMT == MG_KV_INT4) sc[3 * page + t] = m;
    }
  }
  if (!mine) return;
  if (FMT == MG_KV_INT4) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      uint32_t *w = reinterpret_cast<uint32_t *>(vc) + ((int64_t)(g.slot / 4) * a.c.dp + d0 + e) / 2;
      uint32_t mask = 0, bits = 0;
#pragma unroll
      for (int t = 0; t < kTok; t++)
        if (g.in[t]) {
          mask |= 0xfu << 4 * v4_nibble(t, 0) | 0xfu << 4 * v4_nibble(t, 1);
          bits |= vcode[t][e] << 4 * v4_nibble(t, 0) | vcode[t][e + 1] << 4 * v4_nibble(t, 1);
        }
      *w = mask == 0xffffffffu ? bits : ((*w & ~mask) | bits);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) {
      uint32_t *w = reinterpret_cast<uint32_t *>(vc) + (int64_t)(g.slot / 4) * a.c.dp + d0 + e;
      uint32_t mask = 0, bits = 0;
#pragma unroll
      for (int t = 0; t < kTok; t++)
        if (g.in[t]) {
          mask |= 0xffu << 8 * t;
          bits |= vcode[t][e] << 8 * t;
        }
      *w = mask == 0xffffffffu ? bits : ((*w & ~mask) | bits);
    }
  }
}

template <int FMT, int E>
__global__ __launch_bounds__(256) void k_read(const KvRows a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = blockIdx.y * 4 + wave;
  Group g;
  if (!group_of(a, blockIdx.z, blockIdx.x, &g)) return;
  if (g.page < 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
  if (h >= a.c.kv_heads) return;
  const int d0 = lane * E, page = 1 << a.c.plog;
  if (d0 >= a.c.d) return;
  const int64_t ph = (g.page < 0 ? 0 : g.page) * a.c.kv_heads + h;
  const float *sc = a.c.sc + ph * kv_scales(FMT) * page + g.slot;
  const uint8_t *kc = a.c.k + ph * page * (a.c.dp * kv_bits(FMT) / 8);
  const uint8_t *vc = a.c.v + ph * page * (a.c.dp * kv_bits(FMT) / 8);
  uint32_t vw[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int64_t at = (int64_t)(g.slot / 4) * a.c.dp + d0 + e;
    vw[e] = FMT == MG_KV_INT4 ? reinterpret_cast<const uint32_t *>(vc)[at / 2]
                              : reinterpret_cast<const uint32_t *>(vc)[at];
  }
#pragma unroll
  for (int t = 0; t < kTok; t++) {
    if (!g.in[t]) continue;
    const int64_t row = g.q.start + (g.pos + t - g.q.past);
    const bool bad = g.page < 0;
    const float nan = __builtin_nanf("");
    const float s = bad ? nan : sc[t], m = FMT == MG_KV_INT4 ? sc[2 * page + t] : 0.f;
    const float vs = bad ? nan : sc[page + t], vm = FMT == MG_KV_INT4 ? sc[3 * page + t] : 0.f;
    const int64_t at = (int64_t)(g.slot + t) * a.c.dp + d0;
    float *ko = a.ko + row * a.ks + (int64_t)h * a.c.d + d0;
    float *vo = a.vo + row * a.vs + (int64_t)h * a.c.d + d0;
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (d0 + e >= a.c.d) continue;
      const uint32_t ck = FMT == MG_KV_INT4 ? kc[(at + e) / 2] >> 4 * (e & 1) & 15u : kc[at + e];
      const uint32_t cv = FMT == MG_KV_INT4 ? vw[e] >> 4 * v4_nibble(t, e & 1) & 15u
                                            : vw[e] >> 8 * t & 255u;
      ko[e] = value_of<FMT>(ck, s, m);
      vo[e] = value_of<FMT>(cv, vs, vm);
    }
  }
}

__global__ __launch_bounds__(256) void k_fill(uint4 *p, int64_t n, uint32_t word) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    p[i] = make_uint4(word, word, word, word);
}

template <int FMT, int E>
mg_status launch(mg_ctx *ctx, const KvRows &a, bool read) {
  // Groups of four that a sequence of max_new rows can touch.
  const int64_t groups = (a.s.max_new + 2) / 4 + 1;
  const dim3 grid((unsigned)groups, (unsigned)((a.c.kv_heads + 3) / 4), (unsigned)a.s.batch);
  if (read)
    k_read<FMT, E><<<grid, dim3(256), 0, ctx->stream>>>(a);
  else
    k_append<FMT, E><<<grid, dim3(256), 0, ctx->stream>>>(a);
  return mg_launch_check(read ? "KV cache read" : "KV cache append");
}

mg_status run(mg_ctx *ctx, const KvRows &a, bool read) {
  const bool wide = a.c.dp > 128;
  switch (a.c.fmt) {
    case MG_KV_INT8:
      return wide ? launch<MG_KV_INT8, 4>(ctx, a, read) : launch<MG_KV_INT8, 2>(ctx, a, read);
    case MG_KV_E4M3:
      return wide ? launch<MG_KV_E4M3, 4>(ctx, a, read) : launch<MG_KV_E4M3, 2>(ctx, a, read);
    default:
      return wide ? launch<MG_KV_INT4, 4>(ctx, a, read) : launch<MG_KV_INT4, 2>(ctx, a, read);
  }
}

}  // namespace

// All codes of value 0 (no NaN code is ever in the cache) and scales 0.
mg_status mg_kv_clear(mg_ctx *ctx, mg_kv_cache *c) {
  const int64_t tokens = c->pages * c->kv_heads << c->plog;
  const int64_t codes = tokens * c->dp * kv_bits(c->fmt) / 8 / 16;
  const int64_t scales = tokens * kv_scales(c->fmt) * 4 / 16;
  const uint32_t zero = c->fmt == MG_KV_INT8 ? 0x80808080u : 0u;
  const auto grid = [](int64_t n) { return dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096)); };
  hipStream_t st = ctx->stream;
  k_fill<<<grid(codes), dim3(256), 0, st>>>(reinterpret_cast<uint4 *>(c->k), codes, zero);
  k_fill<<<grid(codes), dim3(256), 0, st>>>(reinterpret_cast<uint4 *>(c->v), codes, zero);
  k_fill<<<grid(scales), dim3(256), 0, st>>>(reinterpret_cast<uint4 *>(c->sc), scales, 0u);
  k_fill<<<dim3(1), dim3(256), 0, st>>>(reinterpret_cast<uint4 *>(c->refused), 1, 0u);
  return mg_launch_check("KV cache clear");
}

mg_status mg_kv_append_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s,
                           const float *k, int64_t ks, const float *v, int64_t vs,
                           const mg_rope *rope) {
  KvRows a{c, s, k, v, nullptr, nullptr, ks, vs, rope ? *rope : mg_rope{}};
  return run(ctx, a, false);
}

mg_status mg_kv_read_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s, float *k,
                         int64_t ks, float *v, int64_t vs) {
  KvRows a{c, s, nullptr, nullptr, k, v, ks, vs, mg_rope{}};
  return run(ctx, a, true);
}
