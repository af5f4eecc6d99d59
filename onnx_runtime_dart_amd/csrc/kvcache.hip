// Writing rows of keys and values to the quantised cache, and reading them back.
//
// A wave takes the up to four rows of one aligned group of four positions and one head:
// lane (t, c) = (l / 16, l % 16) takes token t's dims [c NB, (c + 1) NB) (NB = padded head size
// / 16), so a vector's extreme values join within 16 lanes (register moves) and all loads and
// stores of full rows are 16 bytes a lane.  Values of four tokens interleave in the cache:
// their codes change lanes through 16 NB words of shared memory, and one wave alone writes every
// byte of such a group (so a half-filled one can be read, merged and written).
//
// Codes are those of the exact quotient x / s, ties to even, whatever the order of the
// arithmetic: a candidate q = rint(x * (1 / s)) in 64 bits is at most one off, and its
// remainder x - q s (exact in a fused 64-bit step: 24-bit x and s, q of at most 8 bits)
// tells by comparison with s / 2 which neighbour is nearer.
//
// One pass of reads and writes bounds both directions.
#include <hip/hip_runtime.h>

#include <cmath>

#include "kv_common.h"
#include "rope_common.h"

namespace {

struct KvRows {
  mg_kv_cache c;
  mg_seq_batch s;
  const float *k, *v;
  float *ko, *vo;
  int64_t ks, vs;
  mg_rope rope;
};

// The group of four positions of a workgroup: blockIdx.x-th of sequence blockIdx.z.
struct Group {
  kv_seq q;
  int64_t page;  // -1: none
  int pos;       // of its first place
  int slot;      // that place in the page
};
// False: nothing to do.
__device__ inline bool group_of(const KvRows &a, Group *o) {
  const int64_t b = blockIdx.z;
  o->q = kv_sequence(a.s, b);
  if (o->q.bad) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
    return false;
  }
  o->pos = (o->q.past & ~3) + 4 * (int)blockIdx.x;
  if (o->pos >= o->q.past + o->q.n) return false;
  o->page = kv_page(a.s, b, o->pos, a.c.plog, a.c.pages);
  o->slot = o->pos & ((1 << a.c.plog) - 1);
  if (o->page < 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
  return true;
}

// Largest of the 16 lanes of a row of lanes.
template <int CTRL>
__device__ inline float turned(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                       0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ inline float max16(float x) {
  x = fmaxf(x, turned<0x128>(x));  // rotations of the row by 8, 4, 2, 1
  x = fmaxf(x, turned<0x124>(x));
  x = fmaxf(x, turned<0x122>(x));
  return fmaxf(x, turned<0x121>(x));
}

// The integer nearest x / s (ties to even) from r = 1 / s, as a double.
__device__ inline double nearest(double x, double s, double r) {
  const double q = rint(x * r), e = fma(-q, s, x);
  const double e2 = 2.0 * fabs(e);
  const bool odd = ((long long)q & 1) != 0;
  return e2 > s || (e2 == s && odd) ? q + copysign(1.0, e) : q;
}

// The codes of a vector, NB elements of it in each of 16 lanes (n of them belong to it).
template <int FMT, int NB>
__device__ inline void quantise(const float (&x)[NB], int n, uint32_t (&code)[NB], float &s,
                                float &m) {
  float hi = -__builtin_inff(), lo = -__builtin_inff();  // of x, of -x
  float odd = 0.f;                                       // Infinity or NaN: not 0
#pragma unroll
  for (int e = 0; e < NB; e++)
    if (e < n) {
      hi = fmaxf(hi, x[e]);
      lo = fmaxf(lo, -x[e]);
      odd = fmaxf(odd, __builtin_fabsf(x[e]) < __builtin_inff() ? 0.f : 1.f);
    }
  const bool ok = max16(odd) == 0.f;
  hi = max16(hi);
  lo = max16(lo);
  if (FMT == MG_KV_INT4) {
    m = (float)(((double)hi - (double)lo) * 0.5);
    s = (float)(((double)hi + (double)lo) / 30.0);
  } else {
    m = 0.f;
    s = (float)((double)fmaxf(hi, lo) / (FMT == MG_KV_INT8 ? 127.0 : 448.0));
  }
  const bool any = ok && s > 0.f;
  const double sd = any ? (double)s : 1.0, r = 1.0 / sd;
#pragma unroll
  for (int e = 0; e < NB; e++) {
    const double xd = any ? (double)x[e] : 0.0;
    if (FMT == MG_KV_INT8) {
      code[e] = (uint32_t)((int)fmin(fmax(nearest(xd, sd, r), -127.0), 127.0) + 128);
    } else if (FMT == MG_KV_INT4) {
      // ((x - m) / s + 15) / 2, its nearest integer by the remainder as above; s = 0: 8.
      const double d = any ? xd - (double)m : 0.0;
      const double q = rint((d * r + 15.0) * 0.5), rem = fma(15.0 - 2.0 * q, sd, d);
      const bool off = fabs(rem) > sd || (fabs(rem) == sd && ((int)q & 1));
      code[e] = (uint32_t)(int)fmin(fmax(off ? q + copysign(1.0, rem) : q, 0.0), 15.0);
    } else {
      // Steps of 2^(ex - 3) with ex the quotient's exponent, -6 at least (a quotient that
      // rounds across a power of two gives the same value from either side).
      const double u = xd * r;
      const int ex = max((int)(__double_as_longlong(u) >> 52 & 2047) - 1023, -6) - 3;
      const double q = fabs(nearest(xd, ldexp(sd, ex), ldexp(r, -ex)));  // 0 .. 16
      const int qi = (int)q;
      // 8 .. 15: mantissa q - 8 under exponent ex + 3; 16: the next power; below: subnormal.
      int bits = qi >= 16 ? (ex + 4 + 7) << 3 : qi >= 8 ? ((ex + 3 + 7) << 3) + qi - 8 : qi;
      bits = min(bits, 0x7e);  // 448
      code[e] = (uint32_t)bits | (__builtin_signbit(xd) ? 0x80u : 0u);
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

// n of NB adjacent elements; VEC: whole quads at 16-byte addresses.
template <int NB, bool VEC>
__device__ inline void load(float (&x)[NB], const float *p, int n) {
#pragma unroll
  for (int e = 0; e < NB; e += 4) {
    if (VEC) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (e < n) v = *reinterpret_cast<const float4 *>(p + e);
      x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) x[e + j] = e + j < n ? p[e + j] : 0.f;
    }
  }
}

// One wave a head: four heads a workgroup.
template <int FMT, int NB, bool VEC>
__global__ __launch_bounds__(256) void k_append(const KvRows a) {
  constexpr int DP = 16 * NB, RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;
  __shared__ uint32_t turn[4][4 * DP / 4];  // a wave's value codes, [token][dim] bytes
  const int lane = threadIdx.x & 63, t = lane >> 4, c = lane & 15, d0 = c * NB;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = blockIdx.y * 4 + wave;
  Group g;
  if (!group_of(a, &g) || g.page < 0 || h >= a.c.kv_heads) return;
  const int page = 1 << a.c.plog, n = a.c.d - d0;
  const int64_t ph = g.page * a.c.kv_heads + h;
  float *sc = a.c.sc + ph * kv_scales(FMT) * page + g.slot + t;
  const int i = g.pos + t - g.q.past;  // the lane's row of the sequence
  const bool in = i >= 0 && i < g.q.n;
  const int64_t row = g.q.start + (in ? i : 0);
  float x[NB], y[NB];
  uint32_t code[NB];
  float s, m;
  const float *kp = a.k + row * a.ks + (int64_t)h * a.c.d, *vp = a.v + row * a.vs + (int64_t)h * a.c.d;
  load<NB, VEC>(x, kp + d0, in ? n : 0);
  load<NB, VEC>(y, vp + d0, in ? n : 0);
  if (a.rope.half_rot) {
    const int half = (int)a.rope.half_rot;
    const int64_t pos = a.rope.positions ? a.rope.positions[row] : g.pos + t;
    if (VEC && !a.rope.interleaved && in && d0 < 2 * half) {
      // (half is a multiple of four: a quad's partners are a quad.)
      const bool known = (uint64_t)pos < (uint64_t)a.rope.max_pos;
      const int64_t at = (known ? pos : 0) * half;
#pragma unroll
      for (int e = 0; e < NB; e += 4) {
        const int d = d0 + e;
        if (d >= 2 * half) break;
        const bool second = d >= half;
        const int j = second ? d - half : d;
        const float4 z = *reinterpret_cast<const float4 *>(kp + (second ? j : d + half));
        const float4 cs = *reinterpret_cast<const float4 *>(a.rope.cos_table + at + j);
        const float4 sn = *reinterpret_cast<const float4 *>(a.rope.sin_table + at + j);
        auto turned_by = [&](float v, float w, float co, float si) {
          const double p = (double)v * co, q = (double)w * si;
          return known ? (float)(second ? p + q : p - q) : __builtin_nanf("");
        };
        x[e] = turned_by(x[e], z.x, cs.x, sn.x);
        x[e + 1] = turned_by(x[e + 1], z.y, cs.y, sn.y);
        x[e + 2] = turned_by(x[e + 2], z.z, cs.z, sn.z);
        x[e + 3] = turned_by(x[e + 3], z.w, cs.w, sn.w);
      }
    } else if (in) {
#pragma unroll
      for (int e = 0; e < NB; e++)
        if (e < n) x[e] = rope_at(kp, d0 + e, pos, a.rope);
    }
  }
  quantise<FMT, NB>(x, n, code, s, m);
  if (in) {
    uint8_t *kc = a.c.k + (ph * page + g.slot + t) * RB + d0 * RB / DP;
    if (c == 0) {
      sc[0] = s;
      if (FMT == MG_KV_INT4) sc[2 * page] = m;
    }
    if (FMT == MG_KV_INT4) {
#pragma unroll
      for (int e = 0; e < NB; e += 4)
        *reinterpret_cast<uint16_t *>(kc + e / 2) =
            (uint16_t)(code[e] | code[e + 1] << 4 | code[e + 2] << 8 | code[e + 3] << 12);
    } else {
#pragma unroll
      for (int e = 0; e < NB; e += 4)
        *reinterpret_cast<uint32_t *>(kc + e) =
            code[e] | code[e + 1] << 8 | code[e + 2] << 16 | code[e + 3] << 24;
    }
  }
  quantise<FMT, NB>(y, n, code, s, m);
  if (in && c == 0) {
    sc[page] = s;
    if (FMT == MG_KV_INT4) sc[3 * page] = m;
  }
  // (The wave's own part of turn: no barrier, only its own reads after its writes.)
  uint32_t *mine = turn[wave];
#pragma unroll
  for (int e = 0; e < NB; e += 4)
    mine[(t * DP + d0 + e) / 4] = code[e] | code[e + 1] << 8 | code[e + 2] << 16 | code[e + 3] << 24;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int first = max(0, g.q.past - g.pos), last = min(4, g.q.past + g.q.n - g.pos);
  uint32_t *vw = reinterpret_cast<uint32_t *>(a.c.v + (ph * page + g.slot) * RB);
  // Lane l: the codes of four dims at a time, all four tokens.
  for (int q = lane; q < DP / 4; q += 64) {
    uint32_t w[4], o[4];
#pragma unroll
    for (int u = 0; u < 4; u++) w[u] = mine[(u * DP) / 4 + q];
    uint32_t keep = 0;  // bits of tokens that are not of this call
    if (FMT == MG_KV_INT4) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        uint32_t bits = 0;
#pragma unroll
        for (int u = 0; u < 4; u++)
          bits |= (w[u] >> 8 * e & 15u) << 4 * v4_nibble(u, 0) |
                  (w[u] >> 8 * (e + 1) & 15u) << 4 * v4_nibble(u, 1);
        o[e / 2] = bits;
      }
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (u < first || u >= last) keep |= 0xfu << 4 * v4_nibble(u, 0) | 0xfu << 4 * v4_nibble(u, 1);
      uint2 *at = reinterpret_cast<uint2 *>(vw) + q;
      uint2 r = make_uint2(o[0], o[1]);
      if (keep) {
        const uint2 old = *at;
        r.x = (r.x & ~keep) | (old.x & keep);
        r.y = (r.y & ~keep) | (old.y & keep);
      }
      *at = r;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        o[e] = (w[0] >> 8 * e & 255u) | (w[1] >> 8 * e & 255u) << 8 | (w[2] >> 8 * e & 255u) << 16 |
               (w[3] >> 8 * e & 255u) << 24;
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (u < first || u >= last) keep |= 0xffu << 8 * u;
      uint4 *at = reinterpret_cast<uint4 *>(vw) + q;
      uint4 r = make_uint4(o[0], o[1], o[2], o[3]);
      if (keep) {
        const uint4 old = *at;
        r.x = (r.x & ~keep) | (old.x & keep);
        r.y = (r.y & ~keep) | (old.y & keep);
        r.z = (r.z & ~keep) | (old.z & keep);
        r.w = (r.w & ~keep) | (old.w & keep);
      }
      *at = r;
    }
  }
}

template <int FMT, int NB, bool VEC>
__global__ __launch_bounds__(256) void k_read(const KvRows a) {
  constexpr int DP = 16 * NB, RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;
  const int lane = threadIdx.x & 63, t = lane >> 4, c = lane & 15, d0 = c * NB;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = blockIdx.y * 4 + wave;
  Group g;
  if (!group_of(a, &g) || h >= a.c.kv_heads) return;
  const int i = g.pos + t - g.q.past, n = a.c.d - d0;
  if (i < 0 || i >= g.q.n || n <= 0) return;
  const int page = 1 << a.c.plog;
  const bool bad = g.page < 0;
  const int64_t ph = (bad ? 0 : g.page) * a.c.kv_heads + h;
  const float *sc = a.c.sc + ph * kv_scales(FMT) * page + g.slot + t;
  const uint8_t *kc = a.c.k + (ph * page + g.slot + t) * RB + d0 * RB / DP;
  const uint32_t *vw = reinterpret_cast<const uint32_t *>(a.c.v + (ph * page + g.slot) * RB);
  const float nan = __builtin_nanf("");
  const float ks = bad ? nan : sc[0], km = FMT == MG_KV_INT4 ? sc[2 * page] : 0.f;
  const float vs = bad ? nan : sc[page], vm = FMT == MG_KV_INT4 ? sc[3 * page] : 0.f;
  const int64_t row = g.q.start + i;
  float *ko = a.ko + row * a.ks + (int64_t)h * a.c.d + d0;
  float *vo = a.vo + row * a.vs + (int64_t)h * a.c.d + d0;
#pragma unroll
  for (int e = 0; e < NB; e += 4) {
    uint32_t kw, cv[4];
    float x[4], y[4];
    if (FMT == MG_KV_INT4) {
      kw = *reinterpret_cast<const uint16_t *>(kc + e / 2);
      const uint2 w = *reinterpret_cast<const uint2 *>(vw + (d0 + e) / 2);
      cv[0] = w.x >> 4 * v4_nibble(t, 0) & 15u, cv[1] = w.x >> 4 * v4_nibble(t, 1) & 15u;
      cv[2] = w.y >> 4 * v4_nibble(t, 0) & 15u, cv[3] = w.y >> 4 * v4_nibble(t, 1) & 15u;
    } else {
      kw = *reinterpret_cast<const uint32_t *>(kc + e);
      const uint4 w = *reinterpret_cast<const uint4 *>(vw + d0 + e);
      cv[0] = w.x >> 8 * t & 255u, cv[1] = w.y >> 8 * t & 255u;
      cv[2] = w.z >> 8 * t & 255u, cv[3] = w.w >> 8 * t & 255u;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t ck = FMT == MG_KV_INT4 ? kw >> 4 * j & 15u : kw >> 8 * j & 255u;
      x[j] = value_of<FMT>(ck, ks, km);
      y[j] = value_of<FMT>(cv[j], vs, vm);
    }
    if (VEC) {
      if (e < n) {
        *reinterpret_cast<float4 *>(ko + e) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(vo + e) = make_float4(y[0], y[1], y[2], y[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (e + j < n) {
          ko[e + j] = x[j];
          vo[e + j] = y[j];
        }
    }
  }
}

__global__ __launch_bounds__(256) void k_fill(uint4 *p, int64_t n, uint32_t word) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    p[i] = make_uint4(word, word, word, word);
}

template <int FMT, int NB, bool VEC>
void launch(mg_ctx *ctx, const KvRows &a, bool read) {
  // Groups of four that a sequence of max_new rows can touch.
  const int64_t groups = (a.s.max_new + 2) / 4 + 1;
  const dim3 grid((unsigned)groups, (unsigned)((a.c.kv_heads + 3) / 4), (unsigned)a.s.batch);
  if (read)
    k_read<FMT, NB, VEC><<<grid, dim3(256), 0, ctx->stream>>>(a);
  else
    k_append<FMT, NB, VEC><<<grid, dim3(256), 0, ctx->stream>>>(a);
}

template <int FMT, bool VEC>
void launch_dims(mg_ctx *ctx, const KvRows &a, bool read) {
  switch (a.c.dp / 64) {
    case 1: return launch<FMT, 4, VEC>(ctx, a, read);
    case 2: return launch<FMT, 8, VEC>(ctx, a, read);
    case 3: return launch<FMT, 12, VEC>(ctx, a, read);
    default: return launch<FMT, 16, VEC>(ctx, a, read);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

mg_status run(mg_ctx *ctx, const KvRows &a, bool read) {
  const bool vec = a.c.d % 4 == 0 && a.ks % 4 == 0 && a.vs % 4 == 0 && aligned16(a.k) &&
                   aligned16(a.v) && aligned16(a.ko) && aligned16(a.vo) &&
                   a.rope.half_rot % 4 == 0 && aligned16(a.rope.cos_table) &&
                   aligned16(a.rope.sin_table);
  switch (a.c.fmt * 2 + vec) {
    case MG_KV_INT8 * 2: launch_dims<MG_KV_INT8, false>(ctx, a, read); break;
    case MG_KV_INT8 * 2 + 1: launch_dims<MG_KV_INT8, true>(ctx, a, read); break;
    case MG_KV_E4M3 * 2: launch_dims<MG_KV_E4M3, false>(ctx, a, read); break;
    case MG_KV_E4M3 * 2 + 1: launch_dims<MG_KV_E4M3, true>(ctx, a, read); break;
    case MG_KV_INT4 * 2: launch_dims<MG_KV_INT4, false>(ctx, a, read); break;
    default: launch_dims<MG_KV_INT4, true>(ctx, a, read); break;
  }
  return mg_launch_check(read ? "KV cache read" : "KV cache append");
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
