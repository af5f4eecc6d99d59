// Writing rows of keys and values to the quantised cache, and reading them back.
//
// A wave takes four aligned positions of one head at a time: lane (t, c) = (l / 16, l % 16)
// takes NB = padded head size / 16 dims of token t, so a vector's extreme values join within 16
// lanes (register moves) and loads and stores of full rows are 16 bytes a lane.  Values of four
// tokens interleave in the cache:
// their codes change lanes through 16 NB words of shared memory, and one wave alone writes every
// byte of such a group (so a half-filled one can be read, merged and written).
//
// Codes are those of the exact quotient x / s, ties to even, whatever the order of the
// arithmetic: the quotient is bracketed in fp32, and only where the bracket's ends round to
// different codes (near a tie, one vector in some hundred) are 64-bit quotients formed.
//
// One pass of reads and writes bounds both directions.  10k tokens of 8 heads of 128 (int8):
// written in 25 us (4.1 TB/s), rotated first in 36 us (what the rotation adds is its chain of
// positions and tables and its 64-bit conversions), read back in 24 us (4.2 TB/s).  A
// wave reads 16 positions (the chain of lengths, page and codes is paid once: 33 -> 24 us) and
// writes four (with 16 the arithmetic of one group waits for the last's: 39 -> 49 us).
#include <hip/hip_runtime.h>

#include <cmath>

#include "kv_common.h"
#include "rope_common.h"

namespace {

constexpr int kWrite = 4, kRead = 16;  // positions a wave takes

struct KvRows {
  mg_kv_cache c;
  mg_seq_batch s;
  const float *k, *v;
  float *ko, *vo;
  int64_t ks, vs;
  mg_rope rope;
  int hpw;  // heads a wave takes (append)
};

// The aligned positions of a workgroup (4 or 16, in one page): blockIdx.x-th such block of
// sequence blockIdx.z.
struct Block {
  kv_seq q;
  int64_t page;     // -1: none
  int pos;          // of its first place
  int slot;         // that place in the page
  int first, last;  // its groups of four that hold rows: first .. last - 1
};
// False: nothing to do.
template <int SPAN>
__device__ inline bool block_of(const KvRows &a, Block *o) {
  const int64_t b = blockIdx.z;
  o->q = kv_sequence(a.s, b);
  if (o->q.bad) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
    return false;
  }
  // (64 bits: past may be near 2^31 and the grid made for more rows than the sequence has.)
  const int end = o->q.past + o->q.n;
  const int64_t at = (o->q.past & ~(SPAN - 1)) + (int64_t)SPAN * blockIdx.x;
  if (o->q.n == 0 || at >= end) return false;
  o->pos = (int)at;
  o->page = kv_page(a.s, b, o->pos, a.c.plog, a.c.pages);
  o->slot = o->pos & ((1 << a.c.plog) - 1);
  o->first = max(o->q.past - o->pos, 0) >> 2;
  o->last = (min(end - o->pos, SPAN) + 3) >> 2;
  if (o->page < 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
  return true;
}

// Joined over the 16 lanes of a row of lanes: rotations of the row by 8, 4, 2, 1.
template <int CTRL>
__device__ inline uint32_t turned(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
__device__ inline uint32_t max16(uint32_t x) {
  x = max(x, turned<0x128>(x));
  x = max(x, turned<0x124>(x));
  x = max(x, turned<0x122>(x));
  return max(x, turned<0x121>(x));
}
__device__ inline float max16(float x) {
  auto with = [&](uint32_t y) { x = fmaxf(x, __uint_as_float(y)); };
  with(turned<0x128>(__float_as_uint(x)));
  with(turned<0x124>(__float_as_uint(x)));
  with(turned<0x122>(__float_as_uint(x)));
  with(turned<0x121>(__float_as_uint(x)));
  return x;
}

// The code of x by the quotients themselves, in 64 bits (any false: of 0).
template <int FMT>
__device__ inline uint32_t exact_code(float x, float s, float m, bool any) {
  const double u = any ? ((double)x - (double)m) / (double)s : 0.0;
  if (FMT == MG_KV_INT8) return (uint32_t)((int)fmin(fmax(rint(u), -127.0), 127.0) + 128);
  if (FMT == MG_KV_INT4) return (uint32_t)(int)fmin(fmax(rint((u + 15.0) * 0.5), 0.0), 15.0);
  // Steps of 2^ex: 2^-3 of the quotient's power of two, 2^-9 at least.
  const int ex = max((int)(__double_as_longlong(u) >> 52 & 2047) - 1023, -6) - 3;
  const int q = (int)fmin(fabs(rint(ldexp(u, -ex))), ldexp(448.0, -ex));  // 0 .. 16
  // 8 .. 15: mantissa q - 8 under exponent ex + 3; 16: the next power; below: subnormal.
  const int bits = q >= 16 ? (ex + 4 + 7) << 3 : q >= 8 ? ((ex + 3 + 7) << 3) + q - 8 : q;
  return (uint32_t)bits | (any ? __float_as_uint(x) >> 24 & 0x80u : 0u);
}

// Four codes from quotients (INT4: already (u + 15) / 2).
template <int FMT>
__device__ inline uint32_t rounded4(float a, float b, float c, float d) {
  if (FMT == MG_KV_E4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
  // Added to 1.5 2^23 a number rounds to an integer, its low byte that of the sum.
  const float big = FMT == MG_KV_INT8 ? 12582912.f + 128.f : 12582912.f;
  const uint32_t p = __builtin_amdgcn_perm(__float_as_uint(b + big), __float_as_uint(a + big), 0x0c0c0400u);
  const uint32_t q = __builtin_amdgcn_perm(__float_as_uint(d + big), __float_as_uint(c + big), 0x04000c0cu);
  return p | q;
}

// The codes of a vector, NB elements of it in each of 16 lanes, four to a dword (INT4: one a byte).
template <int FMT, int NB>
__device__ inline void quantise(const float (&x)[NB], uint32_t (&code)[NB / 4], float &s, float &m) {
  // Sizes as bits: what is not finite is above all that is.
  uint32_t size = 0;
#pragma unroll
  for (int e = 0; e < NB; e++) size = max(size, __float_as_uint(x[e]) & 0x7fffffffu);
  size = max16(size);
  const bool ok = size < 0x7f800000u;
  m = 0.f;
  if (FMT == MG_KV_INT4) {
    float hi = x[0], lo = -x[0];  // of x, of -x
#pragma unroll
    for (int e = 1; e < NB; e++) {
      hi = fmaxf(hi, x[e]);
      lo = fmaxf(lo, -x[e]);
    }
    hi = max16(hi);
    lo = max16(lo);
    m = (float)(((double)hi - (double)lo) * 0.5);
    s = (float)(((double)hi + (double)lo) / 30.0);
  } else {
    s = (float)((double)__uint_as_float(size) / (FMT == MG_KV_INT8 ? 127.0 : 448.0));
  }
  const bool any = ok && s > 0.f;
  // The quotient lies between x r (1 - 2^-21) and x r (1 + 2^-21) (INT4: (u + 15) / 2 within
  // 2^-18 of its fp32 form): where both ends round alike, so does it.
  const float r = any ? 1.f / s : 0.f;
  uint32_t differ = any && s < 0x1p-100f ? 1u : 0u;
#pragma unroll
  for (int e = 0; e < NB; e += 4) {
    float a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (FMT == MG_KV_INT4) {
        // (m is rounded: of extremes few units in the last place apart one may lie beyond 15 steps.)
        const float u = fminf(fmaxf(fmaf(x[e + j] - m, 0.5f * r, 7.5f), 0.f), 15.f);
        a[j] = u - 0x1p-18f;
        b[j] = u + 0x1p-18f;
      } else {
        a[j] = x[e + j] * (r * (1.f - 0x1p-21f));
        b[j] = x[e + j] * (r * (1.f + 0x1p-21f));
      }
    }
    code[e / 4] = rounded4<FMT>(a[0], a[1], a[2], a[3]);
    differ |= code[e / 4] ^ rounded4<FMT>(b[0], b[1], b[2], b[3]);
  }
  if (__any(differ != 0)) {
    asm volatile("");  // (kept a branch: few vectors come here)
#pragma unroll
    for (int e = 0; e < NB; e += 4) {
      code[e / 4] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) code[e / 4] |= exact_code<FMT>(x[e + j], s, m, any) << 8 * j;
    }
  }
  if (!ok) {
#pragma unroll
    for (int e = 0; e < NB / 4; e++) code[e] = 0;
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

// Element e of a lane that writes: adjacent dims, so its codes are adjacent bytes.  One that
// reads back: every fourth quad, so that 16 lanes store 256 adjacent bytes with each access (with
// adjacent dims, half lines at a time: 40k tokens of 8 heads 150 us, not 86).
template <int NB>
__device__ inline int dim_of(int e, int c) {
  return NB * c + e;
}
__device__ inline int read_dim(int e, int c) { return 64 * (e / 4) + 4 * c + e % 4; }

// The lane's elements of a vector of d at p; the padding past its end repeats its first element
// (which changes no extreme).  VEC: d is a multiple of four, quads at 16-byte addresses.
template <int NB, bool VEC>
__device__ inline void load(float (&x)[NB], const float *p, int c, int d) {
#pragma unroll
  for (int e = 0; e < NB; e += 4) {
    const int i = dim_of<NB>(e, c);
    if (VEC) {
      const bool in = i < d;
      const float4 v = *reinterpret_cast<const float4 *>(p + (in ? i : 0));
      x[e] = v.x, x[e + 1] = in ? v.y : v.x, x[e + 2] = in ? v.z : v.x, x[e + 3] = in ? v.w : v.x;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) x[e + j] = p[i + j < d ? i + j : 0];
    }
  }
}

// The pairs' other elements (of elements that are not turned: any).
template <int NB, bool VEC>
__device__ inline void load_others(float (&z)[NB], const float *p, int c, int d, const mg_rope &rope) {
  const int half = (int)rope.half_rot;
#pragma unroll
  for (int e = 0; e < NB; e += 4) {
    const int i0 = dim_of<NB>(e, c) < d ? dim_of<NB>(e, c) : 0;
    if (VEC && !rope.interleaved) {
      // (half is a multiple of four: a quad's partners are a quad.)
      const int j = i0 >= 2 * half ? 0 : i0 >= half ? i0 - half : i0 + half;
      const float4 v = *reinterpret_cast<const float4 *>(p + j);
      z[e] = v.x, z[e + 1] = v.y, z[e + 2] = v.z, z[e + 3] = v.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = dim_of<NB>(e + k, c) < d ? dim_of<NB>(e + k, c) : 0;
        const int j = rope.interleaved ? i ^ 1 : i >= half ? i - half : i + half;
        z[e + k] = p[i < 2 * half ? j : 0];
      }
    }
  }
}
// Turns the lane's elements x of a vector of d by the cosines and sines of its token: x c + z s
// with z the pair's other element, s negative for a pair's first.  The products are exact in 64
// bits; the sum rounds there and once more to fp32, as in the rotation of its own.
template <int NB, bool VEC>
__device__ inline void turn_key(float (&x)[NB], const float (&z)[NB], const float *ct, const float *st,
                                int c, int d, int half, bool interleaved) {
#pragma unroll
  for (int e = 0; e < NB; e++) {
    const int i = dim_of<NB>(e, c) < d ? dim_of<NB>(e, c) : 0;
    if (i < 2 * half) {
      const bool second = interleaved ? (i & 1) != 0 : i >= half;
      const int j = interleaved ? i >> 1 : second ? i - half : i;
      const double p = (double)z[e] * (double)st[j];
      x[e] = (float)fma((double)x[e], (double)ct[j], second ? p : -p);
    }
    // (Padding stays the first element, turned; VEC loads put four of it side by side.)
    if (VEC && e % 4 && dim_of<NB>(e, c) >= d) x[e] = x[e & ~3];
  }
}

template <int FMT, int NB, bool VEC, bool ROPE>
__global__ __launch_bounds__(256) void k_append(const KvRows a) {
  constexpr int DP = 16 * NB, RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;
  constexpr int VQ = FMT == MG_KV_INT4 ? 2 : 4;  // dwords of four dims of four values
  constexpr int LQ = (DP / 4 + 63) / 64;         // such runs a lane
  __shared__ uint32_t turn[4][4 * DP / 4];  // a wave's value codes, [token][dim] bytes
  // The four tokens' cosines and sines, for all heads.
  __shared__ float table[ROPE ? 2 : 1][ROPE ? 4 * MG_ROPE_MAX_HALF : 1];
  const int lane = threadIdx.x & 63, t = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h0 = (blockIdx.y * 4 + wave) * a.hpw;
  Block g;
  if (!block_of<kWrite>(a, &g) || g.page < 0) return;
  const int page = 1 << a.c.plog, slot = g.slot;
  const int i = g.pos + t - g.q.past;  // the lane's row of the sequence
  const bool in = i >= 0 && i < g.q.n;
  const int64_t row = g.q.start + min(max(i, 0), g.q.n - 1);  // (lanes without one read another)
  // Bits of the values' dwords that belong to tokens of other calls.
  const int first = max(0, g.q.past - g.pos), last = min(4, g.q.past + g.q.n - g.pos);
  uint32_t keep = 0;
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (k < first || k >= last)
      keep |= FMT == MG_KV_INT4 ? 0xfu << 4 * v4_nibble(k, 0) | 0xfu << 4 * v4_nibble(k, 1)
                                : 0xffu << 8 * k;
  uint32_t *mine = turn[wave];
  const int h1 = min(h0 + a.hpw, a.c.kv_heads);
  float x[NB], y[NB], z[NB];
  auto vectors = [&](int h) {
    const float *kp = a.k + row * a.ks + (int64_t)h * a.c.d;
    load<NB, VEC>(x, kp, c, a.c.d);
    if (ROPE) load_others<NB, VEC>(z, kp, c, a.c.d, a.rope);
    load<NB, VEC>(y, a.v + row * a.vs + (int64_t)h * a.c.d, c, a.c.d);
  };
  const int half = (int)a.rope.half_rot;
  if (ROPE) {
    for (int j = threadIdx.x; j < 4 * half; j += 256) {
      const int k = j / half, n = j - k * half;
      const int at = min(max(g.pos + k - g.q.past, 0), g.q.n - 1);
      const int64_t pos = a.rope.positions ? (int64_t)a.rope.positions[g.q.start + at]
                                           : (int64_t)(g.q.past + at);
      const bool known = (uint64_t)pos < (uint64_t)a.rope.max_pos;
      const int64_t o = (known ? pos : 0) * half + n;
      table[0][j] = known ? a.rope.cos_table[o] : __builtin_nanf("");
      table[ROPE][j] = a.rope.sin_table[o];
    }
  }
  if (h0 < h1) vectors(h0);
  if (ROPE) __syncthreads();
  for (int h = h0; h < h1; h++) {
    const int64_t ph = g.page * a.c.kv_heads + h;
    uint32_t *vw = reinterpret_cast<uint32_t *>(a.c.v + (ph * page + slot) * RB);
    uint32_t old[LQ][VQ] = {};
    if (keep) {
#pragma unroll
      for (int q = 0; q < LQ; q++)
#pragma unroll
        for (int w = 0; w < VQ; w++)
          if (lane + 64 * q < DP / 4) old[q][w] = vw[(lane + 64 * q) * VQ + w];
    }
    if (ROPE)
      turn_key<NB, VEC>(x, z, table[0] + t * half, table[ROPE] + t * half, c, a.c.d, half,
                        a.rope.interleaved);
    uint32_t code[NB / 4];
    float s, m;
    float *sc = a.c.sc + ph * kv_scales(FMT) * page + slot + t;
    quantise<FMT, NB>(x, code, s, m);
    if (in) {
      uint8_t *kc = a.c.k + (ph * page + slot + t) * RB;
      if (c == 0) {
        sc[0] = s;
        if (FMT == MG_KV_INT4) sc[2 * page] = m;
      }
#pragma unroll
      for (int e = 0; e < NB; e += 4) {
        if (FMT == MG_KV_INT4) {
          const uint32_t w = code[e / 4] | code[e / 4] >> 4;  // nibbles 0, 1 and 4, 5
          *reinterpret_cast<uint16_t *>(kc + dim_of<NB>(e, c) / 2) =
              (uint16_t)((w & 0xffu) | (w >> 8 & 0xff00u));
        } else {
          *reinterpret_cast<uint32_t *>(kc + dim_of<NB>(e, c)) = code[e / 4];
        }
      }
    }
    quantise<FMT, NB>(y, code, s, m);
    if (in && c == 0) {
      sc[page] = s;
      if (FMT == MG_KV_INT4) sc[3 * page] = m;
    }
    if (h + 1 < h1) vectors(h + 1);
    // (The wave's own part of turn: no barrier, only its own order of writes and reads.)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < NB; e += 4) mine[(t * DP + dim_of<NB>(e, c)) / 4] = code[e / 4];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // Lane l: the codes of four dims at a time, all four tokens.
#pragma unroll
    for (int q = 0; q < LQ; q++) {
      const int at = lane + 64 * q;
      if (at >= DP / 4) break;
      uint32_t w[4], o[VQ];
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = mine[k * DP / 4 + at];
      if (FMT == MG_KV_INT4) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          uint32_t bits = 0;
#pragma unroll
          for (int k = 0; k < 4; k++)
            bits |= (w[k] >> 8 * e & 15u) << 4 * v4_nibble(k, 0) |
                    (w[k] >> 8 * (e + 1) & 15u) << 4 * v4_nibble(k, 1);
          o[e / 2] = bits;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          o[e % VQ] = (w[0] >> 8 * e & 255u) | (w[1] >> 8 * e & 255u) << 8 |
                      (w[2] >> 8 * e & 255u) << 16 | (w[3] >> 8 * e & 255u) << 24;
      }
#pragma unroll
      for (int k = 0; k < VQ; k++) vw[at * VQ + k] = (o[k] & ~keep) | (old[q][k] & keep);
    }
  }
}

template <int FMT, int NB, bool VEC>
__global__ __launch_bounds__(256) void k_read(const KvRows a) {
  constexpr int DP = 16 * NB, RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;
  const int lane = threadIdx.x & 63, t = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = blockIdx.y * 4 + wave;
  Block g;
  if (!block_of<kRead>(a, &g) || h >= a.c.kv_heads) return;
  const int page = 1 << a.c.plog;
  const bool bad = g.page < 0;
  const int64_t ph = (bad ? 0 : g.page) * a.c.kv_heads + h;
#pragma unroll 2
  for (int u = g.first; u < g.last; u++) {
    const int slot = g.slot + 4 * u;
    const int i = g.pos + 4 * u + t - g.q.past;
    if (i < 0 || i >= g.q.n) continue;
    const float *sc = a.c.sc + ph * kv_scales(FMT) * page + slot + t;
    const uint8_t *kc = a.c.k + (ph * page + slot + t) * RB;
    const uint32_t *vw = reinterpret_cast<const uint32_t *>(a.c.v + (ph * page + slot) * RB);
    const float nan = __builtin_nanf("");
    const float ks = bad ? nan : sc[0], km = FMT == MG_KV_INT4 ? sc[2 * page] : 0.f;
    const float vs = bad ? nan : sc[page], vm = FMT == MG_KV_INT4 ? sc[3 * page] : 0.f;
    const int64_t row = g.q.start + i;
    float *ko = a.ko + row * a.ks + (int64_t)h * a.c.d;
    float *vo = a.vo + row * a.vs + (int64_t)h * a.c.d;
#pragma unroll
    for (int e = 0; e < NB; e += 4) {
      const int d = read_dim(e, c);
      uint32_t kw, cv[4];
      float x[4], y[4];
      if (FMT == MG_KV_INT4) {
        kw = *reinterpret_cast<const uint16_t *>(kc + d / 2);
        const uint2 w = *reinterpret_cast<const uint2 *>(vw + d / 2);
        cv[0] = w.x >> 4 * v4_nibble(t, 0) & 15u, cv[1] = w.x >> 4 * v4_nibble(t, 1) & 15u;
        cv[2] = w.y >> 4 * v4_nibble(t, 0) & 15u, cv[3] = w.y >> 4 * v4_nibble(t, 1) & 15u;
      } else {
        kw = *reinterpret_cast<const uint32_t *>(kc + d);
        const uint4 w = *reinterpret_cast<const uint4 *>(vw + d);
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
        if (d < a.c.d) {
          *reinterpret_cast<float4 *>(ko + d) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4 *>(vo + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (d + j < a.c.d) {
            ko[d + j] = x[j];
            vo[d + j] = y[j];
          }
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
  // Aligned blocks that a sequence of max_new rows can touch.
  const int span = read ? kRead : kWrite;
  const int64_t blocks = (a.s.max_new + span - 2) / span + 1;
  const int heads = 4 * (read ? 1 : a.hpw);
  const dim3 grid((unsigned)blocks, (unsigned)((a.c.kv_heads + heads - 1) / heads), (unsigned)a.s.batch);
  if (read)
    k_read<FMT, NB, VEC><<<grid, dim3(256), 0, ctx->stream>>>(a);
  else if (a.rope.half_rot)
    k_append<FMT, NB, VEC, true><<<grid, dim3(256), 0, ctx->stream>>>(a);
  else
    k_append<FMT, NB, VEC, false><<<grid, dim3(256), 0, ctx->stream>>>(a);
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
  KvRows a{c, s, k, v, nullptr, nullptr, ks, vs, rope ? *rope : mg_rope{}, 1};
  // Two heads a wave share its chain of lengths, page and tables (10k tokens of 8 heads of 128,
  // rotated: 40 -> 36 us) once there are waves enough (one token of 64 sequences: 5.7 -> 8.1 us)
  // and registers (heads of 256: 43 -> 50 us).
  if (c.dp <= 128 && s.batch * ((s.max_new + 6) / 4) * c.kv_heads > 16 * ctx->num_cus) a.hpw = 2;
  return run(ctx, a, false);
}

mg_status mg_kv_read_run(mg_ctx *ctx, const mg_kv_cache &c, const mg_seq_batch &s, float *k,
                         int64_t ks, float *v, int64_t vs) {
  KvRows a{c, s, nullptr, nullptr, k, v, ks, vs, mg_rope{}, 1};
  return run(ctx, a, true);
}
