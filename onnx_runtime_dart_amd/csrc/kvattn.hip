// Attention of single tokens, prompt chunks and drafted trees over the quantised KV cache.
//
// y = sum_t 2^(s_t - m) V_t / sum_t 2^(s_t - m), s_t = scale log2(e) q . K_t, in one pass
// over the keys with a running m.  A wave takes 16 QB rows (a row: one query and one query
// head of the KV head's group, so a group's heads share each key) and tiles of 32 keys:
//   S^T (16 keys x 16 rows, twice) = K . Q^T on v_mfma_f32_16x16x32_f16: lane (g, c) = (l /
//     16, l % 16) supplies key c (A) and row c (B) at the dims [g DP / 4, (g + 1) DP / 4),
//     a contiguous run of the key, 8 a step; the result gives it keys 4 g .. 4 g + 3 of row c.
//   O^T (16 dims x 16 rows) += V^T . P^T over 32 keys: the lane's eight weights are, as
//     they are, the B operand of keys {4 g + r, 16 + 4 g + r}; the A operand of row c of tile
//     i is dim NB c + i (NB = DP / 16) at those keys, and the cache keeps the four keys of a
//     dim in one dword, NB of them in a row: no transposition, no exchange between lanes.
// Codes are exact in fp16.  q is a pair of fp16 digits (22 bits) under a power of two, and so is
// a weight times its key's V scale; the products are exact and summed in fp32.  One digit would
// round scores and weights to 2^-11, which fp32 callers see; the second doubles the products,
// which single tokens have room for under the cached bytes and prompts pay for.
// Digits end at 2^-25, so their unit is that of a row's weights times scales, not of its largest weight
// and its largest scale, which may belong to different keys: 2^(s - m) is kept relative to a
// reference m of the row, a whole number that puts the sum of these products over a tile at 2^9 (scales
// in units of the largest, 2^12; an outlier among them moves m down).  What a key contributes is
// then off by 2^-22 of itself and 2^-33 of what its wave sums, however far its weight and its scale
// lie from the others'.  m moves up only when a product outgrows fp16, so most tiles rescale nothing
// and exchange nothing between lanes.  (With sums at 2^11, 2 x 2048 rows of heads of 64 meet that
// often enough to take 1% longer; with the largest product at 2^12, 10%.)
//
// Few rows (k_kv_keys): four waves take tiles in turn for the same 16 rows, the next tile's loads
// in flight under this one's products; long ones are bound by the cached bytes (one token of 64
// sequences of 2000 to 8000 keys, 8 heads of 128, e4m3: 134 us, 4.9 TB/s; one of 131072 keys,
// int8: 59 us; int4 by its conversions, 153 us for 64 sequences where e4m3 takes 144), short ones by
// a chain of latencies (about 5 us to the first weights, 4 for the join of key splits).  Many
// rows (k_kv_rows): bound by the two-digit products and by the exponentials and digits between
// them (2048 rows over 6000 keys, 32 heads of 128, int8: 468 us, three such chunks 532 TFLOP/s of
// the product's, 1064 with both digits, near what a large fp16 product of the library reaches on
// this card; heads of 64: 334 us and 426 TFLOP/s, where the exponentials weigh twice as much).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "kv_common.h"
#include "rope_common.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -3.0e38f;  // the reference before any score
constexpr float kTop = 65000.f;     // most of a weight times its scale (fp16 ends at 65504)
constexpr int kAim = 9;             // log2 of where a tile's sum of them is put
constexpr int kRoom = 84;           // log2 of a weight so put, at most (their sums have room above)
constexpr float kScales = 4096.f;   // the largest V scale lies in [2^11, 2^12) of their unit

// Four codes of one dword of K (adjacent dims) or V (four keys of a dim) as fp16.
template <int FMT>
__device__ inline void four(uint32_t w, half2v &a, half2v &b) {
  if (FMT == MG_KV_INT8) {
    // 0x6400 | byte is 1024 + byte.
    a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
    b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
    const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
    a -= off;
    b -= off;
  } else {
    a = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    b = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
  }
}
// Nibbles i and i + 4 of a dword as 2 n - 15: 0x6400 | 2 n is 1024 + 2 n.
__device__ inline half2v nib2(uint32_t w, int i) {
  const uint32_t x = i == 0 ? w << 1 : w >> (4 * i - 1);
  const half2v off = {(_Float16)1039.f, (_Float16)1039.f};
  return __builtin_bit_cast(half2v, (x & 0x001e001eu) | 0x64006400u) - off;
}
__device__ inline half2v nib2_any(uint32_t w, int i) {
  const uint32_t x = (uint32_t)(((uint64_t)w << 1) >> (4 * i));
  const half2v off = {(_Float16)1039.f, (_Float16)1039.f};
  return __builtin_bit_cast(half2v, (x & 0x001e001eu) | 0x64006400u) - off;
}
__device__ inline half8v join4(half2v a, half2v b, half2v c, half2v d) {
  half8v r;
  r[0] = a[0];
  r[1] = a[1];
  r[2] = b[0];
  r[3] = b[1];
  r[4] = c[0];
  r[5] = c[1];
  r[6] = d[0];
  r[7] = d[1];
  return r;
}
// The A operand of step s from the lane's run of a key's codes.
template <int FMT, int KW>
__device__ inline half8v k_operand(const uint32_t (&w)[KW], int s) {
  half2v a, b, c, d;
  if (FMT == MG_KV_INT4) {
    a = nib2(w[s], 0), b = nib2(w[s], 1), c = nib2(w[s], 2), d = nib2(w[s], 3);
  } else {
    four<FMT>(w[2 * s], a, b);
    four<FMT>(w[2 * s + 1], c, d);
  }
  return join4(a, b, c, d);
}
// Dim of slot j (of 8) of a step, as k_operand lays the codes out.
template <int FMT>
__device__ constexpr int k_slot(int j) {
  return FMT == MG_KV_INT4 ? (j >> 1) + 4 * (j & 1) : j;
}
// The A operand of dim tile i: four keys of each half tile.
template <int FMT, int KW>
__device__ inline half8v v_operand(const uint32_t (&w0)[KW], const uint32_t (&w1)[KW], int i) {
  half2v a, b, c, d;
  if (FMT == MG_KV_INT4) {
    const int n = 2 * (i & 1);
    a = nib2(w0[i / 2], n), b = nib2(w0[i / 2], n + 1);
    c = nib2(w1[i / 2], n), d = nib2(w1[i / 2], n + 1);
  } else {
    four<FMT>(w0[i], a, b);
    four<FMT>(w1[i], c, d);
  }
  return join4(a, b, c, d);
}

// KW dwords from p (16 bytes a load where they come in fours).
template <int KW>
__device__ inline void load_run(uint32_t (&w)[KW], const uint8_t *p) {
  if (KW % 4 == 0) {
#pragma unroll
    for (int i = 0; i < KW / 4; i++) {
      const uint4 x = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < KW / 2; i++) {
      const uint2 x = reinterpret_cast<const uint2 *>(p)[i];
      w[2 * i] = x.x;
      w[2 * i + 1] = x.y;
    }
  }
}

// Max and sum over the four lanes that hold one row.
__device__ inline float row_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float row_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
__device__ inline float wave_max(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
// 2^-e with |x| in [2^(e-1), 2^e), 2^102 at most; 1 for 0.
__device__ inline float pow2_under(float x) {
  const int e = (int)(__float_as_uint(x) >> 23 & 255u);
  return x == 0.f ? 1.f : ldexpf(1.f, 126 - max(e, 24));
}
// floor(log2 x) of a normal x >= 0; -127 below.
__device__ inline int log2_of(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }
// The second digit of x after the first.  (One mixed fma, exact before its rounding; a -1 that
// the compiler knows is turned into a conversion and a difference.)
__device__ inline _Float16 rest_of(float x, _Float16 hi) {
  float minus = -1.f;
  asm("" : "+s"(minus));
  return (_Float16)fmaf((float)hi, minus, x);
}
__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

template <int FMT, int NB>
struct Shape {
  static constexpr int DP = 16 * NB, KS = DP / 32;
  static constexpr int KW = FMT == MG_KV_INT4 ? DP / 32 : DP / 16;  // dwords of a lane's run, 16 keys
  static constexpr int RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;   // bytes of a vector
};

// Where the two runs of 16 keys of a tile lie: the same for a whole wave, so in scalar registers
// (the lanes add 32-bit offsets).
struct Place {
  int page[2];    // table entries of the tile looked up last, not yet checked; -1: none
  int64_t at[2];  // of the located one: (page, head) times page size plus place
  int64_t sc[2];  // and its scales, in floats
  bool none[2];   // no such page: its keys read as NaN

  // (The entries are first used a tile later, in locate.)
  __device__ inline void look_up(const mg_kv_attn &a, int b, int total, int t0) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int t = t0 + 16 * u;
      const int64_t entry = t >> a.c.plog;
      page[u] = -1;
      if (t >= total) page[u] = 0;
      else if (entry < a.s.table_stride) page[u] = kv_scalar(a.s.page_table + b * a.s.table_stride + entry);
    }
  }
  template <int FMT>
  __device__ inline void locate(const mg_kv_attn &a, int h, int t0) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      none[u] = page[u] < 0 || page[u] >= a.c.pages;
      const int64_t ph = (int64_t)(none[u] ? 0 : page[u]) * a.c.kv_heads + h;
      const int slot = (t0 + 16 * u) & ((1 << a.c.plog) - 1);
      at[u] = (ph << a.c.plog) + slot;
      sc[u] = (ph * kv_scales(FMT) << a.c.plog) + slot;
    }
  }
};

// A tile of 32 keys in a wave's registers: codes and scales.  The parts are loaded apart.
template <int FMT, int NB>
struct Tile {
  using S = Shape<FMT, NB>;
  uint32_t k[2][S::KW], v[2][S::KW];
  float4 ks[2], vs[2], kz[2], vz[2];

  __device__ inline void load_k(const mg_kv_attn &a, const Place &p, int g, int c) {
#pragma unroll
    for (int u = 0; u < 2; u++)
      load_run<S::KW>(k[u], a.c.k + p.at[u] * S::RB + (uint32_t)(c * S::RB + g * (S::RB / 4)));
  }
  __device__ inline void load_v(const mg_kv_attn &a, const Place &p, int g, int c) {
#pragma unroll
    for (int u = 0; u < 2; u++)
      load_run<S::KW>(v[u], a.c.v + p.at[u] * S::RB + (uint32_t)(4 * g * S::RB + c * (4 * S::KW)));
  }
  __device__ inline void load_scales(const mg_kv_attn &a, const Place &p, int g) {
    const uint32_t psize = 1u << a.c.plog;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const float *sc = a.c.sc + p.sc[u];
      ks[u] = *reinterpret_cast<const float4 *>(sc + (uint32_t)(4 * g));
      vs[u] = *reinterpret_cast<const float4 *>(sc + (psize + 4 * g));
      if (FMT == MG_KV_INT4) {
        kz[u] = *reinterpret_cast<const float4 *>(sc + (2 * psize + 4 * g));
        vz[u] = *reinterpret_cast<const float4 *>(sc + (3 * psize + 4 * g));
      }
      if (p.none[u]) {
        const float nan = __builtin_nanf("");
        ks[u] = make_float4(nan, nan, nan, nan);
      }
    }
  }
};

__device__ inline void spread(float (&x)[8], const float4 (&v)[2], float f) {
#pragma unroll
  for (int u = 0; u < 2; u++) {
    x[4 * u] = v[u].x * f;
    x[4 * u + 1] = v[u].y * f;
    x[4 * u + 2] = v[u].z * f;
    x[4 * u + 3] = v[u].w * f;
  }
}

// The workgroup's queries, turned and scaled, in shared memory: `n` rows from row r0 of
// sequence sq; rows past the last are zero.
template <int DP>
__device__ inline void stage_queries(const mg_kv_attn &a, const kv_seq &sq, int h, int r0, int rows,
                                     int n, float *lds) {
  constexpr int QP = DP + 4;
  const int half = (int)a.rope.half_rot;
  if (a.vec) {
    // Units of eight elements: four pairs of halves, or eight adjacent ones.
    constexpr int UNITS = DP / 8;
    const int turned = a.rope.interleaved ? half / 4 : 0;  // units of pairs side by side
    const int halves = a.rope.interleaved ? 0 : half / 4;
    for (int i = threadIdx.x; i < n * UNITS; i += 256) {
      const int r = i / UNITS, u = i - r * UNITS, row = r0 + r;
      const int d0 = u < halves ? 4 * u : halves ? 2 * half + 8 * (u - halves) : 8 * u;
      const int d1 = u < halves ? d0 + half : d0 + 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), z = x;
      if (row < rows && d0 < a.c.d) {
        const int qi = row / a.group, j = row - qi * a.group;
        const int64_t at = sq.start + qi;
        const float *q = a.q + at * a.q_stride + (int64_t)(h * a.group + j) * a.c.d;
        x = *reinterpret_cast<const float4 *>(q + d0);
        if (d1 < a.c.d) z = *reinterpret_cast<const float4 *>(q + d1);
        if (u < halves + turned) {
          const int64_t pos = a.rope.positions ? a.rope.positions[at] : sq.past + qi;
          const bool in = (uint64_t)pos < (uint64_t)a.rope.max_pos;
          const int64_t t = (in ? pos : 0) * half + 4 * u;
          const float4 cs = *reinterpret_cast<const float4 *>(a.rope.cos_table + t);
          const float4 sn = *reinterpret_cast<const float4 *>(a.rope.sin_table + t);
          auto pair = [&](float &p, float &w, float co, float si) {
            const double c = in ? (double)co : __builtin_nan(""), s = si, pd = p, wd = w;
            p = (float)(pd * c - wd * s);
            w = (float)(wd * c + pd * s);
          };
          if (halves) {
            pair(x.x, z.x, cs.x, sn.x);
            pair(x.y, z.y, cs.y, sn.y);
            pair(x.z, z.z, cs.z, sn.z);
            pair(x.w, z.w, cs.w, sn.w);
          } else {
            pair(x.x, x.y, cs.x, sn.x);
            pair(x.z, x.w, cs.y, sn.y);
            pair(z.x, z.y, cs.z, sn.z);
            pair(z.z, z.w, cs.w, sn.w);
          }
        }
      }
      const float f = a.scale2;
      *reinterpret_cast<float4 *>(lds + r * QP + d0) = make_float4(f * x.x, f * x.y, f * x.z, f * x.w);
      *reinterpret_cast<float4 *>(lds + r * QP + d1) = make_float4(f * z.x, f * z.y, f * z.z, f * z.w);
    }
    return;
  }
  for (int i = threadIdx.x; i < n * DP; i += 256) {
    const int r = i / DP, d = i - r * DP, row = r0 + r;
    float x = 0.f;
    if (row < rows && d < a.c.d) {
      const int qi = row / a.group, j = row - qi * a.group;
      const int64_t at = sq.start + qi;
      const int64_t pos = half && a.rope.positions ? a.rope.positions[at] : sq.past + qi;
      x = a.scale2 *
          rope_at(a.q + at * a.q_stride + (int64_t)(h * a.group + j) * a.c.d, d, pos, a.rope);
    }
    lds[r * QP + d] = x;
  }
}

// One tile's weights for QB blocks of 16 rows: 2^(s - m) of the lane's eight keys, and the digits of
// those times the V scales vsn.  l and z are the lane's share of the sum and (INT4) of the sum of
// weights times middles.  masked: only the keys of `seen` count (a branch of the whole wave, or a
// constant), and with UNITS V scales and middles want the factors unit[256 q] of the rows yet.  own: some
// row's products do so with units[256 q].  limit: kTop (over the largest such factor); negative with own,
// and with coarse, which is set for good where scores are too large for the reference to follow.
template <int FMT, int NB, int QB, bool UNITS>
__device__ inline void weigh(bool masked, const float *unit, bool own, const float *units,
                             bool &coarse, float limit, float4v (&acc)[QB][2], const float (&ksf)[8],
                             const float (&vsn)[8], const float (&kzf)[8], const float (&vz)[8],
                             const float (&qs)[QB], const uint32_t (&seen)[QB], float (&m)[QB],
                             float (&l)[QB], float (&z)[QB], float4v (&o)[QB][NB],
                             half8v (&ph)[QB], half8v (&pl)[QB]) {
  float d[QB][8];  // scores less m, of unseen keys too
  auto scores = [&](int q) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float base = FMT == MG_KV_INT4 ? fmaf(qs[q], kzf[j], -m[q]) : -m[q];
      d[q][j] = fmaf(acc[q][j >> 2][j & 3], ksf[j], base);
    }
  };
  auto top = [&](int q) __attribute__((always_inline)) {
    return fmaxf(fmaxf(fmaxf(d[q][0], d[q][1]), fmaxf(d[q][2], d[q][3])),
                 fmaxf(fmaxf(d[q][4], d[q][5]), fmaxf(d[q][6], d[q][7])));
  };
#pragma unroll
  for (int q = 0; q < QB; q++) scores(q);
  float most = top(0);
#pragma unroll
  for (int q = 1; q < QB; q++) most = fmaxf(most, top(q));
  // A bound of the lane's products, and of its weights alone by 2^90.
  float big = 0x1p-74f;
#pragma unroll
  for (int j = 0; j < 8; j++) big = fmaxf(big, vsn[j]);
  // (An unseen key may bring a wave here, where only the seen ones count; and a negative limit does, where
  // products want factors yet.  No branch of their own takes those there: where paths of
  // different length meet behind a matrix product, the compiler (ROCm 7.2) has left out the wait
  // for its result.)
  if (__builtin_expect(__any(exp2_of(most) * big > limit), 0)) {
#pragma unroll
    for (int q = 0; q < QB; q++) {
      const float old = m[q];
      if (own) {
        acc[q][0] *= units[256 * q];
        acc[q][1] *= units[256 * q];
      }
      m[q] = 0.f;
      scores(q);
#pragma unroll
      for (int j = 0; j < 8; j++) d[q][j] = seen[q] >> j & 1 ? d[q][j] : -__builtin_inff();
      const float best = row_max(top(q)), u = UNITS && masked ? unit[256 * q] : 1.f;
      float p = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float x = exp2_of(d[q][j] - best) * vsn[j] * u;
        p += x > 0.f ? x : 0.f;
      }
      // (Whole numbers: outputs and sums are moved without rounding.)
      const float aim = rintf(best + (float)max(log2_of(row_sum(p)) - kAim, -kRoom));
      m[q] = aim > old + 2.f ? aim : old;
      // Scores beyond 2^22 go by their fp32 values, the reference is the largest: differences that are
      // not rounded would tell apart what is equal, and miss the reference.
      const bool far = fabsf(best) > 0x1p22f && best > -__builtin_inff();
      coarse |= __any(far);
      if (far) m[q] = fmaxf(old, best);
      const float by = ldexpf(1.f, (int)fmaxf(old - m[q], -200.f));
      l[q] *= by;
      z[q] *= by;
#pragma unroll
      for (int i = 0; i < NB; i++) o[q][i] *= by;
      if (coarse) {
#pragma unroll
        for (int j = 0; j < 8; j++) d[q][j] -= m[q];
      } else {
        scores(q);
      }
    }
  }
  float e[QB][8], w[QB][8];
#pragma unroll
  for (int q = 0; q < QB; q++)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      e[q][j] = exp2_of(d[q][j]);
      w[q][j] = e[q][j] * vsn[j];
    }
  if (masked) {
    // An unseen key counts nothing, whatever its score and scales are.  (The empty statement
    // keeps the selections in their branch; else every tile does them.)
    asm volatile("");
#pragma unroll
    for (int q = 0; q < QB; q++) {
      const float u = UNITS ? unit[256 * q] : 1.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const bool on = seen[q] >> j & 1;
        e[q][j] = on ? e[q][j] : 0.f;
        w[q][j] = on ? w[q][j] * u : 0.f;
        if (FMT == MG_KV_INT4) z[q] += on ? e[q][j] * (vz[j] * u) : 0.f;
      }
    }
  } else if (FMT == MG_KV_INT4) {
#pragma unroll
    for (int q = 0; q < QB; q++)
#pragma unroll
      for (int j = 0; j < 8; j++) z[q] = fmaf(e[q][j], vz[j], z[q]);
  }
#pragma unroll
  for (int q = 0; q < QB; q++)
#pragma unroll
    for (int j = 0; j < 8; j++) l[q] += e[q][j];
#pragma unroll
  for (int q = 0; q < QB; q++)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const half2v hi = __builtin_convertvector(float2v{w[q][j], w[q][j + 1]}, half2v);
      ph[q][j] = hi[0];
      ph[q][j + 1] = hi[1];
      pl[q][j] = rest_of(w[q][j], hi[0]);
      pl[q][j + 1] = rest_of(w[q][j + 1], hi[1]);
    }
}

// The unit of the row's V scales shrinks to 2^-j of itself: so does what is yet to come, and the
// reference follows it down, which leaves the outputs as they are.  As far as the sum of the
// weights has room; they shrink by the rest.
template <int NB>
__device__ inline void smaller_unit(int j, float &m, float &l, float &z, float4v (&o)[NB]) {
  // (A reference of 2^24 and more does not move by small steps.)
  const int keep = fabsf(m) < 0x1p24f ? max(0, min(j, kRoom - log2_of(row_max(l)))) : 0;
  m -= (float)keep;
  l = ldexpf(l, keep);
  const float by = ldexpf(1.f, keep - j);
  z *= by;
#pragma unroll
  for (int i = 0; i < NB; i++) o[i] *= by;
}

// Which of the lane's eight keys of the tile at t0 a row sees (bit j: key 16 (j / 4) + 4 g + j % 4),
// of those below kfin.
__device__ inline uint32_t seen_keys(const mg_kv_attn &a, const kv_seq &sq, int t0, int g, int see,
                                     int64_t word, int kfin) {
  uint32_t seen = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int k = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
    bool ok = k < see;
    if (a.tree && k >= sq.past && k < sq.past + sq.n)
      ok = a.tree[word + ((k - sq.past) >> 6)] >> ((k - sq.past) & 63) & 1;
    if (ok && k < kfin) seen |= 1u << j;
  }
  return seen;
}

// Largest finite size among n elements.
__device__ inline float largest(const float *x, int n, float mx) {
#pragma unroll
  for (int d = 0; d < n; d++) {
    const float v = fabsf(x[d]);
    mx = v < __builtin_inff() ? fmaxf(mx, v) : mx;
  }
  return mx;
}

// The digits of 16 rows' queries in matrix order from shared memory (x: the lane's run), times a
// power of two: a row's largest element comes under 2^15, so that a digit pair is exact to 2^-22 of
// any element down to 2^-17 of the largest, and to 2^-39 of the largest below.  Rows share the
// power dn of the largest of them all, max; one 2^12 below has its own, and `own` gives its scores
// the units of the others (1 for those): a row does not see how large another is.
// row: the row's largest.
template <int FMT, int KS>
__device__ inline void query_digits(const float *x, float row, float max, float dn, half8v (&qh)[KS],
                                    half8v (&ql)[KS], float &qs, float &own) {
  const bool apart = row != 0.f && row < 0x1p-12f * max;
  const float mine = apart ? 32768.f * pow2_under(row) : dn;
  own = apart ? dn / mine : 1.f;
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < KS; s++)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float v = x[8 * s + k_slot<FMT>(j)] * mine;
      const _Float16 hi = (_Float16)v;
      qh[s][j] = hi;
      ql[s][j] = rest_of(v, hi);
      sum += v;
    }
  qs = FMT == MG_KV_INT4 ? row_sum(sum) * own : 0.f;
}

// Keys to pass over for rows up to `last`: those that it sees, but where every row that sees a key
// past the page table sees the first there, no more than one tile beyond it: that key reads as NaN
// like all after it.  (Drafts see one another by their tree alone: where the past ends within the table
// they are all passed over.)
__device__ inline int keys_of(const mg_kv_attn &a, const kv_seq &sq, int last) {
  const int end = a.tree ? sq.past + sq.n : sq.past + last / a.group + 1;
  if (a.s.table_stride > end >> a.c.plog) return end;
  const int64_t held = a.s.table_stride << a.c.plog;
  if (a.tree && sq.past <= held) return end;
  return (int)min((int64_t)end, held + 32);
}

// Keys of a split of the sequence: its own are shared out, so that a bound far above its length
// costs no more than idle workgroups (one token over 2000 keys, bound 131072: 27 us by the
// bound's share, 12 so).
__device__ inline int split_keys(const mg_kv_attn &a, const kv_seq &sq) {
  if (a.nsplit == 1) return 0x7fffff80;
  const uint32_t all = (uint32_t)keys_of(a, sq, sq.n * a.group - 1);
  // (A division on the way to the first loads: by the reciprocal, up to 192 keys short of 2^31.)
  uint32_t kc = max(128u, ((uint32_t)((float)all * a.share) + 127) & ~127u);
  if ((uint64_t)kc * a.nsplit < all) kc += 128;
  if ((uint64_t)kc * a.nsplit < all) kc += 128;
  return (int)kc;
}

// Which sequence, split, row block and KV head a workgroup has (heads innermost), and its keys.
struct Work {
  kv_seq sq;
  int b, h, split, r0, rows;  // rows: of the sequence
  int kbeg, kend, kfin;       // keys that its last row sees, from its split's first on; its split's
};
// False: nothing to do.
__device__ inline bool work_of(const mg_kv_attn &a, int ROWS, Work *w) {
  int id = (int)blockIdx.x;
  w->h = id % a.c.kv_heads;
  id /= a.c.kv_heads;
  const int blk = a.nblk - 1 - id % a.nblk;  // rows that see most keys first
  id /= a.nblk;
  w->split = id % a.nsplit;
  w->b = id / a.nsplit;
  w->sq = kv_sequence(a.s, w->b);
  if (w->sq.bad) {
    if (blk == 0 && w->split == 0 && w->h == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
    return false;
  }
  w->rows = w->sq.n * a.group;
  w->r0 = blk * ROWS;
  if (w->r0 >= w->rows) return false;
  w->kend = keys_of(a, w->sq, min(w->r0 + ROWS, w->rows) - 1);
  // (A split past the last may begin beyond 32 bits.)
  const int kc = split_keys(a, w->sq);
  const int64_t kbeg = (int64_t)w->split * kc;
  if (kbeg >= w->kend && w->split > 0) return false;
  w->kbeg = (int)kbeg;
  w->kfin = (int)min((int64_t)w->kend, kbeg + kc);
  return true;
}

// Four outputs of row w.r0 + r from dim d, to y or to the split's partial results.
template <int DP>
__device__ inline void put4(const mg_kv_attn &a, const Work &w, int r, int d, float4 v) {
  const int row = w.r0 + r;
  if (row >= w.rows) return;
  if (a.nsplit > 1) {
    const int64_t at = ((int64_t)w.b * a.c.kv_heads + w.h) * a.s.max_new * a.group + row;
    *reinterpret_cast<float4 *>(a.part + (at * a.nsplit + w.split) * DP + d) = v;
    return;
  }
  const int qi = row / a.group, j = row - qi * a.group;
  float *y = a.y + (w.sq.start + qi) * a.y_stride + (int64_t)(w.h * a.group + j) * a.c.d + d;
  if (a.vec) {
    if (d < a.c.d) *reinterpret_cast<float4 *>(y) = v;
  } else {
    if (d < a.c.d) y[0] = v.x;
    if (d + 1 < a.c.d) y[1] = v.y;
    if (d + 2 < a.c.d) y[2] = v.z;
    if (d + 3 < a.c.d) y[3] = v.w;
  }
}
// A part of a row's keys where it is joined with the others: the reference under which the sum l of
// its weights (kept under m) is below 1/4, so that a workgroup's four parts of the largest values have
// a finite sum; and l under a reference that may be higher.
__device__ inline float part_ref(float m, float l) {
  return l == 0.f ? kNoMax : m + (float)(log2_of(l) + 3);
}
__device__ inline float part_sum(float m, float l, float ref) {
  return ldexpf(l, (int)fminf(fmaxf(m - ref, -400.f), 400.f));
}
__device__ inline void put_stat(const mg_kv_attn &a, const Work &w, int r, float m, float l) {
  if (a.nsplit == 1 || w.r0 + r >= w.rows) return;
  const int64_t at = ((int64_t)w.b * a.c.kv_heads + w.h) * a.s.max_new * a.group + w.r0 + r;
  a.part_ml[at * a.nsplit + w.split] = make_float2(m, l);
}

// Few rows: the four waves take tiles in turn for the same 16 rows and join their results.
template <int FMT, int NB>
__global__ __launch_bounds__(256, NB <= 8 ? 2 : 1) void k_kv_keys(const mg_kv_attn a) {
  using S = Shape<FMT, NB>;
  constexpr int DP = S::DP, KS = S::KS, KW = S::KW, QP = DP + 4, STEP = 128;
  // 16 rows' queries; later the four waves' results.
  __shared__ __attribute__((aligned(16))) float lds[64 * QP];
  __shared__ float stat[4][2][16];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  Work w;
  if (!work_of(a, 16, &w)) return;
  const kv_seq &sq = w.sq;
  const int total = sq.past + sq.n;
  const int kfin = w.kfin;
  // Keys below it are seen by every row.
  const int plain = a.tree ? sq.past : sq.past + w.r0 / a.group + 1;
  int t0 = w.kbeg + 32 * wave;
  // The first tile's loads run while the queries are made.
  Tile<FMT, NB> t, next;
  Place p;
  bool refused = false;
  if (t0 < kfin) {
    p.look_up(a, w.b, total, t0);
    p.locate<FMT>(a, w.h, t0);
    t.load_k(a, p, g, c);
    t.load_scales(a, p, g);
    t.load_v(a, p, g, c);
    refused = p.none[0] || p.none[1];
    p.look_up(a, w.b, total, t0 + STEP);
  }
  stage_queries<DP>(a, sq, w.h, w.r0, w.rows, 16, lds);
  __syncthreads();
  const float *x = lds + c * QP + g * (DP / 4);
  const float row = row_max(largest(x, DP / 4, 0.f)), mx = wave_max(row);
  const float dn = 32768.f * pow2_under(mx), f = 1.f / dn;
  half8v qh[KS], ql[KS];
  float qs[1], own;
  query_digits<FMT, KS>(x, row, mx, dn, qh, ql, qs[0], own);
  const float fo = f * own;
  const int qi = min(w.r0 + c, w.rows - 1) / a.group;
  const int see = a.tree ? sq.past : sq.past + qi + 1;
  const int64_t word = (int64_t)(sq.start + qi) * a.tree_words;

  float4v o[1][NB];
#pragma unroll
  for (int i = 0; i < NB; i++) o[0][i] = float4v{0.f, 0.f, 0.f, 0.f};
  float m[1] = {kNoMax}, l[1] = {0.f}, z[1] = {0.f}, vn = ldexpf(1.f, 100);
  bool coarse = false;
  // With registers to spare the next tile's loads start before this one's products, else each
  // part's as soon as this one's is used.
  constexpr bool AHEAD = NB <= 8;
  // One tile; MASKED: some row may not see some key.
  auto tile = [&](auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const int tn = t0 + STEP;
    const bool more = tn < kfin;
    if (more) {
      p.locate<FMT>(a, w.h, tn);
      p.look_up(a, w.b, total, tn + STEP);
      refused |= p.none[0] || p.none[1];
    }
    if (AHEAD && more) {
      next.load_k(a, p, g, c);
      next.load_scales(a, p, g);
      next.load_v(a, p, g, c);
    }
    float4v acc[1][2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      acc[0][u] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const half8v ka = k_operand<FMT, KW>(t.k[u], s);
        acc[0][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[s], acc[0][u], 0, 0, 0);
        acc[0][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[s], acc[0][u], 0, 0, 0);
      }
    }
    if (!AHEAD && more) next.load_k(a, p, g, c);
    float ksf[8], vsn[8], kzf[8], vz[8];
    spread(ksf, t.ks, fo);
    spread(vsn, t.vs, 1.f);
    if (FMT == MG_KV_INT4) {
      spread(kzf, t.kz, f);
      spread(vz, t.vz, 1.f);
    }
    const uint32_t seen[1] = {MASKED ? seen_keys(a, sq, t0, g, see, word, kfin) : 0xffu};
    // V scales (INT4: and middles) relative to the largest that the row has seen.
    float big = 0.f, mid = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (MASKED) vsn[j] = seen[0] >> j & 1 ? vsn[j] : 0.f;
      if (MASKED && FMT == MG_KV_INT4) vz[j] = seen[0] >> j & 1 ? vz[j] : 0.f;
      big = fmaxf(big, vsn[j]);
      if (FMT == MG_KV_INT4) mid = fmaxf(mid, fabsf(vz[j]));
    }
    if (FMT == MG_KV_INT4) big = fmaxf(big, 0.0625f * mid);
    if (__builtin_expect(__any(big * vn > 2.f * kScales), 0)) {
      big = row_max(big);
      const float now = big * vn > 2.f * kScales ? kScales * pow2_under(big) : vn;
      smaller_unit<NB>(log2_of(vn) - log2_of(now), m[0], l[0], z[0], o[0]);
      vn = now;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      vsn[j] *= vn;
      if (FMT == MG_KV_INT4) vz[j] *= vn;
    }
    half8v ph[1], pl[1];
    weigh<FMT, NB, 1, false>(MASKED, nullptr, false, nullptr, coarse, coarse ? -1.f : kTop, acc, ksf,
                             vsn, kzf, vz, qs, seen, m, l, z, o, ph, pl);
    if (!AHEAD && more) next.load_scales(a, p, g);
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const half8v va = v_operand<FMT, KW>(t.v[0], t.v[1], i);
      o[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[0], o[0][i], 0, 0, 0);
      o[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[0], o[0][i], 0, 0, 0);
    }
    if (!AHEAD && more) next.load_v(a, p, g, c);
    t = next;
    t0 = tn;
  };
  while (t0 < kfin && t0 + 32 <= plain) tile(std::false_type{});
  while (t0 < kfin) tile(std::true_type{});

  if (refused && lane == 0) atomicOr(a.c.refused, 1);
  l[0] = row_sum(l[0]);
  z[0] = FMT == MG_KV_INT4 ? row_sum(z[0]) : 0.f;
  if (g == 0) stat[wave][0][c] = part_ref(m[0], l[0]);
  __syncthreads();
  const float all = fmaxf(fmaxf(stat[0][0][c], stat[1][0][c]), fmaxf(stat[2][0][c], stat[3][0][c]));
  const float sum = part_sum(m[0], l[0], all), inv = l[0] == 0.f ? 0.f : 1.f / l[0], by = sum / vn;
  if (g == 0) stat[wave][1][c] = sum;
#pragma unroll
  for (int e = 0; e < 4; e++)
#pragma unroll
    for (int i = 0; i < NB; i += 4)
      *reinterpret_cast<float4 *>(lds + (wave * 16 + c) * QP + NB * (4 * g + e) + i) =
          make_float4((o[0][i][e] + z[0]) * inv * by, (o[0][i + 1][e] + z[0]) * inv * by,
                      (o[0][i + 2][e] + z[0]) * inv * by, (o[0][i + 3][e] + z[0]) * inv * by);
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * DP / 4; i += 256) {
    const int r = i / (DP / 4), d = 4 * (i - r * (DP / 4));
    float mm = stat[0][0][r], ll = stat[0][1][r];
#pragma unroll
    for (int k = 1; k < 4; k++) {
      mm = fmaxf(mm, stat[k][0][r]);
      ll += stat[k][1][r];
    }
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float4 y = *reinterpret_cast<const float4 *>(lds + (k * 16 + r) * QP + d);
      v.x += y.x;
      v.y += y.y;
      v.z += y.z;
      v.w += y.w;
    }
    const float f1 = a.nsplit > 1 ? 1.f : ll == 0.f ? 0.f : 1.f / ll;
    put4<DP>(a, w, r, d, make_float4(v.x * f1, v.y * f1, v.z * f1, v.w * f1));
    if (d == 0) put_stat(a, w, r, mm, ll);
  }
}

// A wave's quarter of a tile's codes on their way to shared memory: a run of steps of one half
// tile's keys, a run of dim tiles of the values; and in one wave the tile's scales, a key a lane.
template <int FMT, int NB>
struct Quarter {
  using S = Shape<FMT, NB>;
  static constexpr int KF = S::KS / 2, VF = NB / 4;  // operands of K and of V that it makes
  static constexpr int KD = FMT == MG_KV_INT4 ? KF : 2 * KF;
  static constexpr int VD = FMT == MG_KV_INT4 ? (VF + 1) / 2 : VF;
  uint32_t k[KD], v[2][VD];
  float ks, vs, kz, vz;
  bool none;  // of the lane's key

  __device__ inline void load(const mg_kv_attn &a, const Place &p, int wave, int lane) {
    const int g = lane >> 4, c = lane & 15;
    const uint8_t *kp = a.c.k + (wave & 2 ? p.at[1] : p.at[0]) * S::RB + (wave & 1) * 4 * KD;
#pragma unroll
    for (int i = 0; i < KD; i++)
      k[i] = *reinterpret_cast<const uint32_t *>(kp + (uint32_t)(c * S::RB + g * (S::RB / 4) + 4 * i));
    const int i0 = wave * VF;  // its first dim tile
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint8_t *vp = a.c.v + p.at[u] * S::RB;
      const uint32_t o = 4 * g * S::RB + 4 * (FMT == MG_KV_INT4 ? (c * NB + i0) >> 1 : c * NB + i0);
#pragma unroll
      for (int i = 0; i < VD; i++) v[u][i] = *reinterpret_cast<const uint32_t *>(vp + (o + 4 * i));
    }
    if (wave == 3) {
      const uint32_t psize = 1u << a.c.plog;
      const bool u = lane >> 4 & 1;
      const float *sc = a.c.sc + (u ? p.sc[1] : p.sc[0]) + c;
      ks = sc[0];
      vs = sc[psize];
      if (FMT == MG_KV_INT4) {
        kz = sc[2 * psize];
        vz = sc[3 * psize];
      }
      none = u ? p.none[1] : p.none[0];
    }
  }
  // The operands, [operand][lane]: K by half tile and step, V by dim tile.
  __device__ inline void convert(uint4 *kt, uint4 *vt, int wave, int lane) const {
#pragma unroll
    for (int i = 0; i < KF; i++)
      kt[(wave * KF + i) * 64 + lane] = __builtin_bit_cast(uint4, k_operand<FMT, KD>(k, i));
#pragma unroll
    for (int i = 0; i < VF; i++) {
      half8v x;
      if (FMT == MG_KV_INT4) {
        // (Its first dim tile may be the second of a dword's pair.)
        const int odd = VF % 2 ? wave & 1 : 0, n = 2 * ((odd + i) & 1), w = (odd + i) >> 1;
        const uint32_t w0 = w ? v[0][VD - 1] : v[0][0], w1 = w ? v[1][VD - 1] : v[1][0];
        x = join4(nib2_any(w0, n), nib2_any(w0, n + 1), nib2_any(w1, n), nib2_any(w1, n + 1));
      } else {
        half2v p, q, r, s;
        four<FMT>(v[0][i % VD], p, q);
        four<FMT>(v[1][i % VD], r, s);
        x = join4(p, q, r, s);
      }
      vt[(wave * VF + i) * 64 + lane] = __builtin_bit_cast(uint4, x);
    }
  }
};

// Many rows: each of the four waves has 16 QB rows of its own.  They convert a quarter of each
// tile each, into shared memory in matrix order (twice, so that one barrier a tile suffices): a
// code is then converted once for 64 QB rows, not by every wave, and its 16-byte operands cost a
// quarter of what the products take.  (Each wave converting all of its tiles in registers: 2048
// rows over 6000 keys, D 128, int8 748 us, not 460; 1500 over 3000, D 256, 502, not 254.)  Pages
// are looked up a tile ahead by scalar loads, whose wait leaves the codes in flight (by vector
// loads 489, D 256 333).  The bounds are the waves a SIMD that the registers allow unspilled.  (128 rows
// of heads of 64 with two, not three: 8 x 2048 rows over 1000 keys 818 us, not 675; 2 x 2048 over 6000,
// which leave the card half empty, 580 and 582.)
template <int FMT, int NB, int QB>
__global__ __launch_bounds__(256, QB * NB <= (FMT == MG_KV_INT4 ? 4 : 8) ? 3 : 2)
void k_kv_rows(const mg_kv_attn a) {
  using S = Shape<FMT, NB>;
  constexpr int DP = S::DP, KS = S::KS, QP = DP + 4, ROWS = 64 * QB;
  constexpr int KO = 2 * KS * 64, VO = NB * 64;  // operands of a tile
  union Shared {
    float q[ROWS * QP];  // the queries, before the tiles
    struct {
      uint4 k[2][KO], v[2][VO];
    } t;
  };
  __shared__ __attribute__((aligned(16))) Shared sh;
  // Scales of a tile's keys: K, V, and INT4 their middles; V's in units, and as they are (for masked tiles).
  __shared__ __attribute__((aligned(16))) float sc[2][2][4][32];
  __shared__ float unit[2], size[4], units[QB * 256], mine[QB * 256];  // of a lane's rows
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  Work w;
  if (!work_of(a, ROWS, &w)) return;
  const kv_seq &sq = w.sq;
  const int total = sq.past + sq.n;
  const int kfin = w.kfin;  // of the workgroup
  const int wr0 = wave * 16 * QB, first = w.r0 + wr0;  // the wave's first row
  // Keys that some row of the wave sees, and those that all of them see.
  const int wfin = first >= w.rows ? 0
                   : a.tree        ? kfin
                        : min(kfin, sq.past + (min(first + 16 * QB, w.rows) - 1) / a.group + 1);
  const int plain = a.tree ? sq.past : sq.past + min(first, w.rows - 1) / a.group + 1;
  const int all = a.tree ? sq.past : sq.past + w.r0 / a.group + 1;  // of the workgroup
  Quarter<FMT, NB> raw;
  Place p;
  bool refused = false;
  // The codes of the tile at t (looked up before), and the pages of the next.
  auto fetch = [&](int t) __attribute__((always_inline)) {
    p.locate<FMT>(a, w.h, t);
    raw.load(a, p, wave, lane);
    refused |= p.none[0] || p.none[1];
    p.look_up(a, w.b, total, t + 32);
  };
  p.look_up(a, w.b, total, w.kbeg);
  if (w.kbeg < kfin) fetch(w.kbeg);

  stage_queries<DP>(a, sq, w.h, w.r0, w.rows, ROWS, sh.q);
  __syncthreads();
  float row[QB], mx = 0.f;
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    row[qb] = row_max(largest(sh.q + (wr0 + qb * 16 + c) * QP + g * (DP / 4), DP / 4, 0.f));
    mx = fmaxf(mx, row[qb]);
  }
  mx = wave_max(mx);
  if (lane == 0) size[wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(size[0], size[1]), fmaxf(size[2], size[3]));
  const float dn = 32768.f * pow2_under(mx), f = 1.f / dn;
  half8v qh[QB][KS], ql[QB][KS];
  float qs[QB];
  bool uneven = false;
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    float own;
    query_digits<FMT, KS>(sh.q + (wr0 + qb * 16 + c) * QP + g * (DP / 4), row[qb], mx, dn, qh[qb],
                          ql[qb], qs[qb], own);
    uneven |= __any(own != 1.f);
    units[qb * 256 + threadIdx.x] = own;
  }
  __syncthreads();  // the queries' place is the tiles' now

  // Wave 3 keeps the unit of the V scales (INT4: and middles), under the largest so far.
  float vn = ldexpf(1.f, 100);
  auto stage = [&](int at, int t0) __attribute__((always_inline)) {
    raw.convert(sh.t.k[at], sh.t.v[at], wave, lane);
    if (wave == 3) {
      const bool in = t0 + (lane & 31) < total;
      const float vs = in ? raw.vs : 0.f, vz = FMT == MG_KV_INT4 && in ? raw.vz : 0.f;
      const float big = fmaxf(vs, 0.0625f * fabsf(vz));
      if (__builtin_expect(__any(big * vn > 2.f * kScales), 0)) vn = kScales * pow2_under(wave_max(big));
      if (lane < 32) {
        const float ks = raw.none ? __builtin_nanf("") : raw.ks * f, kz = raw.kz * f;
        sc[at][0][0][lane] = ks;
        sc[at][0][1][lane] = vs * vn;
        if (FMT == MG_KV_INT4) {
          sc[at][0][2][lane] = kz;
          sc[at][0][3][lane] = vz * vn;
        }
        if (t0 + 32 > all) {
          sc[at][1][0][lane] = ks;
          sc[at][1][1][lane] = vs;
          if (FMT == MG_KV_INT4) {
            sc[at][1][2][lane] = kz;
            sc[at][1][3][lane] = vz;
          }
        }
      }
      if (lane == 0) unit[at] = vn;
    }
  };

  float4v o[QB][NB];
  float m[QB], l[QB], z[QB];
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    m[qb] = kNoMax;
    l[qb] = z[qb] = 0.f;
#pragma unroll
    for (int i = 0; i < NB; i++) o[qb][i] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  // The units of the wave's outputs: of plain tiles, and (mine) by rows.
  float last = vn;
  bool coarse = false;
#pragma unroll
  for (int qb = 0; qb < QB; qb++) mine[qb * 256 + threadIdx.x] = last;
  auto tile = [&](int at, int t0, float unit_at) __attribute__((always_inline)) {
    // Some row may not see some key.  (A number: as a condition, it is made one of each lane.)
    const uint32_t part = (uint32_t)(plain - (t0 + 32)) >> 31;
    const bool masked = part;
    float4v acc[QB][2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int qb = 0; qb < QB; qb++) acc[qb][u] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const half8v ka = __builtin_bit_cast(half8v, sh.t.k[at][(u * KS + s) * 64 + lane]);
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
          acc[qb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[qb][s], acc[qb][u], 0, 0, 0);
          acc[qb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[qb][s], acc[qb][u], 0, 0, 0);
        }
      }
    }
    float x[4][8];
#pragma unroll
    for (int k = 0; k < (FMT == MG_KV_INT4 ? 4 : 2); k++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const float4 v = *reinterpret_cast<const float4 *>(&sc[at][part][k][16 * u + 4 * g]);
        x[k][4 * u] = v.x, x[k][4 * u + 1] = v.y, x[k][4 * u + 2] = v.z, x[k][4 * u + 3] = v.w;
      }
    // The eight wait states of the last product's result, written out: where paths of different length
    // meet behind a matrix product, the compiler (ROCm 7.2) has left them out.
    if constexpr (QB == 1)
      asm volatile("s_nop 7" : "+v"(acc[0][0]), "+v"(acc[0][1]));
    else
      asm volatile("s_nop 7" : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]));
    half8v ph[QB], pl[QB];
    uint32_t seen[QB];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) seen[qb] = 0xffu;
    // Units of the V scales: a tile that every row sees has the workgroup's, the rows of a
    // masked one their own, by the keys that they see.  (Masked tiles come last.)
    const float now = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(unit_at)));
    float limit = uneven || coarse ? -1.f : kTop;
    if (__builtin_expect(masked || now != last, 0)) {
      float most = 0.f;
#pragma unroll
      for (int qb = 0; qb < QB; qb++) {
        const float was = mine[qb * 256 + threadIdx.x];
        float next = now;
        if (masked) {
          const int qi = min(first + qb * 16 + c, w.rows - 1) / a.group;
          seen[qb] = seen_keys(a, sq, t0, g, a.tree ? sq.past : sq.past + qi + 1,
                               (int64_t)(sq.start + qi) * a.tree_words, kfin);
          float big = 0.f;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float v = FMT == MG_KV_INT4 ? fmaxf(x[1][j], 0.0625f * fabsf(x[3][j])) : x[1][j];
            big = seen[qb] >> j & 1 ? fmaxf(big, v) : big;
          }
          big = row_max(big);
          next = big * was > 2.f * kScales ? kScales * pow2_under(big) : was;
        }
        smaller_unit<NB>(log2_of(was) - log2_of(next), m[qb], l[qb], z[qb], o[qb]);
        mine[qb * 256 + threadIdx.x] = next;
        most = fmaxf(most, next);
      }
      // (2^20 at most: the bound of the weights alone has no such factor.)
      if (masked && limit > 0.f) limit = fminf(kTop / most, 0x1p20f);
      last = now;
    }
    weigh<FMT, NB, QB, true>(masked, mine + threadIdx.x, uneven, units + threadIdx.x, coarse, limit, acc,
                             x[0], x[1], x[2], x[3], qs, seen, m, l, z, o, ph, pl);
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const half8v va = __builtin_bit_cast(half8v, sh.t.v[at][i * 64 + lane]);
#pragma unroll
      for (int qb = 0; qb < QB; qb++) {
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[qb], o[qb][i], 0, 0, 0);
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[qb], o[qb][i], 0, 0, 0);
      }
    }
  };

  if (w.kbeg < kfin) stage(0, w.kbeg);
  if (w.kbeg + 32 < kfin) fetch(w.kbeg + 32);
  int at = 0;
  for (int t0 = w.kbeg; t0 < kfin; t0 += 32) {
    __syncthreads();  // tile t0 is there, and every wave is done with the one before
    const float unit_at = unit[at];
    if (t0 + 32 < kfin) {
      stage(at ^ 1, t0 + 32);
      if (t0 + 64 < kfin) fetch(t0 + 64);
    }
    if (t0 < wfin) tile(at, t0, unit_at);
    at ^= 1;
  }

  if (refused && lane == 0) atomicOr(a.c.refused, 1);
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    const int r = wr0 + qb * 16 + c;
    const float ll = row_sum(l[qb]), zz = FMT == MG_KV_INT4 ? row_sum(z[qb]) : 0.f;
    const float ref = part_ref(m[qb], ll), sum = a.nsplit > 1 ? part_sum(m[qb], ll, ref) : 1.f;
    const float inv = ll == 0.f ? 0.f : 1.f / ll, by = sum / mine[qb * 256 + threadIdx.x];
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
      for (int i = 0; i < NB; i += 4)
        put4<DP>(a, w, r, NB * (4 * g + e) + i,
                 make_float4((o[qb][i][e] + zz) * inv * by, (o[qb][i + 1][e] + zz) * inv * by,
                             (o[qb][i + 2][e] + zz) * inv * by, (o[qb][i + 3][e] + zz) * inv * by));
    if (g == 0) put_stat(a, w, r, ref, sum);
  }
}

// Joins a row's splits, a workgroup a row: LP lanes take four dims each, 256 / LP groups of
// them take splits in turn.
template <int LP>
__global__ __launch_bounds__(256) void k_kv_join(const mg_kv_attn a) {
  constexpr int G = 256 / LP;
  __shared__ float4 sum[256];
  __shared__ float sl[G];
  const int per = (int)a.s.max_new * a.group;  // rows of a (sequence, KV head)
  const int64_t at = blockIdx.x;
  const int bh = (int)(at / per), row = (int)(at - (int64_t)bh * per);
  const int b = bh / a.c.kv_heads, h = bh - b * a.c.kv_heads;
  const kv_seq sq = kv_sequence(a.s, b);
  if (sq.bad || row >= sq.n * a.group) return;
  const int last = min((row / a.rows_wg + 1) * a.rows_wg, sq.n * a.group) - 1;
  const int kend = keys_of(a, sq, last);
  const uint32_t kc = (uint32_t)split_keys(a, sq);
  const int n = max(1, min(a.nsplit, (int)(((uint32_t)kend + kc - 1) / kc)));
  const int dp = a.c.dp, grp = threadIdx.x / LP, d = 4 * (threadIdx.x % LP);
  const float2 *ml = a.part_ml + at * a.nsplit;
  const float *p = a.part + at * a.nsplit * dp + d;
  // (Each wave finds the maximum for itself.)
  float all = kNoMax;
  for (int i = threadIdx.x & 63; i < n; i += 64) all = fmaxf(all, ml[i].x);
  all = wave_max(all);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (d < dp) {
#pragma unroll 4
    for (int i = grp; i < n; i += G) {
      const float2 s = ml[i];
      const float4 x = *reinterpret_cast<const float4 *>(p + (int64_t)i * dp);
      // (2^-10: a row has fewer splits, whose sum then is finite too.)
      const float by = exp2_of(s.x - all - 10.f);
      l += s.y * by;
      v.x += x.x * by;
      v.y += x.y * by;
      v.z += x.z * by;
      v.w += x.w * by;
    }
  }
  sum[threadIdx.x] = v;
  if (threadIdx.x % LP == 0) sl[grp] = l;
  __syncthreads();
  if (threadIdx.x >= LP || d >= a.c.d) return;
  for (int i = 1; i < G; i++) {
    const float4 x = sum[i * LP + threadIdx.x];
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
    l = i == 1 ? sl[0] + sl[1] : l + sl[i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int qi = row / a.group, j = row - qi * a.group;
  float *y = a.y + (sq.start + qi) * a.y_stride + (int64_t)(h * a.group + j) * a.c.d + d;
  y[0] = v.x * inv;
  if (d + 1 < a.c.d) y[1] = v.y * inv;
  if (d + 2 < a.c.d) y[2] = v.z * inv;
  if (d + 3 < a.c.d) y[3] = v.w * inv;
}

template <int FMT, int NB>
void launch(mg_ctx *ctx, const mg_kv_attn &a) {
  const dim3 grid((unsigned)(a.s.batch * a.nsplit * a.nblk * a.c.kv_heads));
  hipStream_t st = ctx->stream;
  if (a.keys)
    k_kv_keys<FMT, NB><<<grid, dim3(256), 0, st>>>(a);
  else if (a.rows_wg == 64)
    k_kv_rows<FMT, NB, 1><<<grid, dim3(256), 0, st>>>(a);
  else if constexpr (NB <= 8)
    k_kv_rows<FMT, NB, 2><<<grid, dim3(256), 0, st>>>(a);
}

template <int FMT>
void launch_dims(mg_ctx *ctx, const mg_kv_attn &a) {
  switch (a.c.dp / 64) {
    case 1: return launch<FMT, 4>(ctx, a);
    case 2: return launch<FMT, 8>(ctx, a);
    case 3: return launch<FMT, 12>(ctx, a);
    default: return launch<FMT, 16>(ctx, a);
  }
}

}  // namespace

size_t mg_kv_attn_plan(const mg_ctx *ctx, mg_kv_attn *a, bool split) {
  const int64_t rows = a->s.max_new * a->group, heads = a->s.batch * a->c.kv_heads;
  // Fills the plan with workgroups of rows_wg rows, `per_cu` of which run at once on a compute unit,
  // and returns about how many microseconds it takes, with `start` for a workgroup's lengths, pages
  // and queries and `tile` for 32 keys.
  const auto plan = [&](int rows_wg, int per_cu, double start, double tile) {
    const int64_t room = (int64_t)per_cu * ctx->num_cus;
    a->rows_wg = rows_wg;
    a->nblk = (int)((rows + rows_wg - 1) / rows_wg);
    // Key splits to fill the room, 128 keys each at least; none for sequences of up to 512, which
    // cost less than the join.
    const int64_t base = heads * a->nblk;
    const int64_t want = split && a->s.max_len > 512 ? std::max<int64_t>(1, room / base) : 1;
    int64_t kc = (a->s.max_len + want - 1) / want;
    kc = std::max<int64_t>(128, (kc + 127) / 128 * 128);
    a->nsplit = want == 1 ? 1 : (int)std::max<int64_t>(1, (a->s.max_len + kc - 1) / kc);
    // The join writes and reads partial results, at some 4 MB a microsecond.
    const double join = a->nsplit > 1 ? 4 + 2e-6 * (double)(heads * rows * a->nsplit * a->c.dp) : 0;
    // All at once: as long as the longest.  Else the room shares the keys, and at the end half of
    // one of the last, which have fewest, is not shared.
    const double len = (double)a->s.max_len, spread = a->tree ? 0 : (double)a->s.max_new;
    const double n = (double)base / (double)room;
    if (base * a->nsplit <= room) return start + join + tile / 32 * (double)(a->nsplit > 1 ? kc : a->s.max_len);
    return start * std::ceil(n) + tile / 32 * (n * (len - spread / 2) + (len - spread) / 2);
  };
  // Measured at full use and with few workgroups (int8, D 128): a tile of 32 keys takes one of 16
  // rows 0.5 us (its four waves have four tiles under way), one of 64 rows 1.8, one of 128 rows
  // 2.1; heads above 128 have the registers for one workgroup of 16 rows a compute unit, two of 64.
  // Chosen so against the other two kinds: 256 rows' prompt over 2000 keys, D 64, by 16 rows 24 us,
  // 64 44, 128 47; 4096 rows of D 96 from none 220, 160 and 205; 2048 rows over 6000 keys, D 128,
  // 680, 561 and 454.
  const bool wide = a->c.dp > 128;
  const double size = a->c.dp / 128.0;
  const auto by16 = [&] { return plan(16, wide ? 1 : 2, 5, 0.5 * size); };
  const auto by64 = [&] { return plan(64, wide ? 2 : 3, 9, wide ? 2 : 0.4 + 1.4 * size); };
  const auto by128 = [&] { return plan(128, 2, 12, 0.5 + 1.6 * size); };
  const double none = std::numeric_limits<double>::infinity();
  const double t128 = wide || rows <= 64 ? none : by128(), t64 = rows <= 16 ? none : by64();
  const double t16 = by16();
  a->keys = t16 <= std::min(t64, t128);
  if (!a->keys) t64 <= t128 ? by64() : by128();
  a->parts = heads * rows * a->nsplit;
  return a->nsplit == 1 ? 0 : (size_t)a->parts * (a->c.dp * 4 + sizeof(float2));
}

mg_status mg_kv_attn_run(mg_ctx *ctx, mg_kv_attn a, void *ws) {
  a.share = 1.f / (float)a.nsplit;
  a.part = static_cast<float *>(ws);
  a.part_ml = reinterpret_cast<float2 *>(a.part + a.parts * a.c.dp);
  const auto odd = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  a.vec = a.c.d % 4 == 0 && a.q_stride % 4 == 0 && a.y_stride % 4 == 0 && !odd(a.q) && !odd(a.y) &&
          a.rope.half_rot % 4 == 0 && !odd(a.rope.cos_table) && !odd(a.rope.sin_table);
  switch (a.c.fmt) {
    case MG_KV_INT8: launch_dims<MG_KV_INT8>(ctx, a); break;
    case MG_KV_E4M3: launch_dims<MG_KV_E4M3>(ctx, a); break;
    default: launch_dims<MG_KV_INT4>(ctx, a); break;
  }
  MG_TRY(mg_launch_check("KV cache attention"));
  if (a.nsplit == 1) return MG_OK;
  const dim3 rows((unsigned)(a.s.batch * a.c.kv_heads * a.s.max_new * a.group));
  if (a.c.dp == 64)
    k_kv_join<16><<<rows, dim3(256), 0, ctx->stream>>>(a);
  else if (a.c.dp == 128)
    k_kv_join<32><<<rows, dim3(256), 0, ctx->stream>>>(a);
  else
    k_kv_join<64><<<rows, dim3(256), 0, ctx->stream>>>(a);
  return mg_launch_check("KV cache attention, join");
}
