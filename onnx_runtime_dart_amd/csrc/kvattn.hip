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
//     dim in one dword, NB of them in a row: no transposition, no exchange between lanes,
//     no shared memory in the loop.
// Codes are exact in fp16.  q is a pair of fp16 digits (22 bits) under a power of two of its
// row, and so is a weight times its key's V scale, which is taken relative to the largest
// power of two seen (vn); the products are exact and summed in fp32.  One digit would round
// scores and weights to 2^-11, which fp32 callers see; the second costs products
// that the cached bytes leave idle anyway.
// m moves only when a score exceeds it by 8 (weights up to 2^8 and their sums have room for
// that), so most tiles rescale nothing and exchange nothing between lanes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv_common.h"
#include "rope_common.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -3.0e38f;  // the running maximum before any score
constexpr float kSlack = 8.f;       // how far a score may exceed it

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
__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

template <int FMT, int NB>
struct Shape {
  static constexpr int DP = 16 * NB, KS = DP / 32;
  static constexpr int KW = FMT == MG_KV_INT4 ? DP / 32 : DP / 16;  // dwords of a lane's run, 16 keys
  static constexpr int RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;   // bytes of a vector
};

// A tile of 32 keys: where its two runs of 16 lie, and the lane's codes and scales.  The
// parts are loaded apart.
template <int FMT, int NB>
struct Tile {
  using S = Shape<FMT, NB>;
  int64_t page[2];  // of the tile to be loaded, -1: none
  int64_t at[2];    // (page, head) times page size plus place
  int64_t ph[2];    // (page, head)
  bool none[2];     // no such page: its keys read as NaN
  uint32_t k[2][S::KW], v[2][S::KW];
  float4 ks[2], vs[2], kz[2], vz[2];

  __device__ inline void look_up(const mg_kv_attn &a, int b, int total, int t0) {
#pragma unroll
    for (int u = 0; u < 2; u++)
      page[u] = t0 + 16 * u < total ? kv_page(a.s, b, t0 + 16 * u, a.c.plog, a.c.pages) : 0;
  }
  __device__ inline void locate(const mg_kv_attn &a, int h, int t0) {
    const int psize = 1 << a.c.plog;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      none[u] = page[u] < 0;
      ph[u] = (page[u] < 0 ? 0 : page[u]) * a.c.kv_heads + h;
      at[u] = (ph[u] << a.c.plog) + ((t0 + 16 * u) & (psize - 1));
    }
  }
  __device__ inline void load_k(const mg_kv_attn &a, int g, int c) {
#pragma unroll
    for (int u = 0; u < 2; u++)
      load_run<S::KW>(k[u], a.c.k + at[u] * S::RB + (c * S::RB + g * (S::RB / 4)));
  }
  __device__ inline void load_v(const mg_kv_attn &a, int g, int c) {
#pragma unroll
    for (int u = 0; u < 2; u++)
      load_run<S::KW>(v[u], a.c.v + at[u] * S::RB + (4 * g * S::RB + c * (4 * S::KW)));
  }
  __device__ inline void load_scales(const mg_kv_attn &a, int g) {
    const int psize = 1 << a.c.plog;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      // (page, head)'s scales: kv_scales runs of psize.
      const float *sc = a.c.sc + (ph[u] * (kv_scales(FMT) - 1) << a.c.plog) + at[u] + 4 * g;
      ks[u] = *reinterpret_cast<const float4 *>(sc);
      vs[u] = *reinterpret_cast<const float4 *>(sc + psize);
      if (FMT == MG_KV_INT4) {
        kz[u] = *reinterpret_cast<const float4 *>(sc + 2 * psize);
        vz[u] = *reinterpret_cast<const float4 *>(sc + 3 * psize);
      }
      if (none[u]) {
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

// KEYS: the four waves take tiles in turn for the same rows; else rows of their own.
template <int FMT, int NB, int QB, bool KEYS>
__global__ __launch_bounds__(256, NB * QB <= 8 ? 2 : 1) void k_kv_attn(const mg_kv_attn a) {
  using S = Shape<FMT, NB>;
  constexpr int DP = S::DP, KS = S::KS, KW = S::KW;
  constexpr int ROWS = 16 * QB * (KEYS ? 1 : 4);  // rows of the workgroup
  constexpr int QP = DP + 4;
  // The rows' queries; later (KEYS) the four waves' results.
  __shared__ __attribute__((aligned(16))) float lds[64 * QB * QP];
  __shared__ float stat[4][2][16 * QB];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // Workgroup -> (sequence, split, row block, KV head), heads innermost.
  int id = (int)blockIdx.x;
  const int h = id % a.c.kv_heads;
  id /= a.c.kv_heads;
  const int blk = a.nblk - 1 - id % a.nblk;  // rows that see most keys first
  id /= a.nblk;
  const int split = id % a.nsplit;
  const int b = id / a.nsplit;
  const kv_seq sq = kv_sequence(a.s, b);
  if (sq.bad) {
    if (blk == 0 && split == 0 && h == 0 && threadIdx.x == 0) atomicOr(a.c.refused, 1);
    return;
  }
  const int rows = sq.n * a.group, r0 = blk * ROWS;
  if (r0 >= rows) return;
  // Keys of this workgroup: those its last row sees, of its split.
  const int total = sq.past + sq.n;
  const int kend = a.tree ? total : sq.past + (min(r0 + ROWS, rows) - 1) / a.group + 1;
  const int kbeg = split * a.kc;
  if (kbeg >= kend && split > 0) return;
  const int wr0 = KEYS ? 0 : wave * 16 * QB;  // the wave's first row
  // Keys that some row of the wave sees, of this split, and those that all of them see.
  const int wend = r0 + wr0 >= rows ? 0
                   : a.tree         ? total
                                    : sq.past + (min(r0 + wr0 + 16 * QB, rows) - 1) / a.group + 1;
  const int kfin = min(wend, kend - kbeg > a.kc ? kbeg + a.kc : kend);
  const int plain = a.tree ? sq.past : sq.past + min(r0 + wr0, rows - 1) / a.group + 1;
  constexpr int STEP = KEYS ? 128 : 32;
  // With registers to spare the next tile's loads start before this one's products, else each
  // part's as soon as this one's is used.
  constexpr bool AHEAD = QB == 1 && NB <= 8;
  int t0 = kbeg + (KEYS ? 32 * wave : 0);
  // The first tile's loads run while the queries are made.
  Tile<FMT, NB> t, next;
  bool refused = false;
  if (t0 < kfin) {
    t.look_up(a, b, total, t0);
    t.locate(a, h, t0);
    t.load_k(a, g, c);
    t.load_scales(a, g);
    t.load_v(a, g, c);
    refused = t.none[0] || t.none[1];
    next.look_up(a, b, total, t0 + STEP);
  }

  stage_queries<DP>(a, sq, h, r0, rows, ROWS, lds);
  __syncthreads();
  half8v qh[QB][KS], ql[QB][KS];
  float qs[QB];
  int see[QB];       // keys below it are seen (tree: past)
  int64_t word[QB];  // the row's words of the tree
  float f;
  {
    // One power of two for the wave's rows: the largest element under 2^15, so that a
    // digit pair is exact to 2^-22 of any element down to 2^-17 of it, and to 2^-39 of it below.
    float mx = 0.f;
#pragma unroll
    for (int qb = 0; qb < QB; qb++)
#pragma unroll
      for (int d = 0; d < DP / 4; d++) {
        const float v = fabsf(lds[(wr0 + qb * 16 + c) * QP + g * (DP / 4) + d]);
        mx = v < __builtin_inff() ? fmaxf(mx, v) : mx;
      }
    const float dn = 32768.f * pow2_under(wave_max(mx));
    f = 1.f / dn;
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
      const float *x = lds + (wr0 + qb * 16 + c) * QP + g * (DP / 4);
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float v = x[8 * s + k_slot<FMT>(j)] * dn;
          const _Float16 hi = (_Float16)v;
          qh[qb][s][j] = hi;
          ql[qb][s][j] = (_Float16)(v - (float)hi);
          sum += v;
        }
      qs[qb] = FMT == MG_KV_INT4 ? row_sum(sum) : 0.f;
      const int row = min(r0 + wr0 + qb * 16 + c, rows - 1), qi = row / a.group;
      see[qb] = a.tree ? sq.past : sq.past + qi + 1;
      word[qb] = (int64_t)(sq.start + qi) * a.tree_words;
    }
  }

  float4v o[QB][NB];
  float m[QB], l[QB], z[QB];
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    m[qb] = kNoMax;
    l[qb] = z[qb] = 0.f;
#pragma unroll
    for (int i = 0; i < NB; i++) o[qb][i] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  float vn = ldexpf(1.f, 100);

  // One tile; MASKED: some row may not see some key.
  auto tile = [&](auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const int tn = t0 + STEP;
    const bool more = tn < kfin;
    if (AHEAD && more) {
      next.locate(a, h, tn);
      next.load_k(a, g, c);
      next.load_scales(a, g);
      next.load_v(a, g, c);
      refused |= next.none[0] || next.none[1];
      next.look_up(a, b, total, tn + STEP);
    }
    auto key = [&](int j) { return t0 + 16 * (j >> 2) + 4 * g + (j & 3); };
    float4v acc[QB][2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int qb = 0; qb < QB; qb++) acc[qb][u] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const half8v ka = k_operand<FMT, KW>(t.k[u], s);
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
          acc[qb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[qb][s], acc[qb][u], 0, 0, 0);
          acc[qb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[qb][s], acc[qb][u], 0, 0, 0);
        }
      }
    }
    if (!AHEAD && more) {
      next.locate(a, h, tn);
      next.load_k(a, g, c);
      next.look_up(a, b, total, tn + STEP);
    }
    float ksf[8], vsn[8], kzf[8], vz[8];
    spread(ksf, t.ks, f);
    spread(vsn, t.vs, 1.f);
    if (FMT == MG_KV_INT4) {
      spread(kzf, t.kz, f);
      spread(vz, t.vz, 1.f);
    }
    // V scales relative to the largest seen.
    {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (MASKED && key(j) >= kfin) vsn[j] = 0.f;
        big = fmaxf(big, vsn[j]);
      }
      if (__builtin_expect(__any(big * vn > 16.f), 0)) {
        const float now = 8.f * pow2_under(wave_max(big)), by = now / vn;
        vn = now;
#pragma unroll
        for (int qb = 0; qb < QB; qb++)
#pragma unroll
          for (int i = 0; i < NB; i++) o[qb][i] *= by;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) vsn[j] *= vn;
    }
    half8v ph[QB], pl[QB];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
      uint32_t seen = 0xff;
      if (MASKED) {
        seen = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int k = key(j);
          bool ok = k < see[qb];
          if (a.tree && k >= sq.past && k < total)
            ok = a.tree[word[qb] + ((k - sq.past) >> 6)] >> ((k - sq.past) & 63) & 1;
          if (ok && k < kfin) seen |= 1u << j;
        }
      }
      // Scores less `from`, -inf where not seen.
      float d[8];
      auto scores = [&](float from) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float base = FMT == MG_KV_INT4 ? fmaf(qs[qb], kzf[j], -from) : -from;
          d[j] = fmaf(acc[qb][j >> 2][j & 3], ksf[j], base);
          if (MASKED) d[j] = seen >> j & 1 ? d[j] : -__builtin_inff();
        }
      };
      auto top = [&]() {
        return fmaxf(fmaxf(fmaxf(d[0], d[1]), fmaxf(d[2], d[3])),
                     fmaxf(fmaxf(d[4], d[5]), fmaxf(d[6], d[7])));
      };
      scores(m[qb]);
      if (__builtin_expect(__any(top() > kSlack), 0)) {
        scores(0.f);
        const float now = fmaxf(m[qb], row_max(top()));
        const float by = exp2_of(m[qb] - now);
        m[qb] = now;
        l[qb] *= by;
        z[qb] *= by;
#pragma unroll
        for (int i = 0; i < NB; i++) o[qb][i] *= by;
        scores(now);
      }
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float p0 = exp2_of(d[j]), p1 = exp2_of(d[j + 1]);
        l[qb] += p0;
        l[qb] += p1;
        float w0 = p0 * vsn[j], w1 = p1 * vsn[j + 1];
        // (MASKED: 0 times a NaN that the row does not see.)
        if (MASKED) {
          w0 = seen >> j & 1 ? w0 : 0.f;
          w1 = seen >> (j + 1) & 1 ? w1 : 0.f;
        }
        if (FMT == MG_KV_INT4) {
          const float z0 = p0 * vz[j], z1 = p1 * vz[j + 1];
          z[qb] += !MASKED || seen >> j & 1 ? z0 : 0.f;
          z[qb] += !MASKED || seen >> (j + 1) & 1 ? z1 : 0.f;
        }
        const half2v hi = __builtin_convertvector(float2v{w0, w1}, half2v);
        const half2v lo =
            __builtin_convertvector(float2v{w0 - (float)hi[0], w1 - (float)hi[1]}, half2v);
        ph[qb][j] = hi[0];
        ph[qb][j + 1] = hi[1];
        pl[qb][j] = lo[0];
        pl[qb][j + 1] = lo[1];
      }
    }
    if (!AHEAD && more) {
      next.load_scales(a, g);
      refused |= next.none[0] || next.none[1];
    }
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const half8v va = v_operand<FMT, KW>(t.v[0], t.v[1], i);
#pragma unroll
      for (int qb = 0; qb < QB; qb++) {
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[qb], o[qb][i], 0, 0, 0);
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[qb], o[qb][i], 0, 0, 0);
      }
    }
    if (!AHEAD && more) next.load_v(a, g, c);
    t = next;
    t0 = tn;
  };
  while (t0 < kfin && t0 + 32 <= plain) tile(std::false_type{});
  while (t0 < kfin) tile(std::true_type{});
  if (refused && lane == 0) atomicOr(a.c.refused, 1);
  const float iv = 1.f / vn;
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    l[qb] = row_sum(l[qb]);
    z[qb] = FMT == MG_KV_INT4 ? row_sum(z[qb]) : 0.f;
  }
  // A run of n outputs of row r0 + r from dim d, to y or to the split's partial results.
  const int64_t prow = ((int64_t)b * a.c.kv_heads + h) * a.s.max_new * a.group;
  auto put4 = [&](int r, int d, float4 v, float ll) {
    const int row = r0 + r;
    if (row >= rows) return;
    if (a.nsplit > 1) {
      *reinterpret_cast<float4 *>(a.part + ((prow + row) * a.nsplit + split) * DP + d) = v;
      return;
    }
    const int qi = row / a.group, j = row - qi * a.group;
    float *y = a.y + (sq.start + qi) * a.y_stride + (int64_t)(h * a.group + j) * a.c.d + d;
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    if (a.vec) {
      if (d < a.c.d) *reinterpret_cast<float4 *>(y) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    } else {
      if (d < a.c.d) y[0] = v.x * inv;
      if (d + 1 < a.c.d) y[1] = v.y * inv;
      if (d + 2 < a.c.d) y[2] = v.z * inv;
      if (d + 3 < a.c.d) y[3] = v.w * inv;
    }
  };
  auto put_stat = [&](int r, float mm, float ll) {
    if (r0 + r < rows && a.nsplit > 1)
      a.part_ml[(prow + r0 + r) * a.nsplit + split] = make_float2(mm, ll);
  };
  if (KEYS) {
    // The four waves' results of the same rows, joined.
    if (g == 0) {
#pragma unroll
      for (int qb = 0; qb < QB; qb++) {
        stat[wave][0][qb * 16 + c] = m[qb];
        stat[wave][1][qb * 16 + c] = l[qb];
      }
    }
    __syncthreads();
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
      const int r = qb * 16 + c;
      const float all =
          fmaxf(fmaxf(stat[0][0][r], stat[1][0][r]), fmaxf(stat[2][0][r], stat[3][0][r]));
      const float by = exp2_of(m[qb] - all);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int i = 0; i < NB; i += 4)
          *reinterpret_cast<float4 *>(lds + (wave * ROWS + r) * QP + NB * (4 * g + e) + i) =
              make_float4((o[qb][i][e] * iv + z[qb]) * by, (o[qb][i + 1][e] * iv + z[qb]) * by,
                          (o[qb][i + 2][e] * iv + z[qb]) * by, (o[qb][i + 3][e] * iv + z[qb]) * by);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * DP / 4; i += 256) {
      const int r = i / (DP / 4), d = 4 * (i - r * (DP / 4));
      float mm = stat[0][0][r], ll = 0.f;
#pragma unroll
      for (int w = 1; w < 4; w++) mm = fmaxf(mm, stat[w][0][r]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; w++) {
        ll += stat[w][1][r] * exp2_of(stat[w][0][r] - mm);
        const float4 x = *reinterpret_cast<const float4 *>(lds + (w * ROWS + r) * QP + d);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      put4(r, d, v, ll);
      if (d == 0) put_stat(r, mm, ll);
    }
  } else {
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
      const int r = wr0 + qb * 16 + c;
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int i = 0; i < NB; i += 4)
          put4(r, NB * (4 * g + e) + i,
               make_float4(o[qb][i][e] * iv + z[qb], o[qb][i + 1][e] * iv + z[qb],
                           o[qb][i + 2][e] * iv + z[qb], o[qb][i + 3][e] * iv + z[qb]),
               l[qb]);
      if (g == 0) put_stat(r, m[qb], l[qb]);
    }
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
  const int kend = a.tree ? sq.past + sq.n : sq.past + last / a.group + 1;
  const int n = max(1, min(a.nsplit, (kend + a.kc - 1) / a.kc));
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
      const float by = exp2_of(s.x - all);
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
  if (a.keys) {
    k_kv_attn<FMT, NB, 1, true><<<grid, dim3(256), 0, st>>>(a);
  } else if (a.rows_wg == 64) {
    k_kv_attn<FMT, NB, 1, false><<<grid, dim3(256), 0, st>>>(a);
  } else if constexpr (NB <= 8) {
    k_kv_attn<FMT, NB, 2, false><<<grid, dim3(256), 0, st>>>(a);
  }
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
  // Workgroups that run at once, two a compute unit: more start late, and a start (lengths,
  // pages, queries) costs what some ten tiles do.
  const int64_t room = 2 * ctx->num_cus;
  a->rows_wg = a->c.dp <= 128 ? 128 : 64;
  if (rows <= a->rows_wg / 2) a->rows_wg = 64;
  a->keys = rows <= 16 || (rows <= 256 && heads * ((rows + 15) / 16) <= room / 2);
  if (a->keys) a->rows_wg = 16;
  a->nblk = (int)((rows + a->rows_wg - 1) / a->rows_wg);
  // Key splits to fill the room, 128 keys each at least; none for sequences of up to 512, which
  // cost less than the join.
  const int64_t base = heads * a->nblk;
  const int64_t want = split && a->s.max_len > 512 ? std::max<int64_t>(1, room / base) : 1;
  int64_t kc = (a->s.max_len + want - 1) / want;
  kc = std::max<int64_t>(128, (kc + 127) / 128 * 128);
  a->nsplit = (int)std::max<int64_t>(1, (a->s.max_len + kc - 1) / kc);
  if (want == 1) a->nsplit = 1;
  a->kc = a->nsplit > 1 ? (int)kc : 0x7fffff80;
  a->parts = heads * rows * a->nsplit;
  return a->nsplit == 1 ? 0 : (size_t)a->parts * (a->c.dp * 4 + sizeof(float2));
}

mg_status mg_kv_attn_run(mg_ctx *ctx, mg_kv_attn a, void *ws) {
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
