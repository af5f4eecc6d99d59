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

#include <cmath>

#include "kv_common.h"
#include "rope_common.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
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

// Max over the four lanes that hold one row.
__device__ inline float row_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float row_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
// 2^-e with |x| in [2^(e-1), 2^e), 2^102 at most; 1 for 0, Infinity and NaN.
__device__ inline float pow2_under(float x) {
  const int e = (int)(__float_as_uint(x) >> 23 & 255u);
  if (e == 255 || x == 0.f) return 1.f;
  return ldexpf(1.f, 126 - max(e, 24));
}

// Floats of a row's partial result: DP outputs, the maximum, the sum, padded.
__host__ __device__ constexpr int part_row(int dp) { return dp + 4; }

struct Tile {
  int64_t page[2];  // of each 16 keys, 0 where there is none
  bool none[2];
};

template <int FMT, int NB, int QB, bool KEYS>
__global__ __launch_bounds__(256) void k_kv_attn(const mg_kv_attn a) {
  constexpr int DP = 16 * NB, KS = DP / 32;
  constexpr int KW = FMT == MG_KV_INT4 ? DP / 32 : DP / 16;  // dwords of a lane's run, 16 keys
  constexpr int RB = DP * (FMT == MG_KV_INT4 ? 4 : 8) / 8;   // bytes of a vector
  constexpr int ROWS = 16 * QB * (KEYS ? 1 : 4);             // rows of the workgroup
  constexpr int QP = DP + 4;
  // 64 rows' queries; later the four waves' results of the same 16 rows.
  static_assert(!KEYS || QB == 1, "the waves' results fill the queries' place");
  __shared__ __attribute__((aligned(16))) float lds[64 * QP];
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
  const int last = min(r0 + ROWS, rows) - 1;
  const int kend = a.tree ? total : sq.past + last / a.group + 1;
  const int kbeg = split * a.kc;
  if (kbeg >= kend && split > 0) return;
  half8v qh[QB][KS], ql[QB][KS];
  float f[QB], qs[QB];
  int see[QB];               // keys below it are seen (tree: past)
  int64_t word[QB];          // the row's words of the tree
  const int wr0 = KEYS ? 0 : wave * 16 * QB;
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    // Queries: turned and scaled in shared memory, 16 rows of each wave at a time.
    constexpr int STAGED = KEYS ? 16 : 64;
    __syncthreads();
    for (int i = threadIdx.x; i < STAGED * DP; i += 256) {
      const int r = i / DP, d = i - r * DP;
      const int row = r0 + (r >> 4) * 16 * QB + qb * 16 + (r & 15);
      float x = 0.f;
      if (row < rows && d < a.c.d) {
        const int qi = row / a.group, j = row - qi * a.group;
        const int64_t at = sq.start + qi;
        const int64_t pos = a.rope.half_rot && a.rope.positions ? a.rope.positions[at] : sq.past + qi;
        x = a.scale2 *
            rope_at(a.q + at * a.q_stride + (int64_t)(h * a.group + j) * a.c.d, d, pos, a.rope);
      }
      lds[r * QP + d] = x;
    }
    __syncthreads();
    const float *x = lds + ((KEYS ? 0 : wave * 16) + c) * QP + g * (DP / 4);
    float mx = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 4; d++) mx = fmaxf(mx, fabsf(x[d]));
    mx = row_max(mx);
    const float dn = 1024.f * pow2_under(mx);
    f[qb] = 1.f / dn;
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
  // Keys below `plain` are seen by every row of the wave.
  const int plain = a.tree ? sq.past : sq.past + min(r0 + wr0, rows - 1) / a.group + 1;
  // Keys that some row of the wave sees, of this split.
  const int wend = r0 + wr0 >= rows ? 0
                   : a.tree         ? total
                                    : sq.past + (min(r0 + wr0 + 16 * QB, rows) - 1) / a.group + 1;
  const int kfin = min(wend, kend - kbeg > a.kc ? kbeg + a.kc : kend);

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

  const int psize = 1 << a.c.plog;
  auto pages = [&](int t0, Tile &t) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int64_t p = t0 + 16 * u < total ? kv_page(a.s, b, t0 + 16 * u, a.c.plog, a.c.pages) : 0;
      t.none[u] = p < 0;
      t.page[u] = p < 0 ? 0 : p;
    }
  };
  bool refused = false;
  const int step = KEYS ? 128 : 32;
  for (int t0 = kbeg + (KEYS ? 32 * wave : 0); t0 < kfin; t0 += step) {
    Tile t;
    pages(t0, t);
    uint32_t kw[2][KW], vw[2][KW];
    float4 ks[2], vs[2], kz[2], vz[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int64_t ph = t.page[u] * a.c.kv_heads + h;
      const int slot = (t0 + 16 * u) & (psize - 1);
      load_run<KW>(kw[u], a.c.k + (ph * psize + slot + c) * RB + g * (RB / 4));
      load_run<KW>(vw[u], a.c.v + (ph * psize + slot + 4 * g) * RB + c * (4 * KW));
      const float *sc = a.c.sc + ph * kv_scales(FMT) * psize + slot + 4 * g;
      ks[u] = *reinterpret_cast<const float4 *>(sc);
      vs[u] = *reinterpret_cast<const float4 *>(sc + psize);
      if (FMT == MG_KV_INT4) {
        kz[u] = *reinterpret_cast<const float4 *>(sc + 2 * psize);
        vz[u] = *reinterpret_cast<const float4 *>(sc + 3 * psize);
      }
      if (t.none[u]) {
        const float nan = __builtin_nanf("");
        ks[u] = make_float4(nan, nan, nan, nan);
        refused = true;
      }
    }
    float ksa[8], vsa[8], kza[8], vza[8];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      ksa[4 * u] = ks[u].x, ksa[4 * u + 1] = ks[u].y, ksa[4 * u + 2] = ks[u].z, ksa[4 * u + 3] = ks[u].w;
      vsa[4 * u] = vs[u].x, vsa[4 * u + 1] = vs[u].y, vsa[4 * u + 2] = vs[u].z, vsa[4 * u + 3] = vs[u].w;
      if (FMT == MG_KV_INT4) {
        kza[4 * u] = kz[u].x, kza[4 * u + 1] = kz[u].y, kza[4 * u + 2] = kz[u].z, kza[4 * u + 3] = kz[u].w;
        vza[4 * u] = vz[u].x, vza[4 * u + 1] = vz[u].y, vza[4 * u + 2] = vz[u].z, vza[4 * u + 3] = vz[u].w;
      }
    }
    const bool masked = t0 + 32 > plain;  // some row may not see some key
    auto key = [&](int j) { return t0 + 16 * (j >> 2) + 4 * g + (j & 3); };
    // V scales relative to the largest seen.
    {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (masked && key(j) >= kfin) vsa[j] = 0.f;
        big = fmaxf(big, vsa[j]);
      }
      if (__any(big * vn > 16.f)) {
        big = row_max(big);
        for (int x = 1; x < 16; x <<= 1) big = fmaxf(big, __shfl_xor(big, x));
        const float now = 8.f * pow2_under(big), by = now / vn;
        vn = now;
#pragma unroll
        for (int qb = 0; qb < QB; qb++)
#pragma unroll
          for (int i = 0; i < NB; i++) o[qb][i] *= by;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) vsa[j] *= vn;
    }
    float4v acc[QB][2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int qb = 0; qb < QB; qb++) acc[qb][u] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const half8v ka = k_operand<FMT, KW>(kw[u], s);
#pragma unroll
        for (int qb = 0; qb < QB; qb++) {
          acc[qb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[qb][s], acc[qb][u], 0, 0, 0);
          acc[qb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[qb][s], acc[qb][u], 0, 0, 0);
        }
      }
    }
    half8v ph[QB], pl[QB];
#pragma unroll
    for (int qb = 0; qb < QB; qb++) {
      float s[8], w[8];
      uint32_t seen = 0xff;
      if (masked) {
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
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float x = acc[qb][j >> 2][j & 3] * f[qb];
        s[j] = x * ksa[j];
        if (FMT == MG_KV_INT4) s[j] = fmaf(qs[qb] * f[qb], kza[j], s[j]);
        if (masked && !(seen >> j & 1)) s[j] = -__builtin_inff();
      }
      float top = s[0];
#pragma unroll
      for (int j = 1; j < 8; j++) top = fmaxf(top, s[j]);
      if (__any(top > m[qb] + kSlack)) {
        const float now = fmaxf(m[qb], row_max(top));
        const float by = exp2f(m[qb] - now);
        m[qb] = now;
        l[qb] *= by;
        z[qb] *= by;
#pragma unroll
        for (int i = 0; i < NB; i++) o[qb][i] *= by;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float p = exp2f(s[j] - m[qb]);
        l[qb] += p;
        w[j] = p * vsa[j];
        if (FMT == MG_KV_INT4) {
          const float pz = p * vza[j];
          z[qb] += masked && !(seen >> j & 1) ? 0.f : pz;
        }
        if (masked && !(seen >> j & 1)) w[j] = 0.f;
        const _Float16 hi = (_Float16)w[j];
        ph[qb][j] = hi;
        pl[qb][j] = (_Float16)(w[j] - (float)hi);
      }
    }
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const half8v va = v_operand<FMT, KW>(vw[0], vw[1], i);
#pragma unroll
      for (int qb = 0; qb < QB; qb++) {
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[qb], o[qb][i], 0, 0, 0);
        o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[qb], o[qb][i], 0, 0, 0);
      }
    }
  }
  if (refused && lane == 0) atomicOr(a.c.refused, 1);
  const float iv = 1.f / vn;
#pragma unroll
  for (int qb = 0; qb < QB; qb++) {
    l[qb] = row_sum(l[qb]);
    z[qb] = FMT == MG_KV_INT4 ? row_sum(z[qb]) : 0.f;
  }
  // Where a row's outputs and statistics go: y, or its partial of this split.
  const int64_t prow = ((int64_t)b * a.c.kv_heads + h) * a.s.max_new * a.group;
  auto put = [&](int r, int d, float v, float mm, float ll) {
    const int row = r0 + r;
    if (row >= rows) return;
    if (a.nsplit > 1) {
      float *p = a.part + ((prow + row) * a.nsplit + split) * part_row(DP);
      p[d] = v;
      if (d == 0) {
        p[DP] = mm;
        p[DP + 1] = ll;
      }
    } else if (d < a.c.d) {
      const int qi = row / a.group, j = row - qi * a.group;
      a.y[(sq.start + qi) * a.y_stride + (int64_t)(h * a.group + j) * a.c.d + d] =
          ll == 0.f ? 0.f : v / ll;
    }
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
      const float all = fmaxf(fmaxf(stat[0][0][r], stat[1][0][r]), fmaxf(stat[2][0][r], stat[3][0][r]));
      const float by = exp2f(m[qb] - all);
#pragma unroll
      for (int i = 0; i < NB; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          lds[(wave * 16 + r) * QP + NB * (4 * g + e) + i] = (o[qb][i][e] * iv + z[qb]) * by;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * DP; i += 256) {
      const int r = i / DP, d = i - r * DP;
      float all = stat[0][0][r], ll = 0.f, v = 0.f;
#pragma unroll
      for (int w = 1; w < 4; w++) all = fmaxf(all, stat[w][0][r]);
#pragma unroll
      for (int w = 0; w < 4; w++) {
        ll += stat[w][1][r] * exp2f(stat[w][0][r] - all);
        v += lds[(w * 16 + r) * QP + d];
      }
      put(r, d, v, all, ll);
    }
  } else {
#pragma unroll
    for (int qb = 0; qb < QB; qb++)
#pragma unroll
      for (int i = 0; i < NB; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          put(wr0 + qb * 16 + c, NB * (4 * g + e) + i, o[qb][i][e] * iv + z[qb], m[qb], l[qb]);
  }
}

// Joins a row's splits: one wave a row.
__global__ __launch_bounds__(256) void k_kv_join(const mg_kv_attn a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t per = a.s.max_new * a.group;  // rows of a (sequence, KV head)
  const int64_t at = (int64_t)blockIdx.x * 4 + wave;
  const int64_t bh = at / per;
  const int row = (int)(at - bh * per);
  const int b = (int)(bh / a.c.kv_heads), h = (int)(bh - (int64_t)b * a.c.kv_heads);
  if (b >= a.s.batch) return;
  const kv_seq sq = kv_sequence(a.s, b);
  if (sq.bad || row >= sq.n * a.group) return;
  const int last = min((row / a.rows_wg + 1) * a.rows_wg, sq.n * a.group) - 1;
  const int kend = a.tree ? sq.past + sq.n : sq.past + last / a.group + 1;
  const int n = max(1, min(a.nsplit, (kend + a.kc - 1) / a.kc));
  const int dp = a.c.dp, pr = part_row(dp);
  const float *p = a.part + at * a.nsplit * pr;
  float all = kNoMax;
  for (int i = lane; i < n; i += 64) all = fmaxf(all, p[(int64_t)i * pr + dp]);
#pragma unroll
  for (int x = 32; x; x >>= 1) all = fmaxf(all, __shfl_xor(all, x));
  float v[4] = {}, l = 0.f;
  for (int i = 0; i < n; i++) {
    const float *q = p + (int64_t)i * pr;
    const float by = exp2f(q[dp] - all);
    l += q[dp + 1] * by;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (lane + 64 * e < dp) v[e] += q[lane + 64 * e] * by;
  }
  const int qi = row / a.group, j = row - qi * a.group;
  float *y = a.y + (sq.start + qi) * a.y_stride + (int64_t)(h * a.group + j) * a.c.d;
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (lane + 64 * e < a.c.d) y[lane + 64 * e] = l == 0.f ? 0.f : v[e] / l;
}

template <int FMT, int NB>
mg_status launch(mg_ctx *ctx, const mg_kv_attn &a) {
  const dim3 grid((unsigned)(a.s.batch * a.nsplit * a.nblk * a.c.kv_heads));
  constexpr int QB = NB > 8 ? 1 : 2;
  hipStream_t st = ctx->stream;
  if (a.mode == 0)
    k_kv_attn<FMT, NB, 1, true><<<grid, dim3(256), 0, st>>>(a);
  else if (a.mode == 1)
    k_kv_attn<FMT, NB, 1, false><<<grid, dim3(256), 0, st>>>(a);
  else
    k_kv_attn<FMT, NB, QB, false><<<grid, dim3(256), 0, st>>>(a);
  return mg_launch_check("KV cache attention");
}

template <int FMT>
mg_status launch_dims(mg_ctx *ctx, const mg_kv_attn &a) {
  switch (a.c.dp / 64) {
    case 1: return launch<FMT, 4>(ctx, a);
    case 2: return launch<FMT, 8>(ctx, a);
    case 3: return launch<FMT, 12>(ctx, a);
    default: return launch<FMT, 16>(ctx, a);
  }
}

}  // namespace

size_t mg_kv_attn_plan(const mg_ctx *ctx, mg_kv_attn *a, bool split) {
  const int64_t rows = a->s.max_new * a->group;
  const int qb = a->c.dp > 128 ? 1 : 2;
  a->mode = rows <= 16 ? 0 : rows <= 64 || qb == 1 ? 1 : 2;
  a->rows_wg = a->mode == 0 ? 16 : a->mode == 1 ? 64 : 64 * qb;
  a->nblk = (int)((rows + a->rows_wg - 1) / a->rows_wg);
  // Key splits: enough workgroups for two a compute unit, 128 keys a split at least.
  const int64_t base = a->s.batch * a->nblk * a->c.kv_heads;
  const int64_t want = split ? std::max<int64_t>(1, 4 * ctx->num_cus / base) : 1;
  int64_t kc = (a->s.max_len + want - 1) / want;
  kc = std::max<int64_t>(128, (kc + 127) / 128 * 128);
  a->nsplit = (int)std::max<int64_t>(1, (a->s.max_len + kc - 1) / kc);
  a->kc = a->nsplit > 1 ? (int)kc : 0x7fffff80;
  if (a->nsplit == 1) return 0;
  return (size_t)(a->s.batch * a->c.kv_heads * rows * a->nsplit) * part_row(a->c.dp) * 4;
}

mg_status mg_kv_attn_run(mg_ctx *ctx, const mg_kv_attn &a) {
  switch (a.c.fmt) {
    case MG_KV_INT8: MG_TRY(launch_dims<MG_KV_INT8>(ctx, a)); break;
    case MG_KV_E4M3: MG_TRY(launch_dims<MG_KV_E4M3>(ctx, a)); break;
    default: MG_TRY(launch_dims<MG_KV_INT4>(ctx, a)); break;
  }
  if (a.nsplit == 1) return MG_OK;
  const int64_t rows = a.s.batch * a.c.kv_heads * a.s.max_new * a.group;
  k_kv_join<<<dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, ctx->stream>>>(a);
  return mg_launch_check("KV cache attention, join");
}
