// Log probabilities of given tokens, entropy and the largest logits of each row, in one
// pass over the logits.
//
// With m the row's running maximum, S = sum e^(x - m) and A = sum e^(x - m) (x - m):
//   log p_t = x_t - m - log S,   H = log S - A / S,
// both parts of H being >= 0, so nothing cancels.  When m grows to m', S and A become
// e^(m - m') S and e^(m - m') (A + (m - m') S).  Each lane keeps its own m, S and A over 16
// logits at a time: fp32 sums of at most 128 terms, each at most 1, which then go into sums in 64
// bits, so a long row costs no accuracy; lanes and waves join in 64 bits.  A NaN or +inf logit
// makes S NaN, a row of -inf leaves S 0: neither has a distribution.
//
// The alternatives: each wave keeps its 64 largest entries sorted across its lanes, as
// (key, token) with key the logit's bits in an order that unsigned integers have (NaN
// above all).  An entry enters when it beats the top-th one, found by one comparison per 16
// logits and lane; the top-th largest of the maxima of groups of the first chunk's logits
// bounds the row's top-th from below, so that few entries enter only to leave again.  Up to ten
// alternatives: entries enter one by one, and the sorted lists of waves and of a row's runs
// join by taking the largest head, top times.  More: a chunk's entries are sorted 64 at a time
// by a bitonic network of register moves, and lists join by its last six stages (1000 rows of
// 32000, 64 alternatives: 119 us one by one, 68 so; 8 rows of 151936, 64: 61 and 19, 20: 20 and
// 18, but 1: 9 and 16).
//
// The pass over the logits bounds it, 16-byte loads of which every lane has four in flight:
// 1000 rows of 128256 with 8 alternatives in 105 us (4.9 TB/s, this card's copy rate; one logit
// a lane at a time and every entry offered to the list: 358 us).  Few rows are bound by latency:
// 8 rows of 151936 take 7 us without alternatives.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mg_internal.h"
#include "logprobs_common.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

__device__ inline uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) {
  if (k == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

struct Sums {
  float m;
  double s, a;
};
constexpr float kLowest = -3.402823466e38f;  // the running maximum before any logit

// e^d; d below -200 (that of -inf included) counts as -200: 0 in fp32.
__device__ inline float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// Sums of x brought to the maximum m >= x.m.
__device__ inline Sums moved(const Sums &x, float m) {
  const float d = fmaxf(x.m - m, -200.f), e = x.m == m ? 1.f : exp_of(d);
  return Sums{m, x.s * e, (x.a + (double)d * x.s) * e};
}

// x of another lane by a register move (0 where there is none; rows: those that take part).
template <int CTRL, int ROWS = 0xf>
__device__ inline uint32_t moved_lane(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, true);
}
// Over the wave: within rows of 16 lanes, then across them (0x142, 0x143: a row's last lane to
// the next row's, the second row's to the last two); lane 63 has it all.
__device__ inline uint32_t wave_max(uint32_t x) {
  x = max(x, moved_lane<0x111>(x));
  x = max(x, moved_lane<0x112>(x));
  x = max(x, moved_lane<0x114>(x));
  x = max(x, moved_lane<0x118>(x));
  x = max(x, moved_lane<0x142>(x));
  x = max(x, moved_lane<0x143>(x));
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ inline float wave_sum(float x) {
  auto with = [&](uint32_t y) { x += __uint_as_float(y); };
  with(moved_lane<0x111>(__float_as_uint(x)));
  with(moved_lane<0x112>(__float_as_uint(x)));
  with(moved_lane<0x114>(__float_as_uint(x)));
  with(moved_lane<0x118>(__float_as_uint(x)));
  with(moved_lane<0x142, 0xa>(__float_as_uint(x)));
  with(moved_lane<0x143, 0xc>(__float_as_uint(x)));
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
// A wave's sums from its lanes' (of at most 64 fp32 terms each way).
__device__ inline Sums wave_join(float m, float s, float a) {
  const float all = of_key(wave_max(key_of(m)));
  const float d = fmaxf(m - all, -200.f), e = m == all ? 1.f : exp_of(d);
  return Sums{all, (double)wave_sum(s * e), (double)wave_sum((a + d * s) * e)};
}

// The value of lane l - 1 (lane 0: any).
template <class T>
__device__ inline T lane_before(T x) {
  const int u = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(u, u, 0x138, 0xf, 0xf, false));
}
template <class T>
__device__ inline T lane_value(T x, int l) {
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
}

// A wave's sorted entries, one a lane, and the top-th of them.
struct List {
  uint32_t key, tk;
  int id, ti;
};
__device__ inline bool beats(uint32_t k, int i, uint32_t ok, int oi) {
  return k > ok || (k == ok && i < oi);
}
// Puts in each lane's entry (of lanes with ok) that beats the top-th.
__device__ inline void offer(List &l, uint32_t key, int id, bool ok, int top, int lane) {
  uint64_t want = __ballot(ok && beats(key, id, l.tk, l.ti));
  while (want) {
    const int w = __builtin_ctzll(want);
    const uint32_t k = lane_value(key, w);
    const int i = lane_value(id, w);
    const int at = __popcll(__ballot(beats(l.key, l.id, k, i)));
    const uint32_t pk = lane_before(l.key);
    const int pi = lane_before(l.id);
    if (lane >= at) {
      l.key = lane == at ? k : pk;
      l.id = lane == at ? i : pi;
    }
    l.tk = lane_value(l.key, top - 1);
    l.ti = lane_value(l.id, top - 1);
    want &= want - 1;
    want &= __ballot(beats(key, id, l.tk, l.ti));
  }
}
// A bound from below of the n-th largest (from 1) of the lanes' N keys each, exact to its upper
// half: the largest number with zeros in its lower half that n of them reach.
template <int N>
__device__ inline uint32_t nth_largest(const uint32_t (&x)[N], int n) {
  uint32_t least = 0;
#pragma unroll
  for (int b = 31; b >= 16; b--) {
    const uint32_t t = least | 1u << b;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; i++) count += __popcll(__ballot(x[i] >= t));
    if (count >= n) least = t;
  }
  return least;
}

// The value of lane l ^ X.
template <int X>
__device__ inline uint32_t across(uint32_t x) {
  if constexpr (X == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true);
  if constexpr (X == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true);
  if constexpr (X == 4) {
    // Four lanes up in a row's quads 0 and 2, four down in 1 and 3.
    const int up = __builtin_amdgcn_update_dpp(0, (int)x, 0x104, 0xf, 0x5, false);
    return (uint32_t)__builtin_amdgcn_update_dpp(up, (int)x, 0x114, 0xf, 0xa, false);
  }
  if constexpr (X == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true);
  // (Both results of a swap of x with itself: the even parts' values, the odd parts'.)
  if constexpr (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  }
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return threadIdx.x & 32 ? r[0] : r[1];
}
// Orders entries of lanes l and l ^ X: the better to the lane that has bit X clear, or (up) set.
template <int X>
__device__ inline void order(uint32_t &key, int &id, bool up, int lane) {
  const uint32_t k = across<X>(key);
  const int i = (int)across<X>((uint32_t)id);
  const bool first = ((lane & X) == 0) != up;
  if (beats(k, i, key, id) == first) {  // (no two entries are equal but those of no token)
    key = k;
    id = i;
  }
}
// Sorts a bitonic sequence of 2 X entries in every 2 X lanes.
template <int X>
__device__ inline void order_all(uint32_t &key, int &id, bool up, int lane) {
  order<X>(key, id, up, lane);
  if constexpr (X > 1) order_all<X / 2>(key, id, up, lane);
}
// The best 64 of the list, best first, and of entries given worst first.
__device__ inline void merge(uint32_t &lk, int &li, uint32_t key, int id, int lane) {
  if (beats(key, id, lk, li)) {
    lk = key;
    li = id;
  }
  order_all<32>(lk, li, false, lane);
}
// Puts 64 entries, one a lane, in any order, into the list.
__device__ inline void merge_unsorted(List &l, uint32_t key, int id, int top, int lane) {
  order_all<1>(key, id, (lane & 2) != 0, lane);
  order_all<2>(key, id, (lane & 4) != 0, lane);
  order_all<4>(key, id, (lane & 8) != 0, lane);
  order_all<8>(key, id, (lane & 16) != 0, lane);
  order_all<16>(key, id, (lane & 32) != 0, lane);
  order_all<32>(key, id, true, lane);
  merge(l.key, l.id, key, id, lane);
  l.tk = lane_value(l.key, top - 1);
  l.ti = lane_value(l.id, top - 1);
}
// The wave's own shared memory: writes before it are there for reads after it.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Joins up to 64 sorted lists of `top` entries, lane l's at key[l * pitch], id[l * pitch]
// (n of them): lane j gets the j-th entry of all.  Each lane holds its list's next two.
__device__ inline void join_lists(const uint32_t *key, const int *id, int pitch, int n, int top,
                                  int lane, uint32_t &ok, int &oi) {
  int at = 1;
  uint32_t k = 0, k1 = 0;
  int i = 0x7fffffff, i1 = 0x7fffffff;
  const bool mine = lane < n;
  if (mine) {
    k = key[lane * pitch];
    i = id[lane * pitch];
    if (top > 1) {
      k1 = key[lane * pitch + 1];
      i1 = id[lane * pitch + 1];
    }
  }
  for (int j = 0; j < top; j++) {
    const uint32_t bk = wave_max(k);
    // The lowest token of those with the largest key.
    uint64_t who = __ballot(k == bk);
    int l = __builtin_ctzll(who);
    int bi = lane_value(i, l);
    for (who &= who - 1; who; who &= who - 1) {
      const int o = __builtin_ctzll(who), t = lane_value(i, o);
      if (t < bi) {
        bi = t;
        l = o;
      }
    }
    if (lane == j) {
      ok = bk;
      oi = bi;
    }
    if (lane == l) {
      k = k1;
      i = i1;
      at++;
      const bool more = mine && at < top;
      k1 = more ? key[lane * pitch + at] : 0;
      i1 = more ? id[lane * pitch + at] : 0x7fffffff;
    }
  }
}

// The logit of the row's given token (NaN: none), asked for early by the wave that finishes.
__device__ inline float given(const mg_logprobs &p, int64_t row) {
  if (!p.logprob) return 0.f;
  const int tok = p.tokens[row];
  return tok < 0 || tok >= p.vocab ? __builtin_nanf("") : p.x[row * p.stride + tok];
}
// The row's results, by one wave that holds its sums and list.
__device__ inline void finish(const mg_logprobs &p, int64_t row, const Sums &t, uint32_t lk, int li,
                              float xt, int lane) {
  const double lz = t.s > 0 ? log(t.s) : __builtin_nan("");
  if (lane == 0) {
    if (p.logprob) p.logprob[row] = (float)((double)xt - (double)t.m - lz);
    if (p.entropy) p.entropy[row] = (float)(lz - t.a / t.s);
  }
  if (lane < p.top) {
    p.ids[row * p.top + lane] = li;
    p.lps[row * p.top + lane] = (float)((double)of_key(lk) - (double)t.m - lz);
  }
}

constexpr int kQuads = 4;              // quads of logits a lane takes at a time
constexpr int kChunk = 64 * 4 * kQuads;  // logits a wave takes at a time
constexpr int kFold = 8;               // chunks of a wave whose sums stay in fp32
// Candidates of a chunk put into the list one by one (some 120 cycles each); more are sorted 64 at a
// time (some 1200).
constexpr int kFew = 10;

enum { NONE, FEW, MANY };  // alternatives: none, kFew at most, more

// One workgroup a row (nsplit 1) or one of nsplit runs of a row; its waves take chunks of
// the run in turn.
template <int TOP>
__global__ __launch_bounds__(256) void k_logprobs(const mg_logprobs p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t row = blockIdx.x / (unsigned)p.nsplit;
  const int split = blockIdx.x % (unsigned)p.nsplit;
  const float *x = p.x + row * p.stride;
  // Quads start at 16-byte addresses: logit v is element v + off of the quads.
  const int off = (int)(reinterpret_cast<uintptr_t>(x) >> 2 & 3);
  const float *base = x - off;
  // (64 bits: a vocabulary may come near 2^31.)
  const int64_t end = (int64_t)p.vocab + off;
  const int64_t e0 = (int64_t)split * p.run, e1 = min(end, e0 + p.run);
  const float xt = wave == 0 && p.nsplit == 1 ? given(p, row) : 0.f;
  float m = kLowest, s = 0.f, a = 0.f;
  Sums far{kLowest, 0, 0};
  List l{0, 0, 0x7fffffff, 0x7fffffff};
  bool first = true;
  __shared__ uint32_t ck[4][TOP == MANY ? 128 : 1];  // a wave's candidates, 64 to be sorted at once
  __shared__ int ci[4][TOP == MANY ? 128 : 1];
  int64_t fold = e0 + kFold * 4 * kChunk;
  for (int64_t c0 = e0 + wave * kChunk; c0 < e1; c0 += 4 * kChunk) {
    if (c0 >= fold) {
      far = moved(far, m);
      far.s += s;
      far.a += a;
      s = a = 0.f;
      fold = c0 + kFold * 4 * kChunk;
    }
    float z[kQuads][4];
    const int64_t mine = c0 + lane * 4;
    if (c0 >= off && c0 + kChunk <= e1) {
#pragma unroll
      for (int q = 0; q < kQuads; q++) {
        const float4 v = *reinterpret_cast<const float4 *>(base + mine + q * 256);
        z[q][0] = v.x, z[q][1] = v.y, z[q][2] = v.z, z[q][3] = v.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < kQuads; q++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t e = mine + q * 256 + j;
          z[q][j] = e >= off && e < e1 ? base[e] : -__builtin_inff();
        }
    }
    float big = z[0][0];
#pragma unroll
    for (int q = 0; q < kQuads; q++)
#pragma unroll
      for (int j = 0; j < 4; j++) big = fmaxf(big, z[q][j]);
    const float now = fmaxf(m, big);
    const float d = fmaxf(m - now, -200.f), by = exp_of(d);
    a = (a + d * s) * by;
    s *= by;
    m = now;
#pragma unroll
    for (int q = 0; q < kQuads; q++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float t = z[q][j] - m, e = exp_of(t);
        s += e;
        a = fmaf(e, fmaxf(t, -200.f), a);
      }
    if (TOP) {
      // (NaN: never the maximum, always a candidate.)
      uint32_t quad[kQuads];
      uint32_t bk = 0;
#pragma unroll
      for (int q = 0; q < kQuads; q++) {
        quad[q] = key_of(fmaxf(fmaxf(z[q][0], z[q][1]), fmaxf(z[q][2], z[q][3])));
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 4; j++) odd |= z[q][j] != z[q][j];
        if (odd) quad[q] = 0xffffffffu;
        bk = max(bk, quad[q]);
      }
      uint32_t least = l.tk;
      if (first) {
        const uint32_t one[1] = {bk};
        least = max(least, TOP == FEW ? nth_largest(one, p.top) : nth_largest(quad, p.top));
        first = false;
      }
      if (__any(bk >= least)) {
        int count = 0;
        if (TOP == MANY) {
#pragma unroll
          for (int q = 0; q < kQuads; q++)
#pragma unroll
            for (int j = 0; j < 4; j++) count += __popcll(__ballot(key_of(z[q][j]) >= least));
        }
        int n = 0;
#pragma unroll
        for (int q = 0; q < kQuads; q++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int64_t e = mine + q * 256 + j;
            const int id = (int)(e - off);
            const uint32_t k = key_of(z[q][j]);
            const bool in = e >= off && e < e1 && k >= least;
            if (TOP == FEW || count <= kFew) {
              offer(l, k, id, in, p.top, lane);
              continue;
            }
            const bool ok = in && beats(k, id, l.tk, l.ti);
            const uint64_t who = __ballot(ok);
            if (!who) continue;
            if (ok) {
              const int to = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                                           __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
              ck[wave][to] = k;
              ci[wave][to] = id;
            }
            n += __popcll(who);
            wave_sync();
            if (n < 64) continue;
            merge_unsorted(l, ck[wave][lane], ci[wave][lane], p.top, lane);
            n -= 64;
            const uint32_t rk = ck[wave][64 + lane];
            const int ri = ci[wave][64 + lane];
            wave_sync();
            if (lane < n) {
              ck[wave][lane] = rk;
              ci[wave][lane] = ri;
            }
            wave_sync();
          }
        if (TOP == MANY && n)
          merge_unsorted(l, lane < n ? ck[wave][lane] : 0, lane < n ? ci[wave][lane] : 0x7fffffff, p.top,
                         lane);
        wave_sync();
      }
    }
  }
  far = moved(far, m);
  Sums t = wave_join(m, (float)far.s + s, (float)far.a + a);
  __shared__ Sums st[4];
  __shared__ uint32_t sk[4 * 64];
  __shared__ int si[4 * 64];
  if (lane == 0) st[wave] = t;
  if (TOP) {
    sk[threadIdx.x] = l.key;
    si[threadIdx.x] = l.id;
  }
  __syncthreads();
  if (wave) return;
  float all = st[0].m;
#pragma unroll
  for (int w = 1; w < 4; w++) all = fmaxf(all, st[w].m);
  t = Sums{all, 0, 0};
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const Sums y = moved(st[w], all);
    t.s += y.s;
    t.a += y.a;
  }
  uint32_t lk = l.key;
  int li = l.id;
  if (TOP == FEW) join_lists(sk, si, 64, 4, p.top, lane, lk, li);
  if (TOP == MANY)
    for (int w = 1; w < 4; w++) merge(lk, li, sk[w * 64 + 63 - lane], si[w * 64 + 63 - lane], lane);
  if (p.nsplit == 1) {
    finish(p, row, t, lk, li, xt, lane);
    return;
  }
  mg_logprobs_part &o = p.part[blockIdx.x];
  if (lane == 0) {
    o.m = t.m;
    o.s = t.s;
    o.a = t.a;
  }
  if (lane < p.top) {
    o.key[lane] = lk;
    o.id[lane] = li;
  }
}

// Joins the at most 64 runs of a row: four waves fetch the lists; one joins them, or each merges a
// quarter of them.
template <int TOP>
__global__ __launch_bounds__(256) void k_logprobs_join(const mg_logprobs p) {
  constexpr int T = MG_LOGPROBS_MAX_TOP, PITCH = TOP == FEW ? kFew + 1 : T;
  __shared__ uint32_t sk[TOP ? 64 * PITCH : 1];
  __shared__ int si[TOP ? 64 * PITCH : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const mg_logprobs_part *o = p.part + row * p.nsplit;
  float xt = 0.f;
  Sums t{kLowest, 0, 0};
  if (wave == 0) {
    xt = given(p, row);
    if (lane < p.nsplit) t = Sums{o[lane].m, o[lane].s, o[lane].a};
  }
  uint32_t lk = 0;
  int li = 0x7fffffff;
  if (TOP) {
#pragma unroll 4
    for (int e = threadIdx.x; e < p.nsplit * PITCH; e += 256) {
      const int r = e / PITCH, j = e % PITCH;
      sk[e] = j < p.top ? o[r].key[j] : 0;
      si[e] = j < p.top ? o[r].id[j] : 0x7fffffff;
    }
    __syncthreads();
  }
  if (TOP == MANY) {
    for (int r = wave; r < p.nsplit; r += 4) merge(lk, li, sk[r * T + 63 - lane], si[r * T + 63 - lane], lane);
    __syncthreads();
    sk[threadIdx.x] = lk;
    si[threadIdx.x] = li;
    __syncthreads();
  }
  if (wave) return;
  // (64 bits: the runs' sums may differ by far in size and number.)
  t = moved(t, of_key(wave_max(key_of(t.m))));
#pragma unroll
  for (int w = 32; w; w >>= 1) {
    t.s += __shfl_xor(t.s, w);
    t.a += __shfl_xor(t.a, w);
  }
  if (TOP == FEW) join_lists(sk, si, PITCH, p.nsplit, p.top, lane, lk, li);
  if (TOP == MANY)
    for (int w = 1; w < 4; w++) merge(lk, li, sk[w * 64 + 63 - lane], si[w * 64 + 63 - lane], lane);
  finish(p, row, t, lk, li, xt, lane);
}

template <int TOP>
mg_status launch(mg_ctx *ctx, const mg_logprobs &p) {
  k_logprobs<TOP><<<dim3((unsigned)(p.rows * p.nsplit)), dim3(256), 0, ctx->stream>>>(p);
  MG_TRY(mg_launch_check("log probabilities"));
  if (p.nsplit == 1) return MG_OK;
  k_logprobs_join<TOP><<<dim3((unsigned)p.rows), dim3(256), 0, ctx->stream>>>(p);
  return mg_launch_check("log probabilities, join");
}

}  // namespace

size_t mg_logprobs_plan(const mg_ctx *ctx, mg_logprobs *p, bool split) {
  // Runs for about one workgroup a compute unit, of one chunk a wave at least and at most 64 a
  // row (one lane each where they join).
  int64_t n = 1;
  if (split && p->rows < ctx->num_cus)
    n = std::min<int64_t>({2 * ctx->num_cus / p->rows, (p->vocab + 4 * kChunk - 1) / (4 * kChunk), 64});
  // (Whole chunks of every wave.)
  p->run = (int)std::min<int64_t>(((p->vocab + 3 + n - 1) / n + 4 * kChunk - 1) / (4 * kChunk) *
                                      (4 * kChunk), 0x7fffe000);
  p->nsplit = (int)(((int64_t)p->vocab + 3 + p->run - 1) / p->run);
  return p->nsplit > 1 ? (size_t)p->rows * p->nsplit * sizeof(mg_logprobs_part) : 0;
}

mg_status mg_logprobs_run(mg_ctx *ctx, const mg_logprobs &p) {
  return p.top == 0 ? launch<NONE>(ctx, p) : p.top <= kFew ? launch<FEW>(ctx, p) : launch<MANY>(ctx, p);
}
