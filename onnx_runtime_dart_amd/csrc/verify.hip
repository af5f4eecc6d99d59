// Verification of drafted tokens against the target's distributions.
//
// With m the largest of a row's logits and c = log2(e) / temperature, its weights are
// 2^((x - m) c) and their sum s; the drafted tokens need the weights of single logits only, the
// last token of a sequence a running sum over one row.  Tokens of a large vocabulary have borders
// closer than 1e-5 of each other in that running sum, so weights and sums are in 64 bits: with
// 32 one draw in a hundred would take a neighbour.
//
//   k_stats   (m, s) of every run of 2048 logits, one wave each: the pass over all logits
//   k_walk    a sequence's rows joined, its drafted tokens tried in order (a workgroup each); without
//             draft logits it also draws the last token, from the runs' sums that are there
//   k_masses  with them: the weights left in each run of the one row that it is drawn from
//   k_pick    and the run, and the token in it, that the random number falls into
//
// k_stats is bound by bytes: 98 us for 64 sequences of 5 to 9 rows of 151936 logits of both kinds (12 of
// them at temperature 0, whose draft rows are not read: 767 rows, 466 MB), 4.8 TB/s, the rate of a copy
// (reads alone reach 6.1 to 6.4); the series of 64 bits costs nothing there.  A wave for 2048 logits,
// all loads at once, is the smallest part whose start is hidden.  The others are chains of loads and
// steps of a workgroup: k_walk 5 to 7 us, 15 to 16 with the draw for trees of 25 tokens, k_masses 16 (64
// rows of both kinds, once more), k_pick 6.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mg_internal.h"
#include "verify_common.h"

namespace {

constexpr double kLog2e = 1.44269504088896340736;
constexpr int kLane = MG_DRAFTS_RUN / 64;  // logits of a lane
constexpr float kInf = __builtin_inff();

// 2^t, t at most 0 and a few units above; NaN counts as far below.  The series of e^(f ln 2) for
// |f| <= 1/2: 14 terms, off by (ln 2 / 2)^14 / 14! = 4e-18.
__device__ inline double exp2_of(double t) {
  t = fmax(t, -1100.0);
  const double n = rint(t), f = t - n;
  double y = 1.3691488853904124e-12;
  y = fma(y, f, 2.5678435993488196e-11);
  y = fma(y, f, 4.44553827187081e-10);
  y = fma(y, f, 7.054911620801121e-09);
  y = fma(y, f, 1.0178086009239696e-07);
  y = fma(y, f, 1.3215486790144305e-06);
  y = fma(y, f, 1.5252733804059838e-05);
  y = fma(y, f, 0.00015403530393381606);
  y = fma(y, f, 0.0013333558146428441);
  y = fma(y, f, 0.009618129107628477);
  y = fma(y, f, 0.055504108664821576);
  y = fma(y, f, 0.2402265069591007);
  y = fma(y, f, 0.6931471805599453);
  y = fma(y, f, 1.0);
  return ldexp(y, (int)n);
}
__device__ inline double weight(float x, float m, double c) {
  return exp2_of(((double)x - (double)m) * c);
}

struct Seq {
  int start, n;
};
// Sequence b's rows; n = 0 where it breaks a bound.
__device__ inline Seq sequence(const mg_drafts &d, int64_t b) {
  const int64_t r0 = d.row_start[b], r1 = d.row_start[b + 1];
  const bool bad = r0 < 0 || r1 < r0 || r1 > d.rows || r1 - r0 > d.max_new;
  return bad ? Seq{0, 0} : Seq{(int)r0, (int)(r1 - r0)};
}
__device__ inline float temperature(const mg_drafts &d, int64_t b) {
  return d.temperature ? d.temperature[b] : 1.f;
}

// (Rows need not begin at 16 bytes; the loads may be of four all the same.)
struct __attribute__((packed, aligned(4))) Four {
  float x[4];
};
// The lane's logits of a run: four adjacent ones of every 256.  Past the row's end: -inf.
__device__ inline void load(float (&x)[kLane], const float *row, int64_t first, int64_t vocab,
                            int lane) {
  const float *p = row + first;
  if (first + MG_DRAFTS_RUN <= vocab) {
#pragma unroll
    for (int j = 0; j < kLane / 4; j++) {
      const Four v = *reinterpret_cast<const Four *>(p + 256 * j + 4 * lane);
#pragma unroll
      for (int k = 0; k < 4; k++) x[4 * j + k] = v.x[k];
    }
  } else {
    const int n = (int)(vocab - first);
#pragma unroll
    for (int j = 0; j < kLane; j++) {
      const int i = 256 * (j / 4) + 4 * lane + j % 4;
      x[j] = i < n ? p[i] : -kInf;
    }
  }
}

// x of another lane by a register move (`none` where there is none, or the row takes no part).
template <int CTRL, int ROWS = 0xf>
__device__ inline int moved(int x, int none) {
  return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ inline double moved(double x) {
  const uint64_t u = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)moved<CTRL, ROWS>((int)(uint32_t)u, 0);
  const uint32_t hi = (uint32_t)moved<CTRL, ROWS>((int)(uint32_t)(u >> 32), 0);
  return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}
// Running sums over the wave: within rows of 16 lanes, then across them (0x142, 0x143: a row's last
// lane to the next row's, the second row's to the last two).
__device__ inline double wave_scan(double x) {
  x += moved<0x111>(x);
  x += moved<0x112>(x);
  x += moved<0x114>(x);
  x += moved<0x118>(x);
  x += moved<0x142, 0xa>(x);
  return x + moved<0x143, 0xc>(x);
}
__device__ inline double lane63(double x) {
  const uint64_t u = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}
__device__ inline double wave_sum(double x) { return lane63(wave_scan(x)); }
__device__ inline float wave_max(float x) {
  const int none = (int)__float_as_uint(-kInf);
  auto with = [&](int y) { x = fmaxf(x, __uint_as_float((uint32_t)y)); };
  with(moved<0x111>((int)__float_as_uint(x), none));
  with(moved<0x112>((int)__float_as_uint(x), none));
  with(moved<0x114>((int)__float_as_uint(x), none));
  with(moved<0x118>((int)__float_as_uint(x), none));
  with(moved<0x142>((int)__float_as_uint(x), none));
  with(moved<0x143>((int)__float_as_uint(x), none));
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
__device__ inline int wave_min(int x) {
  x = min(x, moved<0x111>(x, 0x7fffffff));
  x = min(x, moved<0x112>(x, 0x7fffffff));
  x = min(x, moved<0x114>(x, 0x7fffffff));
  x = min(x, moved<0x118>(x, 0x7fffffff));
  x = min(x, moved<0x142>(x, 0x7fffffff));
  x = min(x, moved<0x143>(x, 0x7fffffff));
  return __builtin_amdgcn_readlane(x, 63);
}

__global__ __launch_bounds__(256) void k_stats(const mg_verify v) {
  const mg_drafts &d = v.d;
  const int lane = threadIdx.x & 63;
  const int run = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t b = blockIdx.z;
  const Seq q = sequence(d, b);
  const bool drafted = blockIdx.y >= (unsigned)d.max_new;
  const int i = (int)blockIdx.y - (drafted ? (int)d.max_new : 0);
  const float temp = temperature(d, b);
  // (Nothing was drafted after the last row; the largest logit needs no draft.)
  if (run >= v.nrun || i >= q.n || (drafted && (i + 1 == q.n || !(temp > 0.f)))) return;
  const int64_t row = q.start + i;
  float x[kLane];
  load(x, drafted ? d.draft + row * d.draft_stride : d.target + row * d.target_stride,
       (int64_t)run * MG_DRAFTS_RUN, d.vocab, lane);
  float m = -kInf;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kLane; j++) {
    m = fmaxf(m, x[j]);
    bad |= !(x[j] < kInf);
  }
  m = __any(bad) ? kInf : wave_max(m);
  double s = 0.0;
  if (temp > 0.f && m < kInf) {
    const double c = kLog2e / (double)temp;
#pragma unroll
    for (int j = 0; j < kLane; j++) s += weight(x[j], m, c);
    s = wave_sum(s);
  }
  if (lane == 0) v.part[((drafted ? d.rows : 0) + row) * v.nrun + run] = mg_drafts_part{s, m, 0.f};
}

// A row's maximum and sum from its runs', by a wave; *at: the first run with the maximum.
__device__ inline void join(const mg_drafts_part *p, int nrun, double c, int lane, float *m, double *s,
                            int *at) {
  constexpr int kHeld = 2;  // runs that a lane keeps: vocabularies of up to 262144 are read once
  float top = -kInf, hm[kHeld];
  double hs[kHeld];
  int first = 0x7fffffff;
  auto with = [&](int r, float y) {
    if (y > top || first == 0x7fffffff) first = r;
    top = fmaxf(top, y);
  };
#pragma unroll
  for (int i = 0; i < kHeld; i++) {
    const mg_drafts_part q = p[min(lane + 64 * i, nrun - 1)];
    hm[i] = q.m;
    hs[i] = lane + 64 * i < nrun ? q.s : 0.0;
  }
#pragma unroll
  for (int i = 0; i < kHeld; i++)
    if (lane + 64 * i < nrun) with(lane + 64 * i, hm[i]);
  for (int r = lane + 64 * kHeld; r < nrun; r += 64) with(r, p[r].m);
  const float all = wave_max(top);
  *at = wave_min(top == all ? first : 0x7fffffff);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kHeld; i++) sum += hs[i] * exp2_of(((double)hm[i] - (double)all) * c);
  for (int r = lane + 64 * kHeld; r < nrun; r += 64) sum += p[r].s * exp2_of(((double)p[r].m - (double)all) * c);
  *m = all;
  *s = wave_sum(sum);
}

// The weight left of a token with logits x and (mode 2) y.
__device__ inline double left_of(const mg_drafts_last &l, int mode, float x, float y) {
  const double p = weight(x, l.m, l.c) * l.s;
  return mode == 2 ? fmax(p - weight(y, l.qm, l.c) * l.qs, 0.0) : p;
}
// A run's sum of p's weights.
__device__ inline double mass_of(const mg_drafts_part &p, const mg_drafts_last &l) {
  return p.s * exp2_of(((double)p.m - (double)l.m) * l.c) * l.s;
}

constexpr int kPick = 1024;  // threads that draw a token

// The running sum over the workgroup's threads before this one and up to it (the next one's
// before is this one's up to, bit for bit), and the whole.
struct Sums {
  double before, upto, all;
};
__device__ inline Sums scan(double x, double *part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_scan(x);
  __syncthreads();
  if (lane == 63) part[wave] = x;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int k = 0; k < kPick / 64; k++) {
    if (k == wave) before = all;
    all += part[k];
  }
  // (0x138: the value of the lane before, 0 for the first.)
  return Sums{before + moved<0x138>(x), before + x, all};
}

// Tokens without weight and their probabilities (shared memory), and room for the sums of their runs
// without them.
struct Gone {
  const int *token;
  const double *p;
  int *run;
  double *mass;
  int n;
};
// The last token of a sequence, by the whole workgroup (kPick threads).
__device__ inline void draw_token(const mg_verify &v, const mg_drafts_last &l, int64_t b, const Gone &gone) {
  constexpr int kEach = MG_DRAFTS_RUN / kPick;
  __shared__ double part[kPick / 64], below;
  __shared__ int run, pick, highest, lowest;
  const mg_drafts &d = v.d;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float *x = d.target + l.row * d.target_stride;
  const mg_drafts_part *parts = v.part + l.row * v.nrun;
  // Runs of tokens without weight, a wave each (of tokens of one run: the first).  Where 2^-20 of the
  // run is left or more, that is the difference (sums of 2048 weights are right to 2^-47, so it is to
  // 2^-27); else the run is summed again.
  for (int k = wave; k < gone.n; k += kPick / 64) {
    const int own = __builtin_amdgcn_readfirstlane(gone.token[k]) / MG_DRAFTS_RUN;
    const double whole = mass_of(parts[own], l);
    bool again = false;
    double w = 0.0;
    for (int i0 = 0; i0 < gone.n; i0 += 64) {
      const int i = min(i0 + lane, gone.n - 1);
      const bool in = i0 + lane < gone.n && gone.token[i] / MG_DRAFTS_RUN == own;
      const uint64_t here = __ballot(in);
      again |= here && i0 + __builtin_ctzll(here) < k;
      if (in) w += gone.p[i];
    }
    w = whole - wave_sum(w);
    if (!again && !(w > whole * 0x1p-20)) {
      w = 0.0;
      for (int j0 = 0; j0 < MG_DRAFTS_RUN; j0 += 512) {
        const int64_t first = (int64_t)own * MG_DRAFTS_RUN + j0 + lane;
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = first + 64 * j < d.vocab ? x[first + 64 * j] : -kInf;
        for (int i = 0; i < gone.n; i++) {
          const int64_t at = gone.token[i] - first;
#pragma unroll
          for (int j = 0; j < 8; j++) z[j] = at == 64 * j ? -kInf : z[j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) w += weight(z[j], l.m, l.c) * l.s;
      }
      w = wave_sum(w);
    }
    if (lane == 0) {
      gone.run[k] = again ? -1 : own;
      gone.mass[k] = w;
    }
  }
  if (gone.n) __syncthreads();
  int mode = l.mode;
  const int per = (v.nrun + kPick - 1) / kPick;
  const int r0 = min((int)threadIdx.x * per, v.nrun), r1 = min(r0 + per, v.nrun);
  auto mass = [&](int r) {
    if (mode == 2) return v.mass[b * v.nrun + r];
    int k = -1;
    for (int i = 0; i < gone.n; i++) k = gone.run[i] == r ? i : k;
    return k < 0 ? mass_of(parts[r], l) : gone.mass[k];
  };
  Sums sum;
  double mine;
  for (;;) {
    mine = 0.0;
    for (int r = r0; r < r1; r++) mine += mass(r);
    sum = scan(mine, part);
    if (mode == 1 || sum.all > 0x1p-40) break;
    mode = 1;
  }
  const double want = l.u * sum.all;
  if (threadIdx.x == 0) run = -1, highest = -1, pick = 0x7fffffff, lowest = kPick;
  __syncthreads();
  // The first run whose running sum exceeds it, else (rounding) the last one that has any.  Lanes add
  // the same weights in orders of their own, so sums may fall by a rounding from one to the next, and
  // rise where there is no weight: the first of those with weight counts.
  const uint64_t over = __ballot(mine > 0.0 && sum.upto > want);
  if (over && lane == __builtin_ctzll(over)) atomicMin(&lowest, (int)threadIdx.x);
  __syncthreads();
  if ((int)threadIdx.x == lowest) {
    double at = sum.before, base = at;
    int found = -1;
    for (int r = r0; r < r1; r++) {
      const double w = mass(r);
      if (!(w > 0.0)) continue;
      found = r;
      base = at;
      at += w;
      if (at > want) break;
    }
    run = found;
    below = base;
  }
  __syncthreads();
  if (run < 0) {
    for (int r = r0; r < r1; r++)
      if (mass(r) > 0.0) atomicMax(&highest, r);
    __syncthreads();
    if (threadIdx.x == 0) run = highest, below = 0.0;
    __syncthreads();
  }
  if (run < 0) {
    if (threadIdx.x == 0) v.out[l.out] = -1;
    return;
  }
  const bool end = highest >= 0;
  const float *y = mode == 2 ? d.draft + l.row * d.draft_stride : x;
  double w[kEach], own = 0.0;
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    const int64_t e = (int64_t)run * MG_DRAFTS_RUN + kEach * (int)threadIdx.x + j;
    bool none = e >= d.vocab;
    for (int k = 0; k < gone.n; k++) none |= gone.token[k] == e;
    w[j] = none ? 0.0 : left_of(l, mode, x[e], y[e]);
    own += w[j];
  }
  __syncthreads();
  if (threadIdx.x == 0) highest = -1;
  double at = below + scan(own, part).before;
  int top = -1, here = 0x7fffffff;
#pragma unroll
  for (int j = 0; j < kEach; j++) {
    at += w[j];
    if (w[j] > 0.0) {
      top = kEach * (int)threadIdx.x + j;
      if (!end && at > want) here = min(here, top);
    }
  }
  // (Tokens rise with the lanes: the last lane that has any, the first that is beyond.)
  const uint64_t any = __ballot(top >= 0), beyond = __ballot(here < 0x7fffffff);
  if (any && lane == 63 - __builtin_clzll(any)) atomicMax(&highest, top);
  if (beyond && lane == __builtin_ctzll(beyond)) atomicMin(&pick, here);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int in = pick < 0x7fffffff ? pick : highest;
    v.out[l.out] = in < 0 ? -1 : run * MG_DRAFTS_RUN + in;
  }
}

// DRAFT: the last token is drawn by later launches; else here.
template <bool DRAFT>
__global__ __launch_bounds__(1024) void k_walk(const mg_verify v) {
  constexpr int kMost = MG_DRAFTS_MOST;
  // Rows' sums of weights, tokens' probabilities after their parents (0: never, and for a token
  // that an earlier row after the same one has too).
  __shared__ double s[kMost], qs[kMost], pt[kMost], qt[kMost];
  __shared__ float m[kMost], qm[kMost], u01[kMost];
  __shared__ int token[kMost], parent[kMost], best[kMost];  // best of greedy rows, else rejected tokens
  __shared__ uint16_t child[kMost], next[kMost];  // the first row after a row, the next one after the same; 0: none
  __shared__ int kept_n;
  const mg_drafts &d = v.d;
  const int64_t b = blockIdx.x;
  const Seq q = sequence(d, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ mg_drafts_last last;
  if (q.n == 0) {
    if (threadIdx.x == 0) {
      v.count[b] = 0;
      if (DRAFT) v.last[b].mode = 0;
    }
    return;
  }
  const float temp = temperature(d, b);
  const bool greedy = !(temp > 0.f);
  const double c = greedy ? 0.0 : kLog2e / (double)temp;
  // A row a thread.  Its token's logits are asked for before the rows' parts.
  static_assert(kMost <= 1024, "rows of a sequence");
  const int me = threadIdx.x;
  const int t = me < q.n ? d.tokens[q.start + me] : -1;
  const int up = me < q.n && d.parent ? d.parent[q.start + me] : me - 1;
  const bool hangs = me > 0 && me < q.n && up >= 0 && up < me;
  const bool inside = hangs && t >= 0 && t < d.vocab && !greedy;
  float x = -kInf, y = -kInf;
  if (inside) x = d.target[(q.start + up) * d.target_stride + t];
  if (DRAFT && inside) y = d.draft[(q.start + up) * d.draft_stride + t];
  if (me < q.n) {
    token[me] = t;
    parent[me] = up;
    u01[me] = d.uniform[q.start + me];
  }
  bool same = false;
  int below = 0, beside = 0;
  if (d.parent) {
    __syncthreads();
    if (wave * 64 < q.n) {
#pragma unroll 4
      for (int j = q.n - 1; j > 0; j--) {
        const int pj = parent[j], tj = token[j];
        same |= j < me && pj == up && tj == t;
        if (j > me && pj == me) below = j;
        if (j > me && pj == up) beside = j;
      }
    }
    if (!hangs) beside = 0;
  } else {
    below = me + 1 < q.n ? me + 1 : 0;
  }
  // (The first waves have the rows' threads too.)
  for (int i = 15 - wave; i < q.n; i += 16) {
    const int64_t row = q.start + i;
    float top;
    double sum;
    int at, ignored;
    join(v.part + row * v.nrun, v.nrun, c, lane, &top, &sum, &at);
    if (greedy) {
      // The first logit that is the largest: in its run.
      const int64_t first = (int64_t)at * MG_DRAFTS_RUN;
      float z[kLane];
      load(z, d.target + row * d.target_stride, first, d.vocab, lane);
      int here = 0x7fffffff;
#pragma unroll
      for (int j = kLane - 1; j >= 0; j--)
        if (z[j] == top) here = (int)first + 256 * (j / 4) + 4 * lane + j % 4;
      here = wave_min(here);
      if (lane == 0) best[i] = here;
    }
    if (lane == 0) {
      m[i] = top;
      s[i] = sum;
    }
    if (DRAFT && !greedy && i + 1 < q.n) {
      join(v.part + (d.rows + row) * v.nrun, v.nrun, c, lane, &top, &sum, &ignored);
      if (lane == 0) {
        qm[i] = top;
        qs[i] = sum;
      }
    }
  }
  __syncthreads();
  if (me < q.n) {
    // (A token of weight 0 stays so: the sum is 1 at least.)
    pt[me] = inside && !same ? weight(x, m[up], c) / s[up] : 0.0;
    qt[me] = DRAFT && inside ? weight(y, qm[up], c) / qs[up] : 0.0;
    child[me] = (uint16_t)below;
    next[me] = (uint16_t)beside;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int cur = 0, n = 1, rejected = 0;
    double left = 1.0;
    bool rest = false;
    v.kept[q.start] = 0;
    // (Rows after a row come behind it: children in order are rows in order.)
    bool has = fabsf(m[0]) < kInf;
    for (int i = child[0]; i;) {
      const double u = (double)u01[i], p = pt[i];
      bool stays = has && p > 0.0;
      if (greedy) {
        stays = has && token[i] == best[cur];
      } else if (DRAFT) {
        const bool known = fabsf(qm[cur]) < kInf;
        stays = stays && known && u * qt[i] < p;
        rest = known && !stays;
      } else if (stays && !(u * left < p)) {
        stays = false;
        left -= p;
        qs[rejected] = p;
        best[rejected++] = token[i];
      }
      if (!stays) {
        i = next[i];
        continue;
      }
      v.out[q.start + n - 1] = token[i];
      v.kept[q.start + n++] = i;
      cur = i;
      has = fabsf(m[cur]) < kInf;
      left = 1.0;
      rejected = 0;
      rest = false;
      i = child[i];
    }
    const bool drawn = greedy || !has;
    if (drawn) v.out[q.start + n - 1] = has ? best[cur] : -1;
    last.s = 1.0 / s[cur];
    last.qs = rest ? 1.0 / qs[cur] : 1.0;
    last.c = c;
    last.u = (double)u01[0];
    last.m = m[cur];
    last.qm = rest ? qm[cur] : 0.f;
    last.row = q.start + cur;
    last.mode = drawn ? 0 : rest ? 2 : 1;
    last.rejected = rejected;
    last.out = q.start + n - 1;
    if (DRAFT) v.last[b] = last;
    v.count[b] = n;
    kept_n = n;
  }
  __syncthreads();
  for (int i = kept_n + (int)threadIdx.x; i < q.n; i += 1024) {
    v.out[q.start + i] = -1;
    v.kept[q.start + i] = -1;
  }
  // (parent and pt have been read: they take the runs of rejected tokens.)
  if (!DRAFT && last.mode) draw_token(v, last, b, Gone{best, qs, parent, pt, last.rejected});
}

constexpr int kOne = MG_DRAFTS_RUN / 256;  // logits of a thread of k_masses

// The sums of the weights max(p - q, 0) of a run.
__global__ __launch_bounds__(256) void k_masses(const mg_verify v) {
  __shared__ double part[4];
  const mg_drafts &d = v.d;
  const int64_t b = blockIdx.y;
  if (v.last[b].mode != 2) return;
  const mg_drafts_last l = v.last[b];
  const int64_t first = (int64_t)blockIdx.x * MG_DRAFTS_RUN;
  const float *xr = d.target + l.row * d.target_stride, *yr = d.draft + l.row * d.draft_stride;
  float x[kOne], y[kOne];
  if (first + MG_DRAFTS_RUN <= d.vocab) {
    const int64_t at = first + 4 * (int)threadIdx.x;
    Four v4[kOne / 4], u4[kOne / 4];
#pragma unroll
    for (int j = 0; j < kOne / 4; j++) {
      v4[j] = *reinterpret_cast<const Four *>(xr + at + 1024 * j);
      u4[j] = *reinterpret_cast<const Four *>(yr + at + 1024 * j);
    }
#pragma unroll
    for (int j = 0; j < kOne; j++) {
      x[j] = v4[j / 4].x[j % 4];
      y[j] = u4[j / 4].x[j % 4];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kOne; j++) {
      const int64_t e = first + 1024 * (j / 4) + 4 * (int)threadIdx.x + j % 4;
      x[j] = e < d.vocab ? xr[e] : -kInf;
      y[j] = e < d.vocab ? yr[e] : -kInf;
    }
  }
  double w = 0.0;
#pragma unroll
  for (int j = 0; j < kOne; j++) w += left_of(l, 2, x[j], y[j]);
  w = wave_sum(w);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0) v.mass[b * v.nrun + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ __launch_bounds__(kPick) void k_pick(const mg_verify v) {
  const mg_drafts_last l = v.last[blockIdx.x];
  if (l.mode) draw_token(v, l, blockIdx.x, Gone{nullptr, nullptr, nullptr, nullptr, 0});
}

}  // namespace

size_t mg_verify_plan(mg_verify *v, void *ws) {
  v->nrun = (int)((v->d.vocab + MG_DRAFTS_RUN - 1) / MG_DRAFTS_RUN);
  const size_t parts = mg_align((size_t)v->d.rows * v->nrun * (v->d.draft ? 2 : 1) * sizeof(mg_drafts_part));
  const size_t masses = v->d.draft ? mg_align((size_t)v->d.batch * v->nrun * 8) : 0;
  const size_t lasts = v->d.draft ? mg_align((size_t)v->d.batch * sizeof(mg_drafts_last)) : 0;
  char *p = static_cast<char *>(ws);
  if (p) {
    v->part = reinterpret_cast<mg_drafts_part *>(p);
    v->mass = reinterpret_cast<double *>(p + parts);
    v->last = reinterpret_cast<mg_drafts_last *>(p + parts + masses);
  }
  return parts + masses + lasts;
}

// The grid of k_stats.
struct Grid {
  int64_t x, y, z;
};
static Grid stats_grid(const mg_drafts &d) {
  const int64_t runs = (d.vocab + MG_DRAFTS_RUN - 1) / MG_DRAFTS_RUN;
  return Grid{(runs + 3) / 4, d.max_new * (d.draft ? 2 : 1), d.batch};
}
int64_t mg_verify_groups(const mg_drafts &d) {
  const Grid g = stats_grid(d);
  const int64_t masses = d.draft ? (d.vocab + MG_DRAFTS_RUN - 1) / MG_DRAFTS_RUN * d.batch : 0;
  return std::max(g.x * g.y * g.z, masses);
}

mg_status mg_verify_run(mg_ctx *ctx, const mg_verify &v) {
  const mg_drafts &d = v.d;
  hipStream_t st = ctx->stream;
  const Grid g = stats_grid(d);
  if (d.max_new > 0)
    k_stats<<<dim3((unsigned)g.x, (unsigned)g.y, (unsigned)g.z), dim3(256), 0, st>>>(v);
  if (d.draft) {
    k_walk<true><<<dim3((unsigned)d.batch), dim3(1024), 0, st>>>(v);
    k_masses<<<dim3((unsigned)v.nrun, (unsigned)d.batch), dim3(256), 0, st>>>(v);
    k_pick<<<dim3((unsigned)d.batch), dim3(kPick), 0, st>>>(v);
  } else {
    k_walk<false><<<dim3((unsigned)d.batch), dim3(1024), 0, st>>>(v);
  }
  return mg_launch_check("VerifyDrafts");
}
