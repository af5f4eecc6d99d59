// Log probabilities of given tokens, entropy and the largest logits of each row, in one
// pass over the logits.
//
// With m the row's running maximum, S = sum e^(x - m) and A = sum e^(x - m) (x - m):
//   log p_t = x_t - m - log S,   H = log S - A / S,
// both parts of H being >= 0, so nothing cancels.  When m grows to m', S and A become
// e^(m - m') S and e^(m - m') (A + (m - m') S).
//
// The alternatives: each wave keeps its 64 largest entries sorted across its lanes, as
// (key, token) with key the logit's bits in an order that unsigned integers have (NaN
// above all).  An entry enters when it beats the top-th one; after the first few hundred
// elements of a row that is rare (about top ln(n / top) times in n).
#include <hip/hip_runtime.h>

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
// The sums of two parts of a row.
__device__ inline Sums join(const Sums &x, const Sums &y) {
  if (!(x.m > -INFINITY) && x.m == x.m && x.s == 0) return y;
  if (!(y.m > -INFINITY) && y.m == y.m && y.s == 0) return x;
  Sums r;
  r.m = fmaxf(x.m, y.m);
  const double dx = (double)x.m - r.m, dy = (double)y.m - r.m;
  const double ex = exp(dx), ey = exp(dy);
  r.s = x.s * ex + y.s * ey;
  r.a = ex * (x.a + (x.s > 0 ? dx * x.s : 0)) + ey * (y.a + (y.s > 0 ? dy * y.s : 0));
  return r;
}

// Puts (k, id) into the sorted list of the wave (key, then lower token first).
__device__ inline void insert(uint32_t &lk, int &li, uint32_t k, int id, int lane) {
  const bool ahead = lk > k || (lk == k && li < id);
  const int at = __popcll(__ballot(ahead));
  const uint32_t pk = __shfl_up(lk, 1);
  const int pi = __shfl_up(li, 1);
  if (lane == at) {
    lk = k;
    li = id;
  } else if (lane > at) {
    lk = pk;
    li = pi;
  }
}

// Offers each lane's (k, id) to the list; only lanes with ok.
__device__ inline void offer(uint32_t &lk, int &li, uint32_t k, int id, bool ok, int top, int lane) {
  uint32_t tk = __shfl(lk, top - 1);
  int ti = __shfl(li, top - 1);
  uint64_t want = __ballot(ok && (k > tk || (k == tk && id < ti)));
  while (want) {
    const int l = __ffsll((unsigned long long)want) - 1;
    want &= want - 1;
    insert(lk, li, __shfl(k, l), __shfl(id, l), lane);
  }
}

__device__ inline Sums wave_join(Sums x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    Sums y;
    y.m = __shfl_xor(x.m, o);
    y.s = __shfl_xor(x.s, o);
    y.a = __shfl_xor(x.a, o);
    x = join(x, y);
  }
  return x;
}

// The row's results, by one wave that holds its sums and list.
__device__ inline void finish(const mg_logprobs &p, int64_t row, Sums t, bool nan, uint32_t lk,
                              int li, int lane) {
  const float *x = p.x + row * p.stride;
  // NaN and +inf anywhere, and nothing but -inf, leave no distribution.
  const bool none = nan || !(t.m > -INFINITY) || t.m == INFINITY;
  const double lz = none ? __builtin_nan("") : log(t.s);
  if (lane == 0) {
    if (p.logprob) {
      const int tok = p.tokens[row];
      p.logprob[row] = tok < 0 || tok >= p.vocab ? __builtin_nanf("")
                                                 : (float)((double)x[tok] - (double)t.m - lz);
    }
    if (p.entropy) p.entropy[row] = (float)(lz - t.a / t.s);
  }
  if (lane < p.top) {
    p.ids[row * p.top + lane] = li;
    p.lps[row * p.top + lane] = (float)((double)of_key(lk) - (double)t.m - lz);
  }
}

// One workgroup a row (nsplit 1) or one of nsplit runs of a row.
__global__ __launch_bounds__(256) void k_logprobs(mg_logprobs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / p.nsplit;
  const int split = blockIdx.x % p.nsplit;
  const int v0 = split * p.run, v1 = min(p.vocab, v0 + p.run);
  const float *x = p.x + row * p.stride;
  float m = -INFINITY, s = 0.f, a = 0.f;
  bool nan = false;
  uint32_t lk = 0;
  int li = 0x7fffffff;
  for (int v = v0 + wave * 64; v < v1; v += 256) {
    const int id = v + lane;
    const bool ok = id < v1;
    const float z = ok ? x[id] : -INFINITY;
    nan |= z != z;
    if (z > m) {
      const float d = m - z, e = m > -INFINITY ? exp2f(d * kLog2e) : 0.f;
      a = m > -INFINITY ? e * (a + d * s) : 0.f;
      s *= e;
      m = z;
    }
    if (z > -INFINITY) {
      const float d = z - m, e = exp2f(d * kLog2e);
      s += e;
      a += e * d;
    }
    if (p.top > 0) offer(lk, li, key_of(z), id, ok, p.top, lane);
  }
  nan = __any(nan);
  Sums t = wave_join(Sums{m, (double)s, (double)a});
  __shared__ Sums st[4];
  __shared__ int sn[4];
  __shared__ uint32_t sk[4][64];
  __shared__ int si[4][64];
  if (lane == 0) {
    st[wave] = t;
    sn[wave] = nan;
  }
  sk[wave][lane] = lk;
  si[wave][lane] = li;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < 4; w++) {
    t = join(t, st[w]);
    nan |= sn[w] != 0;
    if (p.top > 0) offer(lk, li, sk[w][lane], si[w][lane], lane < p.top && si[w][lane] != 0x7fffffff, p.top, lane);
  }
  if (p.nsplit == 1) {
    finish(p, row, t, nan, lk, li, lane);
    return;
  }
  mg_logprobs_part &o = p.part[blockIdx.x];
  if (lane == 0) {
    o.m = t.m;
    o.nan = nan;
    o.s = t.s;
    o.a = t.a;
  }
  if (lane < p.top) {
    o.key[lane] = lk;
    o.id[lane] = li;
  }
}

__global__ __launch_bounds__(64) void k_logprobs_join(mg_logprobs p) {
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const mg_logprobs_part *o = p.part + row * p.nsplit;
  Sums t{-INFINITY, 0, 0};
  bool nan = false;
  uint32_t lk = 0;
  int li = 0x7fffffff;
  for (int i = lane; i < p.nsplit; i += 64) {
    t = join(t, Sums{o[i].m, o[i].s, o[i].a});
    nan |= o[i].nan != 0;
  }
  t = wave_join(t);
  nan = __any(nan);
  if (p.top > 0)
    for (int i = 0; i < p.nsplit; i++) {
      const bool ok = lane < p.top;
      const uint32_t k = ok ? o[i].key[lane] : 0;
      const int id = ok ? o[i].id[lane] : 0x7fffffff;
      offer(lk, li, k, id, ok && id != 0x7fffffff, p.top, lane);
    }
  finish(p, row, t, nan, lk, li, lane);
}

}  // namespace

size_t mg_logprobs_plan(const mg_ctx *ctx, mg_logprobs *p, bool split) {
  int64_t n = 1;
  if (split && p->rows < 2 * ctx->num_cus)
    n = std::min<int64_t>((2 * ctx->num_cus + p->rows - 1) / p->rows, (p->vocab + 2047) / 2048);
  n = std::max<int64_t>(1, n);
  p->run = (int)(((p->vocab + n - 1) / n + 255) / 256 * 256);
  p->nsplit = (p->vocab + p->run - 1) / p->run;
  return p->nsplit > 1 ? (size_t)p->rows * p->nsplit * sizeof(mg_logprobs_part) : 0;
}

mg_status mg_logprobs_run(mg_ctx *ctx, const mg_logprobs &p) {
  k_logprobs<<<dim3((unsigned)(p.rows * p.nsplit)), dim3(256), 0, ctx->stream>>>(p);
  MG_TRY(mg_launch_check("log probabilities"));
  if (p.nsplit == 1) return MG_OK;
  k_logprobs_join<<<dim3((unsigned)p.rows), dim3(64), 0, ctx->stream>>>(p);
  return mg_launch_check("log probabilities, join");
}
