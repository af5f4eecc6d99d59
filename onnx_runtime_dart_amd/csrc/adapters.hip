// Low-rank adapters beside shared projections: y = base + f (x A^T) B^T, A [r, K] and B [N, r] of
// each row's own slot.
//
// Two products, the first (down) to r values a row that pass through the workspace.  Few rows: a
// wave per (row, value) streams A, then lanes own outputs and stream B; weights bound it.  Many
// rows are sorted by slot into tiles of 64 rows of one adapter, and both products are made of
// 32 x 32 x 2 fp32 matrix instructions: operands as they are, sums in fp32.  Rows of a tile do
// not touch each other's results, so the order within a slot does not matter.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "adapters_common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;   // rows of a tile
constexpr int kCols = 64;   // values of A's rows that a workgroup takes
constexpr int kOuts = 512;  // outputs that a workgroup takes
constexpr int64_t kFew = 96;

// Four adjacent floats at any address of 4 bytes.
struct __attribute__((packed, aligned(4))) Four {
  float x[4];
};
__device__ inline f32x4 load4(const float *p) {
  const Four v = *reinterpret_cast<const Four *>(p);
  return f32x4{v.x[0], v.x[1], v.x[2], v.x[3]};
}
// Elements k .. k + 3 of a row of K, zeros past its end.
__device__ inline f32x4 load_row(const float *row, int64_t k, int64_t K) {
  if (k + 4 <= K) return load4(row + k);
  f32x4 v = 0;
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (k + e < K) v[e] = row[k + e];
  return v;
}
template <class T>
__device__ inline f32x4 weights(const T *p);
template <>
__device__ inline f32x4 weights<float>(const float *p) {
  return *reinterpret_cast<const f32x4 *>(p);
}
template <>
__device__ inline f32x4 weights<_Float16>(const _Float16 *p) {
  return __builtin_convertvector(*reinterpret_cast<const f16x4 *>(p), f32x4);
}

// ------------------------------------------------------------- filling slots

template <class T>
__global__ __launch_bounds__(256) void k_fill_a(const float *src, T *dst, int64_t K, int64_t kp) {
  const int64_t j = blockIdx.y;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < kp; k += (int64_t)gridDim.x * 256)
    dst[j * kp + k] = (T)(k < K ? src[j * K + k] : 0.f);
}
// B [N, rank] to [rank][np].
template <class T>
__global__ __launch_bounds__(256) void k_fill_b(const float *src, T *dst, int64_t N, int64_t np, int rank) {
  const int64_t j = blockIdx.y;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < np; n += (int64_t)gridDim.x * 256)
    dst[j * np + n] = (T)(n < N ? src[n * rank + j] : 0.f);
}
// (Behind the values, on the same stream: nothing reads a rank without them.)
__global__ void k_fill_slot(int32_t *rank, float *factor, int32_t r, float f) {
  *rank = r;
  *factor = f;
}
__global__ __launch_bounds__(256) void k_empty(int32_t *rank, float *factor, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) rank[i] = 0, factor[i] = 0.f;
}

// ------------------------------------------------------------------ few rows

// The slot of a row: -1 none, -2 beyond the handle's.
__device__ inline int slot_of(const mg_adapt &p, int64_t row) {
  const int s = p.slot[row];
  if (s < 0) return -1;
  if (s >= p.h.slots) return -2;
  return p.h.rank[s] > 0 ? s : -1;
}

// t[row][projection][rank]: a wave per value.
template <class T>
__global__ __launch_bounds__(256) void k_down_few(const mg_adapt p, float *t) {
  const int64_t row = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int col = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int s = slot_of(p, row);
  if (s < 0) return;
  const int rank = p.h.rank[s], i = col / p.h.max_rank, j = col % p.h.max_rank;
  if (i >= p.h.n || j >= rank) return;
  const float *x = p.x + row * p.h.K;
  const T *a = static_cast<const T *>(p.h.a) + s * p.h.a_slot + (int64_t)col * p.h.kp;
  f32x4 sum = 0;
#pragma unroll 4
  for (int64_t k = 4 * lane; k < p.h.kp; k += 256) sum += weights(a + k) * load_row(x, k, p.h.K);
  float v = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if (lane == 0) t[row * p.h.n * p.h.max_rank + col] = v * p.h.factor[s];
}

template <class T>
__global__ __launch_bounds__(64) void k_up_few(const mg_adapt p, const float *t) {
  const int64_t row = blockIdx.y;
  const int i = blockIdx.z;
  const int64_t N = p.h.N[i], n = (int64_t)blockIdx.x * 256 + 4 * threadIdx.x;
  if (n >= N) return;
  const int s = slot_of(p, row);
  const float *base = p.base[i] + row * N;
  float *y = p.y[i] + row * N;
  if (s == -1 && base == y) return;
  f32x4 sum = load_row(base, n, N);
  if (s == -2) sum = __builtin_nanf("");
  if (s >= 0) {
    const int rank = p.h.rank[s];
    const float *tr = t + (row * p.h.n + i) * p.h.max_rank;
    const T *b = static_cast<const T *>(p.h.b) + s * p.h.b_slot + p.h.b_off[i] + n;
    f32x4 add = 0;
#pragma unroll 8
    for (int j = 0; j < rank; j++) add += tr[j] * weights(b + j * p.h.np[i]);
    sum += add;
  }
  if (n + 4 <= N) {
    *reinterpret_cast<Four *>(y + n) = Four{{sum[0], sum[1], sum[2], sum[3]}};
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (n + e < N) y[n + e] = sum[e];
  }
}

// ----------------------------------------------------------------- many rows

// Rows in the order of their slots, and tiles of it.  Buckets: the slots, none, beyond.
struct Tile {
  int slot, start, count, unused;
};
struct Order {
  int32_t *row;  // [rows]
  Tile *tile;    // [most_tiles]
  int32_t *tiles;
};

__global__ __launch_bounds__(1024) void k_sort(const mg_adapt p, const Order o) {
  extern __shared__ int lds[];  // a bucket's rows, then its next place; its first tile
  __shared__ int part[16];
  const int buckets = (int)p.h.slots + 2, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rows = (int)p.rows;
  auto bucket = [&](int s) { return s < 0 ? buckets - 2 : s >= buckets - 2 ? buckets - 1 : s; };
  for (int i = threadIdx.x; i < buckets; i += 1024) lds[i] = 0;
  __syncthreads();
  // (Rows of a prompt lie together: a wave of one bucket counts them at once.)
  auto places = [&](int s, bool in) {
    const int b = in ? bucket(s) : -1;
    const int lead = __builtin_amdgcn_readfirstlane(b);
    int at = 0;
    if (__all(b == lead)) {
      if (lead >= 0) {
        if (lane == 0) at = atomicAdd(lds + lead, 64);
        at = __builtin_amdgcn_readfirstlane(at) + lane;
      }
    } else if (in) {
      at = atomicAdd(lds + b, 1);
    }
    return at;
  };
  // (Eight loads ahead: their latency bounds this.)
  constexpr int kAhead = 8;
  auto each = [&](auto place) {
    for (int r0 = threadIdx.x; r0 - (int)threadIdx.x < rows; r0 += 1024 * kAhead) {
      int s[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; i++) s[i] = p.slot[min(r0 + 1024 * i, rows - 1)];
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const int r = r0 + 1024 * i, to = places(s[i], r < rows);
        if (r < rows) place(r, to);
      }
    }
  };
  each([](int, int) {});
  __syncthreads();
  // First places and tiles, in the buckets' order.
  int at = 0, tiles = 0;
  for (int b0 = 0; b0 < buckets; b0 += 1024) {
    const int b = b0 + threadIdx.x, n = b < buckets ? lds[b] : 0, m = (n + kTile - 1) / kTile;
    int x = n, y = m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(x, d), w = __shfl_up(y, d);
      if (lane >= d) x += u, y += w;
    }
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = at;
    for (int k = 0; k < 16; k++) {
      if (k < wave) before += part[k];
      at += part[k];
    }
    __syncthreads();
    if (lane == 63) part[wave] = y;
    __syncthreads();
    int next = tiles;
    for (int k = 0; k < 16; k++) {
      if (k < wave) next += part[k];
      tiles += part[k];
    }
    const int start = before + x - n;
    next += y - m;
    const int slot = b >= buckets - 1 ? -2 : b == buckets - 2 || n == 0 || p.h.rank[b] == 0 ? -1 : b;
    for (int k = 0; k < m; k++)
      o.tile[next + k] = Tile{slot, start + k * kTile, min(kTile, n - k * kTile), 0};
    if (b < buckets) lds[b] = start;
  }
  if (threadIdx.x == 0) *o.tiles = tiles;
  __syncthreads();
  each([&](int r, int to) { o.row[to] = r; });
}

// Part of t[sorted row][rank * projection + value] of a tile: K's share of blockIdx.y, values
// from kCols * blockIdx.z on.  VEC: K is a multiple of four.
template <class T, bool VEC>
__global__ __launch_bounds__(256, 2) void k_down(const mg_adapt p, const Order o, float *t, int64_t share,
                                                 int64_t cols) {
  constexpr int kDeep = 4;  // steps of eight k that are loaded ahead
  __shared__ float sums[4][64][64];
  if ((int)blockIdx.x >= *o.tiles) return;
  const Tile tile = o.tile[blockIdx.x];
  if (tile.slot < 0) return;
  const int rank = p.h.rank[tile.slot], all = rank * p.h.n, c0 = kCols * blockIdx.z;
  if (c0 >= all) return;
  const int lane = threadIdx.x & 63, hi = lane >> 5, l = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int K = (int)p.h.K;
  const float *x[2];
  const T *a[2];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    x[u] = p.x + (int64_t)o.row[tile.start + min(32 * u + l, tile.count - 1)] * K;
    const int c = min(c0 + 32 * u + l, all - 1), i = c / rank;
    a[u] = static_cast<const T *>(p.h.a) + tile.slot * p.h.a_slot +
           ((int64_t)i * p.h.max_rank + c - i * rank) * p.h.kp;
  }
  f32x16 acc[2][2] = {};
  const int first = (int)(share * blockIdx.y), end = (int)std::min(first + share, p.h.kp);
  // WIDE: a second block of 32 values.  A step is eight k, four for each half of the wave; the four
  // waves take steps in turn.
  auto products = [&](auto wide) {
    constexpr int W = decltype(wide)::value;
#pragma unroll 1
    for (int k0 = first + 8 * wave; k0 < end; k0 += 32 * kDeep) {
      f32x4 xv[kDeep][2], av[kDeep][W];
#pragma unroll
      for (int i = 0; i < kDeep; i++) {
        // (Steps past the end read the last one; x and A count as 0 there.)
        const int k = min(k0 + 32 * i, end - 8) + 4 * hi;
#pragma unroll
        for (int u = 0; u < 2; u++) {
          if (VEC) {
            xv[i][u] = load4(x[u] + min(k, K - 4));
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) xv[i][u][e] = x[u][min(k + e, K - 1)];
          }
        }
#pragma unroll
        for (int w = 0; w < W; w++) av[i][w] = weights(a[w] + k);
      }
#pragma unroll
      for (int i = 0; i < kDeep; i++) {
        const int k = k0 + 32 * i + 4 * hi;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float xe[2], ae[W];
#pragma unroll
          for (int u = 0; u < 2; u++) xe[u] = k + e < K && k < end ? xv[i][u][e] : 0.f;
#pragma unroll
          for (int w = 0; w < W; w++) ae[w] = k < end ? av[i][w][e] : 0.f;
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int w = 0; w < W; w++)
              acc[u][w] = __builtin_amdgcn_mfma_f32_32x32x2f32(xe[u], ae[w], acc[u][w], 0, 0, 0);
        }
      }
    }
  };
  if (c0 + 32 < all)
    products(std::integral_constant<int, 2>());
  else
    products(std::integral_constant<int, 1>());
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int e = 0; e < 16; e++) sums[wave][(2 * u + w) * 16 + e][lane] = acc[u][w][e];
  __syncthreads();
  const float f = p.h.factor[tile.slot];
  t += (int64_t)blockIdx.y * p.rows * cols;
  for (int r = wave; r < 64; r += 4) {
    const int u = r / 32, w = r / 16 % 2, e = r % 16;
    const int row = 32 * u + 8 * (e / 4) + 4 * hi + e % 4, c = c0 + 32 * w + l;
    const float v = (sums[0][r][lane] + sums[1][r][lane]) + (sums[2][r][lane] + sums[3][r][lane]);
    if (row < tile.count && c < all) t[(tile.start + row) * cols + c] = v * f;
  }
}

// Outputs of a tile: kOuts of them of projection blockIdx.z, in blocks of 32 a wave.  stride: of the
// tile's values in shared memory (odd; kHeld of them at a time, rounded up to 32 with zeros).
constexpr int kHeld = 128;
template <class T>
__global__ __launch_bounds__(256, 3) void k_up(const mg_adapt p, const Order o, const float *t, int parts,
                                               int64_t cols, int stride) {
  extern __shared__ float low[];
  __shared__ int row_of[kTile];
  if ((int)blockIdx.x >= *o.tiles) return;
  const Tile tile = o.tile[blockIdx.x];
  const int z = blockIdx.z;
  const int64_t N = p.h.N[z], np = p.h.np[z], n0 = (int64_t)kOuts * blockIdx.y;
  const float *base = p.base[z];
  float *y = p.y[z];
  if (n0 >= N || (tile.slot == -1 && base == y)) return;
  const int lane = threadIdx.x & 63, hi = lane >> 5, l = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int rank = tile.slot >= 0 ? p.h.rank[tile.slot] : 0, steps = (rank + 31) / 32;
  if (threadIdx.x < kTile) row_of[threadIdx.x] = o.row[tile.start + min((int)threadIdx.x, tile.count - 1)];
  auto stage = [&](int j1) {
    const int n = min(kHeld, 32 * steps - j1);
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * n; i += 256) {
      const int r = i / n, j = i % n;
      float v = 0.f;
      if (r < tile.count && j1 + j < rank)
        for (int part = 0; part < parts; part++)
          v += t[((int64_t)part * p.rows + tile.start + r) * cols + z * rank + j1 + j];
      low[r * stride + j] = v;
    }
    __syncthreads();
  };
  stage(0);
  const T *b = static_cast<const T *>(p.h.b) + (int64_t)std::max(tile.slot, 0) * p.h.b_slot + p.h.b_off[z];
  const float *own = low + l * stride + hi;
#pragma unroll 1
  for (int q = 0; q < kOuts / 128; q++) {
    const int64_t at = n0 + 128 * q + 32 * wave, n = std::min(at + l, N - 1);
    if (at >= N && rank <= kHeld) break;  // (else it takes part in what follows)
    float v[2][16];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 16; e++)
        v[u][e] = base[(int64_t)row_of[32 * u + 8 * (e / 4) + 4 * hi + e % 4] * N + n];
    f32x16 acc[2] = {};
#pragma unroll 1
    for (int j0 = 0; j0 < 32 * steps; j0 += 32) {
      if (rank > kHeld && j0 % kHeld == 0) stage(j0);
      float w[16];
      // (Past the rank: its last row, then 0, which no infinity of B turns into NaN.)
#pragma unroll
      for (int j = 0; j < 16; j++) w[j] = (float)b[(int64_t)min(j0 + 2 * j + hi, rank - 1) * np + n];
      if (j0 + 32 > rank) {
#pragma unroll
        for (int j = 0; j < 16; j++) w[j] = j0 + 2 * j + hi < rank ? w[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 16; j++)
#pragma unroll
        for (int u = 0; u < 2; u++)
          acc[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(own[32 * u * stride + j0 % kHeld + 2 * j], w[j], acc[u], 0, 0, 0);
    }
    if (at + l >= N) continue;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int r = 32 * u + 8 * (e / 4) + 4 * hi + e % 4;
        const float sum = tile.slot == -2 ? __builtin_nanf("") : rank ? v[u][e] + acc[u][e] : v[u][e];
        if (r < tile.count) y[(int64_t)row_of[r] * N + n] = sum;
      }
  }
}

int64_t most_tiles(const mg_adapters &h, int64_t rows) {
  return rows / kTile + std::min<int64_t>(h.slots + 2, rows);
}
// The share of K of a workgroup, so that tiles fill the card twice over.
int64_t k_share(const mg_ctx *ctx, const mg_adapters &h, int64_t rows, int *parts) {
  const int64_t groups = (rows + kTile - 1) / kTile * ((h.n * h.max_rank + kCols - 1) / kCols);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(2 * ctx->num_cus / groups, h.kp / 256));
  const int64_t share = ((h.kp + want - 1) / want + 31) / 32 * 32;
  *parts = (int)((h.kp + share - 1) / share);
  return share;
}

template <class T>
void run(mg_ctx *ctx, const mg_adapt &p, void *ws) {
  const mg_adapters &h = p.h;
  hipStream_t st = ctx->stream;
  const unsigned rows = (unsigned)p.rows;
  int64_t most = 0;
  for (int i = 0; i < h.n; i++) most = std::max(most, h.N[i]);
  if (p.rows <= kFew) {
    float *t = static_cast<float *>(ws);
    k_down_few<T><<<dim3((unsigned)((h.n * h.max_rank + 3) / 4), rows), dim3(256), 0, st>>>(p, t);
    k_up_few<T><<<dim3((unsigned)((most + 255) / 256), rows, (unsigned)h.n), dim3(64), 0, st>>>(p, t);
    return;
  }
  int parts;
  const int64_t share = k_share(ctx, h, p.rows, &parts), cols = (int64_t)h.n * h.max_rank;
  const int64_t tiles = most_tiles(h, p.rows);
  char *w = static_cast<char *>(ws);
  Order o;
  o.row = reinterpret_cast<int32_t *>(w);
  w += mg_align((size_t)p.rows * 4);
  o.tiles = reinterpret_cast<int32_t *>(w);
  w += 256;
  o.tile = reinterpret_cast<Tile *>(w);
  w += mg_align((size_t)tiles * sizeof(Tile));
  float *t = reinterpret_cast<float *>(w);
  k_sort<<<dim3(1), dim3(1024), (size_t)(h.slots + 2) * 4, st>>>(p, o);
  const dim3 grid((unsigned)tiles, (unsigned)parts, (unsigned)((cols + kCols - 1) / kCols));
  if (h.K % 4 == 0)
    k_down<T, true><<<grid, dim3(256), 0, st>>>(p, o, t, share, cols);
  else
    k_down<T, false><<<grid, dim3(256), 0, st>>>(p, o, t, share, cols);
  const int stride = std::min((h.max_rank + 31) / 32 * 32, kHeld) + 1;
  k_up<T><<<dim3((unsigned)tiles, (unsigned)((most + kOuts - 1) / kOuts), (unsigned)h.n), dim3(256),
            (size_t)kTile * stride * 4, st>>>(p, o, t, parts, cols, stride);
}

template <class T>
void fill(mg_ctx *ctx, const mg_adapters &h, int64_t slot, int64_t rank, const float *const *a,
          const float *const *b) {
  for (int i = 0; i < h.n; i++) {
    T *ad = static_cast<T *>(h.a) + slot * h.a_slot + (int64_t)i * h.max_rank * h.kp;
    T *bd = static_cast<T *>(h.b) + slot * h.b_slot + h.b_off[i];
    const auto grid = [&](int64_t n) {
      return dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1024), (unsigned)rank);
    };
    k_fill_a<T><<<grid(h.kp), dim3(256), 0, ctx->stream>>>(a[i], ad, h.K, h.kp);
    k_fill_b<T><<<grid(h.np[i]), dim3(256), 0, ctx->stream>>>(b[i], bd, h.N[i], h.np[i], (int)rank);
  }
}

}  // namespace

int64_t mg_adapt_groups(const mg_adapters &h, int64_t rows) {
  int64_t most = 0;
  for (int i = 0; i < h.n; i++) most = std::max(most, h.N[i]);
  return most_tiles(h, std::min(rows, MG_ADAPT_ROWS)) * ((most + kOuts - 1) / kOuts) * h.n;
}

size_t mg_adapt_ws(const mg_ctx *ctx, const mg_adapters &h, int64_t rows) {
  rows = std::min(rows, MG_ADAPT_ROWS);
  const size_t cols = (size_t)h.n * h.max_rank;
  // (A last round of few rows needs no more than a whole one.)
  if (rows <= kFew) return mg_align((size_t)rows * cols * 4);
  int parts;
  k_share(ctx, h, rows, &parts);
  return mg_align((size_t)rows * 4) + 256 + mg_align((size_t)most_tiles(h, rows) * sizeof(Tile)) +
         mg_align((size_t)parts * rows * cols * 4);
}

mg_status mg_adapt_run(mg_ctx *ctx, const mg_adapt &p, void *ws) {
  if (p.h.fmt == MG_ADAPTER_F16)
    run<_Float16>(ctx, p, ws);
  else
    run<float>(ctx, p, ws);
  return mg_launch_check("Adapters");
}

mg_status mg_adapters_fill(mg_ctx *ctx, const mg_adapters &h, int64_t slot, int64_t rank,
                           const float *const *a, const float *const *b, float factor) {
  if (rank) {
    if (h.fmt == MG_ADAPTER_F16)
      fill<_Float16>(ctx, h, slot, rank, a, b);
    else
      fill<float>(ctx, h, slot, rank, a, b);
  }
  k_fill_slot<<<dim3(1), dim3(1), 0, ctx->stream>>>(h.rank + slot, h.factor + slot, (int32_t)rank, factor);
  return mg_launch_check("Adapters fill");
}

mg_status mg_adapters_clear(mg_ctx *ctx, const mg_adapters &h) {
  k_empty<<<dim3((unsigned)((h.slots + 255) / 256)), dim3(256), 0, ctx->stream>>>(h.rank, h.factor, h.slots);
  return mg_launch_check("Adapters clear");
}
