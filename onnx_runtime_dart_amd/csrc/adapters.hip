// Low-rank adapters beside shared projections: y = base + f (x A^T) B^T, A [r, K] and B [N, r] of
// each row's own slot.
//
// Two products, the first (down) to r values a row that pass through the workspace.  Few rows: a
// wave per (row, value) streams A, then lanes own outputs and stream B; weights bound it.  Many
// rows are sorted by slot into tiles of 64 rows of one adapter, and both products are made of
// 32 x 32 x 2 fp32 matrix instructions: operands as they are, sums in fp32.  Rows of a tile do
// not touch each other's results, so the order within a slot does not matter.
//
// 8191 rows of 3 prompts, 2048 -> 2 x 8192 by 64 in fp32: order 10 us, down 60 to 69 (by the matrix
// instructions, whose rate alone asks for 28, and the latency of the loads between them), up 253 to 284
// (by bytes of base and y: 1.08 GB, 3.8 to 4.3 TB/s).  2494 rows of 5 prompts and 48 tokens, 2048 ->
// 2048, 512, 512 by 16 in fp16: 5.5, 20 and 20 (latencies: 8 steps of 32 k a workgroup, 2 blocks of 128
// outputs).  64 rows, 56 of them with one of 44 adapters, 2048 -> 2048 by 32 in fp32: 4.2 and 4.9 us, the
// latencies of two launches (23 MB of weights, 2.5 TB/s).
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
constexpr int kOuts = 256;  // outputs that a workgroup takes at least
// Few rows: up to 512, and 1.2 10^8 multiply-adds.  Measured where both take as long (all rows of one
// slot / of 64 slots in turn), fp32: 2048 -> 2048 by 64, 500 and 384 rows (9 and 11 us at 32 against 25
// and 26 sorted); 2048 -> 2 x 8192 by 64, 115 and 185; by 16, 330 and 340; 1024 -> 4096 by 8, beyond 512.
// In fp16: beyond; 120 and 360; 420 and beyond; beyond.  The numbers of rows, ranks and outputs
// decide, so the rule is that of one slot; where rows are of many slots it sorts too early: 2 x 8192 by
// 64 in 64 slots, 128 rows, 142 us sorted and 102 as few in fp32, 132 and 53 in fp16.
inline bool few_rows(const mg_adapters &h, int64_t rows) {
  int64_t out = 0;
  for (int i = 0; i < h.n; i++) out += h.N[i];
  return rows <= 512 && rows * h.max_rank <= (int64_t)120000000 / (h.n * h.K + out);
}

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

struct Fill {
  mg_adapters h;
  const float *a[MG_ADAPTER_MOST], *b[MG_ADAPTER_MOST];
  int64_t slot;
  int rank;
  float factor;
};
// blockIdx.z: A [rank, K], as it is, and B [N, rank] to [rank][np] with zeros up to a multiple of 32
// ranks, of each projection in turn; blockIdx.y: the rank.
template <class T>
__global__ __launch_bounds__(256) void k_fill(const Fill f) {
  const int i = blockIdx.z >> 1, j = blockIdx.y;
  const mg_adapters &h = f.h;
  if (blockIdx.x + blockIdx.y + blockIdx.z == 0 && threadIdx.x == 0) {
    h.rank[f.slot] = f.rank;
    h.factor[f.slot] = f.factor;
  }
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  if (blockIdx.z & 1) {
    if (j >= (f.rank + 31) / 32 * 32) return;
    T *dst = static_cast<T *>(h.b) + f.slot * h.b_slot + h.b_off[i] + j * h.np[i];
    for (int64_t n = first; n < h.np[i]; n += step)
      dst[n] = (T)(n < h.N[i] && j < f.rank ? f.b[i][n * f.rank + j] : 0.f);
  } else if (j < f.rank) {
    T *dst = static_cast<T *>(h.a) + f.slot * h.a_slot + ((int64_t)i * h.max_rank + j) * h.kp;
    for (int64_t k = first; k < h.kp; k += step) dst[k] = (T)(k < h.K ? f.a[i][j * h.K + k] : 0.f);
  }
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
  int slot, start, count, rank;
};
// (Loads of what stores might change are not scalar by themselves: a tile is made so, and with it
// every address that begins at its adapter.)
__device__ inline Tile uniform(const Tile &t) {
  return Tile{__builtin_amdgcn_readfirstlane(t.slot), __builtin_amdgcn_readfirstlane(t.start),
              __builtin_amdgcn_readfirstlane(t.count), __builtin_amdgcn_readfirstlane(t.rank)};
}
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
  int s[kAhead];
  bool there = false;
  auto each = [&](auto place) {
    for (int r0 = threadIdx.x; r0 - (int)threadIdx.x < rows; r0 += 1024 * kAhead) {
      // (The second time they are there, if these are all.)
      if (!there || rows > 1024 * kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) s[i] = p.slot[min(r0 + 1024 * i, rows - 1)];
      }
      there = true;
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const int r = r0 + 1024 * i;
        if (r - (int)threadIdx.x >= rows) break;
        const int to = places(s[i], r < rows);
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
    const int rank = n && b < buckets - 2 ? p.h.rank[b] : 0;
    const int slot = b >= buckets - 1 ? -2 : rank == 0 ? -1 : b;
    for (int k = 0; k < m; k++)
      o.tile[next + k] = Tile{slot, start + k * kTile, min(kTile, n - k * kTile), rank};
    if (b < buckets) lds[b] = start;
  }
  if (threadIdx.x == 0) *o.tiles = tiles;
  __syncthreads();
  each([&](int r, int to) { o.row[to] = r; });
}

// Part of t[sorted row][rank * projection + value] of a tile: K's share of blockIdx.y, values
// from kCols * blockIdx.z on.  VEC: K is a multiple of four.  Rows and values pass through shared
// memory 32 k at a time (read from memory by the lines: with operands straight from it every
// instruction touches 64 lines, 110 us and not 65 for 8191 rows of 2048 by 128 values); the
// next 32 k are on their way meanwhile.
template <class T, bool VEC>
__global__ __launch_bounds__(256, 4) void k_down(const mg_adapt p, const Order o, float *t, int64_t share,
                                                 int64_t cols) {
  constexpr int kK = 32, kPad = kK + 4;  // (rows 4 banks apart from each other's multiples: no conflicts)
  __shared__ float xs[kTile * kPad], as[kCols * kPad];
  const int tiles = *o.tiles;  // (asked for with the tile: there is one in the list for every workgroup)
  const Tile tile = uniform(o.tile[blockIdx.x]);
  if ((int)blockIdx.x >= tiles || tile.slot < 0) return;
  const int rank = tile.rank, all = rank * p.h.n, c0 = kCols * blockIdx.z;
  if (c0 >= all) return;
  const int lane = threadIdx.x & 63, hi = lane >> 5, l = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int K = (int)p.h.K, first = (int)(share * blockIdx.y), end = (int)std::min(first + share, p.h.kp);
  // A thread brings four k of rows and of values r + 32 u.
  constexpr int kU = kTile / 32;
  const int r = threadIdx.x >> 3, part = 4 * (threadIdx.x & 7);
  const float *x[kU];
  const T *a[kU];
#pragma unroll
  for (int u = 0; u < kU; u++) {
    x[u] = p.x + (int64_t)o.row[tile.start + min(32 * u + r, tile.count - 1)] * K;
    const int c = min(c0 + 32 * u + r, all - 1), i = c / rank;
    a[u] = static_cast<const T *>(p.h.a) + tile.slot * p.h.a_slot +
           ((int64_t)i * p.h.max_rank + c - i * rank) * p.h.kp;
  }
  f32x4 xv[kU], av[kU];
  auto load = [&](int k0) {
    const int k = k0 + part;
#pragma unroll
    for (int u = 0; u < kU; u++) {
      // (Past the end: the last ones, where x and A count as 0.)
      if (VEC) {
        xv[u] = load4(x[u] + min(k, K - 4));
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) xv[u][e] = x[u][min(k + e, K - 1)];
      }
      av[u] = weights(a[u] + min(k, end - 4));
    }
    if (k0 + kK > std::min(end, K)) {
#pragma unroll
      for (int u = 0; u < kU; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          xv[u][e] = k + e < K && k < end ? xv[u][e] : 0.f;
          av[u][e] = k < end ? av[u][e] : 0.f;
        }
    }
  };
  // More than 32 values: a wave takes one block of 32 rows by 32 values; else half of the k of one.
  const bool wide = c0 + 32 < all;
  const int rows0 = 32 * (wave & 1), cols0 = wide ? 32 * (wave >> 1) : 0;
  // (A wave whose rows the tile does not have only brings operands.)
  const int s0 = wide ? 0 : 2 * (wave >> 1), s1 = rows0 >= tile.count ? 0 : wide ? 4 : s0 + 2;
  const float *xl = xs + (rows0 + l) * kPad + 4 * hi, *al = as + (cols0 + l) * kPad + 4 * hi;
  f32x16 acc = {};
  load(first);
  for (int k0 = first; k0 < end; k0 += kK) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kU; u++) {
      *reinterpret_cast<f32x4 *>(xs + (32 * u + r) * kPad + part) = xv[u];
      *reinterpret_cast<f32x4 *>(as + (32 * u + r) * kPad + part) = av[u];
    }
    __syncthreads();
    if (k0 + kK < end) load(k0 + kK);
#pragma unroll
    for (int s = 0; s < 4; s++) {
      if (s < s0 || s >= s1) continue;
      const f32x4 xe = *reinterpret_cast<const f32x4 *>(xl + 8 * s);
      const f32x4 ae = *reinterpret_cast<const f32x4 *>(al + 8 * s);
#pragma unroll
      for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(xe[e], ae[e], acc, 0, 0, 0);
    }
  }
  const float f = p.h.factor[tile.slot];
  t += (int64_t)blockIdx.y * p.rows * cols;
  if (!wide) {
    __syncthreads();
    if (wave >= 2) {
#pragma unroll
      for (int e = 0; e < 16; e++) xs[((wave & 1) * 16 + e) * 64 + lane] = acc[e];
    }
    __syncthreads();
    if (wave >= 2) return;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] += xs[(wave * 16 + e) * 64 + lane];
  }
  const int c = c0 + cols0 + l;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const int row = rows0 + 8 * (e / 4) + 4 * hi + e % 4;
    if (row < tile.count && c < all) t[(tile.start + row) * cols + c] = acc[e] * f;
  }
}

// Outputs of a tile: `outs` of them of projection blockIdx.z, 32 a wave at a time.  Products change
// lanes through the wave's own part of shared memory, so that base and y are read and written 16
// bytes a lane and a line of a row at once; waves wait for each other only at the start.  Weights
// and base of the next block are asked for between a block's products and its stores.  stride: of
// the tile's values in shared memory (odd; kHeld of them at a time, rounded up to 32 with zeros).
constexpr int kHeld = 128, kTurn = 36;
template <class T>
__global__ __launch_bounds__(256, 3) void k_up(const mg_adapt p, const Order o, const float *t, int parts,
                                               int64_t cols, int stride, int outs) {
  extern __shared__ float low[];
  __shared__ float turns[4][32 * kTurn];
  __shared__ int64_t row_of[kTile];  // where the rows' outputs begin
  const int tiles = *o.tiles;
  const Tile tile = uniform(o.tile[blockIdx.y]);
  // The projection and its outputs (all chunks of all projections side by side: a grid with empty
  // places gives some XCDs less to do).
  int z = 0, chunk = blockIdx.x;
  while (z + 1 < p.h.n && chunk >= (int)((p.h.N[z] + outs - 1) / outs)) chunk -= (int)((p.h.N[z++] + outs - 1) / outs);
  const int64_t N = p.h.N[z], np = p.h.np[z], n0 = (int64_t)outs * chunk;
  const float *base = p.base[z];
  float *y = p.y[z];
  if ((int)blockIdx.y >= tiles || (tile.slot == -1 && base == y)) return;
  const int64_t last = std::min(n0 + outs, N);  // of the workgroup's outputs
  const int lane = threadIdx.x & 63, hi = lane >> 5, l = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (threadIdx.x < kTile)
    row_of[threadIdx.x] = o.row[tile.start + min((int)threadIdx.x, tile.count - 1)] * N;
  const int rank = tile.rank;
  const T *b = static_cast<const T *>(p.h.b) + tile.slot * p.h.b_slot + p.h.b_off[z];
  // A lane's outputs of a block: four of rows r8 + 8 i.
  const int r8 = lane >> 3, part4 = 4 * (lane & 7);
  struct Block {
    f32x4 v[8];
  };
  auto load_base = [&](const float *from, int64_t at) {
    Block v;
#pragma unroll
    for (int i = 0; i < 8; i++) v.v[i] = load4(from + row_of[r8 + 8 * i] + at + part4);
    return v;
  };
  if (tile.slot < 0) {
    // No adapter: the base, beyond the slots: NaN.
    __syncthreads();
    const bool none = tile.slot == -1;
    const float nan = __builtin_nanf("");
#pragma unroll 2
    for (int64_t at = n0 + 32 * wave; at < last; at += 128) {
      if (at + 32 <= last) {
        Block v;
#pragma unroll
        for (int i = 0; i < 8; i++) v.v[i] = nan;
        if (none) v = load_base(base, at);
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (r8 + 8 * i < tile.count)
            *reinterpret_cast<Four *>(y + row_of[r8 + 8 * i] + at + part4) =
                Four{{v.v[i][0], v.v[i][1], v.v[i][2], v.v[i][3]}};
      } else {
        for (int r = hi; r < tile.count; r += 2)
          if (at + l < last) y[row_of[r] + at + l] = none ? base[row_of[r] + at + l] : nan;
      }
    }
    return;
  }
  struct Weights {
    float w[16];
  };
  // Weights of 32 ranks from j0 on (past the rank: zeros), by one address a lane and 16 scalar ones.
  auto load_weights = [&](int n, int j0) {
    Weights w;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T *>(b + j0 * np), (short)0, (int)(uint32_t)std::min<int64_t>(32 * np * (int)sizeof(T), 0x7ffffff0),
        0x00020000);
    const unsigned at = (unsigned)(hi * (int)np + n) * (unsigned)sizeof(T);
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const unsigned row = (unsigned)(2 * j) * (unsigned)np * (unsigned)sizeof(T);
      if (sizeof(T) == 4)
        w.w[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at, row, 0));
      else
        w.w[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, row, 0));
    }
    return w;
  };
  const float *own = low + l * stride + hi;
  auto products = [&](const Weights &w, int j0, f32x16 (&acc)[2]) {
#pragma unroll
    for (int j = 0; j < 16; j++)
#pragma unroll
      for (int u = 0; u < 2; u++)
        acc[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(own[32 * u * stride + j0 + 2 * j], w.w[j], acc[u], 0, 0, 0);
  };
  float *turn = turns[wave];
  // (Ranks beyond kHeld are added in rounds: to the base, then to what a lane wrote itself.)
#pragma unroll 1
  for (int j1 = 0; j1 < rank; j1 += kHeld) {
    const int j2 = min(j1 + kHeld, rank);
    __syncthreads();
    // The tile's values: 32 of each row at a time, eight a thread.
#pragma unroll 1
    for (int j0 = j1; j0 < j2; j0 += 32) {
      const int j = j0 + l;
      float v[8] = {};
#pragma unroll 2
      for (int part = 0; part < parts; part++) {
        const float *from = t + ((int64_t)part * p.rows + tile.start) * cols + z * rank;
#pragma unroll
        for (int i = 0; i < 8; i++)
          v[i] += from[(uint32_t)(min(2 * wave + hi + 8 * i, tile.count - 1) * (int)cols + min(j, rank - 1))];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) low[(2 * wave + hi + 8 * i) * stride + j - j1] = j < rank ? v[i] : 0.f;
    }
    __syncthreads();
    const float *from = j1 ? y : base;
    int64_t at = n0 + 32 * wave;
    // (A block of less than 32 outputs, the last one, reads its base at the end.)
    Block v = {};
    Weights w0, w1;
    auto load_both = [&](int64_t to) {
      const int col = (int)std::min(to + l, N - 1);
      w0 = load_weights(col, j1);
      if (j1 + 32 < j2) w1 = load_weights(col, j1 + 32);
    };
    load_both(at);
    if (at + 32 <= last) v = load_base(from, at);
#pragma unroll 1
    for (; at < last; at += 128) {
      asm volatile("" ::: "memory");  // (the tile's values stay in shared memory: registers are for loads)
      f32x16 acc[2] = {};
      products(w0, 0, acc);
      if (j1 + 32 < j2) products(w1, 32, acc);
#pragma unroll 1
      for (int j0 = j1 + 64; j0 < j2; j0 += 32)
        products(load_weights((int)std::min(at + l, N - 1), j0), j0 - j1, acc);
      // (Before this block's stores: what comes behind them is waited for with them.)
      Block next = v;
      if (at + 128 < last) load_both(at + 128);
      if (at + 160 <= last) next = load_base(from, at + 128);
      const int64_t n = at + part4;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 16; e++) turn[(8 * (e / 4) + 4 * hi + e % 4) * kTurn + l] = acc[u][e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (at + 32 <= last) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int r = 32 * u + r8 + 8 * i;
            const f32x4 s = v.v[4 * u + i] + *reinterpret_cast<const f32x4 *>(turn + (r8 + 8 * i) * kTurn + part4);
            if (r < tile.count)
              *reinterpret_cast<Four *>(y + row_of[r] + n) = Four{{s[0], s[1], s[2], s[3]}};
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 16; i++) {
            const int r = 32 * u + 2 * i + hi;
            const int64_t e = row_of[r] + at + l;
            if (r < tile.count && at + l < last) y[e] = from[e] + turn[(2 * i + hi) * kTurn + l];
          }
        }
      }
      v = next;
    }
  }
}

int64_t most_tiles(const mg_adapters &h, int64_t rows) {
  return rows / kTile + std::min<int64_t>(h.slots + 2, rows);
}
// The share of K of a workgroup: as many as are at work together (four a CU), 256 at least.
int64_t k_share(const mg_ctx *ctx, const mg_adapters &h, int64_t rows, int *parts) {
  const int64_t groups = (rows + kTile - 1) / kTile * ((h.n * h.max_rank + kCols - 1) / kCols);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(4 * ctx->num_cus / groups, h.kp / 256));
  const int64_t share = ((h.kp + want - 1) / want + 127) / 128 * 128;
  *parts = (int)((h.kp + share - 1) / share);
  return share;
}

// The outputs of a workgroup: so many that its start (its rows and their values) costs little, so
// few that there are workgroups enough (three a CU at work together).
int64_t up_outs(const mg_ctx *ctx, const mg_adapters &h, int64_t rows) {
  int64_t all = 0;
  for (int i = 0; i < h.n; i++) all += (h.N[i] + 127) / 128;
  const int64_t blocks = (rows + kTile - 1) / kTile * all / (3 * ctx->num_cus);
  return 128 * std::max<int64_t>(2, std::min<int64_t>(blocks, 8));
}

template <class T>
void run(mg_ctx *ctx, const mg_adapt &p, void *ws) {
  const mg_adapters &h = p.h;
  hipStream_t st = ctx->stream;
  const unsigned rows = (unsigned)p.rows;
  int64_t most = 0;
  for (int i = 0; i < h.n; i++) most = std::max(most, h.N[i]);
  if (few_rows(h, p.rows)) {
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
  const int64_t outs = up_outs(ctx, h, p.rows);
  int64_t chunks = 0;
  for (int i = 0; i < h.n; i++) chunks += (h.N[i] + outs - 1) / outs;
  k_up<T><<<dim3((unsigned)chunks, (unsigned)tiles), dim3(256),
            (size_t)kTile * stride * 4, st>>>(p, o, t, parts, cols, stride, (int)outs);
}

}  // namespace

int64_t mg_adapt_groups(const mg_adapters &h, int64_t rows) {
  int64_t most = 0;
  for (int i = 0; i < h.n; i++) most = std::max(most, h.N[i]);
  return most_tiles(h, std::min(rows, MG_ADAPT_ROWS)) * ((most + kOuts - 1) / kOuts) * h.n;
}

static size_t round_ws(const mg_ctx *ctx, const mg_adapters &h, int64_t rows) {
  const size_t cols = (size_t)h.n * h.max_rank;
  if (few_rows(h, rows)) return mg_align((size_t)rows * cols * 4);
  int parts;
  k_share(ctx, h, rows, &parts);
  return mg_align((size_t)rows * 4) + 256 + mg_align((size_t)most_tiles(h, rows) * sizeof(Tile)) +
         mg_align((size_t)parts * rows * cols * 4);
}
size_t mg_adapt_ws(const mg_ctx *ctx, const mg_adapters &h, int64_t rows) {
  // (The last round's rows are fewer, the parts of their K more.)
  const size_t last = round_ws(ctx, h, rows % MG_ADAPT_ROWS);
  return rows < MG_ADAPT_ROWS ? last : std::max(last, round_ws(ctx, h, MG_ADAPT_ROWS));
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
  Fill f{h, {}, {}, slot, (int)rank, factor};
  int64_t most = h.kp;
  for (int i = 0; i < h.n; i++) {
    f.a[i] = rank ? a[i] : nullptr;
    f.b[i] = rank ? b[i] : nullptr;
    most = std::max(most, h.np[i]);
  }
  const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, 64), (unsigned)std::max<int64_t>(1, (rank + 31) / 32 * 32),
                  (unsigned)(2 * h.n));
  if (h.fmt == MG_ADAPTER_F16)
    k_fill<_Float16><<<grid, dim3(256), 0, ctx->stream>>>(f);
  else
    k_fill<float><<<grid, dim3(256), 0, ctx->stream>>>(f);
  return mg_launch_check("Adapters fill");
}

mg_status mg_adapters_clear(mg_ctx *ctx, const mg_adapters &h) {
  k_empty<<<dim3((unsigned)((h.slots + 255) / 256)), dim3(256), 0, ctx->stream>>>(h.rank, h.factor, h.slots);
  return mg_launch_check("Adapters clear");
}
