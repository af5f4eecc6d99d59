// Low-rank adapters of many requests: their memory, and the problem as api.hip hands it to
// adapters.hip.
#pragma once

#include "mg_internal.h"

constexpr int MG_ADAPTER_MOST = 4;  // projections of a handle
constexpr int64_t MG_ADAPTER_SLOTS = 4096;

// Values are fp32 or fp16; per slot A [projection][rank][kp] and, per projection, B transposed
// [rank][np] (so that neighbouring outputs are neighbours), K and N padded to multiples of 8 with
// zeros.  Beyond a slot's own rank A's rows hold anything; B has room for ranks up to a multiple
// of 32, and zeros up to the one that the slot's own reaches.
struct mg_adapters {
  int device = 0, fmt = 0, n = 0, max_rank = 0;
  int64_t K = 0, kp = 0, slots = 0, bytes = 0;
  int64_t N[MG_ADAPTER_MOST] = {}, np[MG_ADAPTER_MOST] = {}, b_off[MG_ADAPTER_MOST] = {};
  int64_t a_slot = 0, b_slot = 0;  // values of a slot
  void *a = nullptr, *b = nullptr;
  int32_t *rank = nullptr;  // [slots]
  float *factor = nullptr;  // [slots]
};

struct mg_adapt {
  mg_adapters h;
  const float *x;
  const int32_t *slot;
  const float *base[MG_ADAPTER_MOST];
  float *y[MG_ADAPTER_MOST];
  int64_t rows;
};
// Most rows of one round of launches.
constexpr int64_t MG_ADAPT_ROWS = 65536;
// The largest launch of a call (workgroups), its workspace, and its launches (p.rows at most MG_ADAPT_ROWS).
int64_t mg_adapt_groups(const mg_adapters &h, int64_t rows);
size_t mg_adapt_ws(const mg_ctx *ctx, const mg_adapters &h, int64_t rows);
mg_status mg_adapt_run(mg_ctx *ctx, const mg_adapt &p, void *ws);
// Fills a slot from device memory.
mg_status mg_adapters_fill(mg_ctx *ctx, const mg_adapters &h, int64_t slot, int64_t rank,
                           const float *const *a, const float *const *b, float factor);
mg_status mg_adapters_clear(mg_ctx *ctx, const mg_adapters &h);
