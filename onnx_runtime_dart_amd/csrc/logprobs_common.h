// Log probabilities: the problem as api.hip hands it to logprobs.hip.
#pragma once

#include "mg_internal.h"

constexpr int MG_LOGPROBS_MAX_TOP = 64;

// A run of a row: its maximum, sums and largest entries.
struct mg_logprobs_part {
  double s, a;
  float m;
  uint32_t key[MG_LOGPROBS_MAX_TOP];
  int32_t id[MG_LOGPROBS_MAX_TOP];
};
struct mg_logprobs {
  const float *x;
  const int32_t *tokens;
  float *logprob, *entropy, *lps;
  int32_t *ids;
  int64_t rows, stride;
  int vocab, top;
  // The plan: runs of `run` logits a row, and their parts.
  int nsplit, run;
  mg_logprobs_part *part;
};
size_t mg_logprobs_plan(const mg_ctx *ctx, mg_logprobs *p, bool split);
mg_status mg_logprobs_run(mg_ctx *ctx, const mg_logprobs &p);
