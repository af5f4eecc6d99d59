// Verification of drafted tokens: the problem as api.hip hands it to verify.hip.
#pragma once

#include "mg_internal.h"

constexpr int MG_DRAFTS_MOST = 1024;  // rows of a sequence
constexpr int MG_DRAFTS_RUN = 2048;   // logits that a wave takes

// A run of a row's logits: its maximum (+inf: it holds NaN or +inf) and sum 2^((x - m) c).
struct mg_drafts_part {
  double s;
  float m, unused;
};
// Where a sequence's last token is drawn, and by what.
struct mg_drafts_last {
  double s, qs, c, u;  // 1 / the sums of p's and q's row, log2(e) / temperature, the random number
  float m, qm;         // maxima of the rows
  int64_t row;
  int32_t mode;     // 0: it is drawn already; 1: by p without the rejected tokens; 2: max(p - q, 0)
  int32_t rejected; // tokens
  int32_t out;      // row that the token goes to
};
struct mg_verify {
  mg_drafts d;
  int32_t *out, *kept, *count;
  int nrun;  // runs of a row
  // Workspace: parts [rows][nrun]; with draft logits as many again, masses [batch][nrun] and lasts
  // [batch].
  mg_drafts_part *part;
  double *mass;
  mg_drafts_last *last;
};
// Workgroups of the largest launch of a call (of 256 threads; those of 1024 are one a sequence).
int64_t mg_verify_groups(const mg_drafts &d);
// The workspace of a problem (its pointers set from ws, where not null).
size_t mg_verify_plan(mg_verify *v, void *ws);
mg_status mg_verify_run(mg_ctx *ctx, const mg_verify &v);
