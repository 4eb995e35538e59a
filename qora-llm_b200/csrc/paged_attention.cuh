// paged_attention.cuh — causal attention of each sequence's newest rows over its paged
// cache:
//   s_j = scale * q . k_j,  max(0, p + 1 - window) <= j <= p   (p: the row's position)
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log(sum_j exp(s_j - m))
// A row that attends to nothing gets out = 0 and lse = -inf.
#pragma once

#include "common.cuh"
#include "paged_rows.cuh"

namespace qora {
namespace paged {

struct AttnArgs {
  const void* q;
  long long q_stride;
  void* out;
  long long out_stride;
  float* lse;  // [rows][hq] or null
  const void *k_pages, *v_pages;
  Pages pg;
  Batch batch;
  int hq, hk, group;  // group = hq / hk
  int group_inv;      // ceil(2^16 / group)
  int window;         // 0: none
  int max_q;          // no sequence has more new rows
  int few;            // new rows up to which a sequence is the token kernel's, not the chunk kernel's
  float scale;
  unsigned* status;
};

// token of packed row r (< 128) of a tile: r / group
QORA_DEV int token_of(const AttnArgs& a, int r) { return (r * a.group_inv) >> 16; }

// The first position that a row at position p attends to. p may be negative (more new rows
// than positions), the window up to 2^31 - 1.
QORA_DEV int first_seen(const AttnArgs& a, int p) { return a.window > 0 ? max(0, max(p, -1) + 1 - a.window) : 0; }

}  // namespace paged
}  // namespace qora
