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
  float scale;
  unsigned* status;
};

// One warp per (row, query head), one position at a time.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(256) attn_row_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = (int)(unit / a.hq), h = (int)(unit % a.hq);
  if (row >= a.batch.rows) return;
  const int s = find_seq(a.batch, row, lane);
  if (s < 0 || s >= a.batch.seqs) return;
  const int q0 = a.batch.q_start[s], q1 = a.batch.q_start[s + 1], len = a.batch.kv_len[s];
  const long long cap = (long long)a.batch.table_stride * a.pg.page_size;
  if (q0 < 0 || row >= q1 || q1 > a.batch.rows || q1 - q0 > a.max_q || len < 0 || len > cap) {
    if (lane == 0 && a.status) *a.status = 5u;
    return;
  }
  const int p = len - (q1 - q0) + (row - q0);
  const int first = a.window > 0 ? max(0, p + 1 - a.window) : 0;
  const T* q = static_cast<const T*>(a.q) + row * a.q_stride + h * D;
  float qv[E], o[E];
  for (int i = 0; i < E; ++i) {
    qv[i] = to_f32(q[lane + 32 * i]);
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const long long hoff = (long long)(h / a.group) * a.pg.head_stride;
  for (int j = first; j <= p; ++j) {
    const int pi = j / a.pg.page_size;
    const int page = a.batch.table[(long long)s * a.batch.table_stride + pi];
    if (page < 0 || page >= a.pg.num_pages) {
      if (lane == 0 && a.status) *a.status = 5u;
      continue;
    }
    const long long off = page * a.pg.page_stride + (long long)(j - pi * a.pg.page_size) * a.pg.slot_stride + hoff;
    const C* k = static_cast<const C*>(a.k_pages) + off;
    const C* v = static_cast<const C*>(a.v_pages) + off;
    float d = 0.0f;
    for (int i = 0; i < E; ++i) d = __fmaf_rn(qv[i], to_f32(k[lane + 32 * i]), d);
    d = __fmul_rn(warp_sum(d), a.scale);
    const float mn = fmaxf(m, d);
    const float mu = mn == -INFINITY ? 0.0f : mn;  // a NaN score does not raise the maximum: its weight is NaN
    const float w = expf(d - mu), c = expf(m - mu);
    l = __fmaf_rn(l, c, w);
    for (int i = 0; i < E; ++i) o[i] = __fmaf_rn(o[i], c, w == 0.0f ? 0.0f : __fmul_rn(w, to_f32(v[lane + 32 * i])));
    m = mn;
  }
  const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
  T* out = static_cast<T*>(a.out) + row * a.out_stride + h * D;
  for (int i = 0; i < E; ++i) out[lane + 32 * i] = from_f32(__fmul_rn(o[i], inv), T());
  if (a.lse && lane == 0) a.lse[(long long)row * a.hq + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace paged
}  // namespace qora
