// paged_rows.cuh — the row work around attention for many requests at once: RMSNorm of
// each head of q and k, split-half rotation, and the append of k and v to a paged cache.
//
// Per head row x[D] of a token at position p, with r rotated pairs (r <= D/2):
//   y_d = gamma_d * x_d / sqrt(mean(x^2) + eps)                      (with a gamma)
//   o_d = y_d cos[p][d] - y_{d+r} sin[p][d]                          (d < r)
//   o_{d+r} = y_{d+r} cos[p][d] + y_d sin[p][d]
//   o_d = y_d                                                        (2r <= d < D)
// (rms_norm_f16 and apply_rope_raw of src/gemv.rs:744-778, per head), in f32 with one
// rounding at the end.
//
// Every byte is read once and written once, so the kernel is a copy that computes on the
// way: a lane holds one 16-byte piece of the lower half of a head row and the piece it is
// rotated with, so the rotation needs no exchange; D/2 elements / piece = 4, 8 or 16 lanes
// make a head row (the norm's sum is 2-4 shuffles), 2 to 8 head rows a warp. A warp walks
// over a token's head rows with one angle, the next ones' loads under way while it computes;
// with few tokens their head rows are spread over more warps.
//
// Measured: norm and rotation of 8,191 bf16 rows of 16 + 4 heads of 128, 88 MB, in 20.5 us =
// 4.3 TB/s; a warp per head row took 36.9 us, a deeper prefetch and other numbers of blocks
// per SM were slower. The append of 5 bf16 prompts, 94 MB, 22.7 us. A plain copy that moves as
// many bytes takes 20.4 and 22.6 us (buffers beyond L2, one call after the other): it is the
// size that keeps these from the bandwidth of long copies. One row: 2.6 us in a graph.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace qora {
namespace paged {

// ---------------------------------------------------------------- element types
template <typename T>
struct Elem;  // kVec: elements of a 16-byte piece
template <>
struct Elem<float> {
  static constexpr int kVec = 4;
};
template <>
struct Elem<__half> {
  static constexpr int kVec = 8;
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kVec = 8;
};

QORA_DEV void unpack(const uint4& u, float (&x)[4], float) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
QORA_DEV void unpack(const uint4& u, float (&x)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
QORA_DEV void unpack(const uint4& u, float (&x)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

QORA_DEV float from_f32(float v, float) { return v; }
QORA_DEV __half from_f32(float v, __half) { return __float2half_rn(v); }
QORA_DEV __nv_bfloat16 from_f32(float v, __nv_bfloat16) { return __float2bfloat16_rn(v); }
QORA_DEV float to_f32(float v) { return v; }
QORA_DEV float to_f32(__half v) { return __half2float(v); }
QORA_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// N consecutive elements, rounded to nearest even (binary16 beyond +-65504: infinity)
template <int N>
QORA_DEV void store_elems(float* p, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <int N, typename T>
QORA_DEV void store_elems(T* p, const float (&x)[N]) {
  static_assert(sizeof(T) == 2 && (N == 4 || N == 8), "16-bit pieces");
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const T a = from_f32(x[2 * i], T()), b = from_f32(x[2 * i + 1], T());
    w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&a) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&b) << 16);
  }
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// ---------------------------------------------------------------- the batch's layout
// One layer's pages: element (page, head, slot, d) at page * page_stride + head *
// head_stride + slot * slot_stride + d (elements, 64-bit).
struct Pages {
  int num_pages, page_size;
  long long page_stride, head_stride, slot_stride;
};

// Sequence s owns rows [q_start[s], q_start[s+1]), its newest positions; kv_len[s]
// positions in all; position p lies in page table[s * table_stride + p / page_size].
struct Batch {
  const int* q_start;
  const int* kv_len;
  const int* table;
  int table_stride, seqs, rows;
};

// The sequence that owns `row`: the last one whose first row is not behind it, found by
// the whole warp, 32 probes at a time (one round of loads up to 32 sequences, two up to
// 1024). Returns seqs or -1 when none does; any contents of q_start keep it in bounds.
QORA_DEV int find_seq(const Batch& b, int row, int lane) {
  int lo = 0, span = b.seqs + 1;  // q_start[lo .. lo + span): the answer is the last <= row
  int found = -1;
  while (span > 0) {
    const int step = (span + 31) / 32;
    const int i = lo + lane * step;
    const bool le = i < lo + span && b.q_start[i] <= row;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    if (!m) break;
    const int k = 31 - __clz(m);
    found = lo + k * step;
    if (step == 1) break;
    const int end = lo + span;
    lo = found;
    span = min(step, end - lo);
  }
  return found;
}

constexpr int kRowWarps = 8;

struct RowArgs {
  const void *q, *k, *v;
  long long q_stride, k_stride, v_stride;  // elements from one row to the next
  int rows, hq, hk, hv;                    // hv: 0 (no append) or hk
  const float *q_gamma, *k_gamma;          // [D] or null (no norm)
  float eps;
  int per_warp;                            // groups of head rows that a warp walks over
  const int* pos;                          // [rows] without a cache; with one, from the batch
  const float *cos_t, *sin_t;              // [rope_rows][r] or null (no rotation)
  int rope_rows, r;
  void *q_out, *k_out;                     // rows (no append: k_out too)
  long long qo_stride, ko_stride;
  void *k_pages, *v_pages;
  Pages pg;
  Batch batch;
  unsigned* status;                        // set to QORA_ERR_RANGE (5) where a row has no place; may be null
};

// T: rows, C: where k and v go (the rows' type, or the cache's). kAppend: k and v go to
// pages.
template <typename T, typename C, int D, bool kAppend>
__global__ void __launch_bounds__(32 * kRowWarps, 4) rows_kernel(const RowArgs a) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kLanes = D / 2 / V;     // lanes of a head row
  constexpr int kHeads = 32 / kLanes;   // head rows a warp holds at once: a group
  const int lane = threadIdx.x & 31;
  const int heads = a.hq + a.hk + a.hv, groups = (heads + kHeads - 1) / kHeads;
  const int parts = (groups + a.per_warp - 1) / a.per_warp;
  const unsigned unit = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int row = (int)(unit / parts), part = (int)(unit % parts);
  if (row >= a.rows) return;
  const int sub = lane % kLanes;
  const int e = sub * V;  // index of the lane's first pair
  const bool turned = e < a.r;
  const int lower = turned ? e : a.r + e;  // pairs past r: the untouched rest, split in halves
  const int upper = lower + (turned ? a.r : D / 2 - a.r);
  const int first = part * a.per_warp, last = min(groups, first + a.per_warp);

  uint4 lo, hi;
  auto load = [&](int it) {
    const int h = it * kHeads + lane / kLanes;
    lo = hi = make_uint4(0, 0, 0, 0);
    if (h < heads) {
      const T* src;
      if (h < a.hq)
        src = static_cast<const T*>(a.q) + row * a.q_stride + h * D;
      else if (h < a.hq + a.hk)
        src = static_cast<const T*>(a.k) + row * a.k_stride + (h - a.hq) * D;
      else
        src = static_cast<const T*>(a.v) + row * a.v_stride + (h - a.hq - a.hk) * D;
      lo = *reinterpret_cast<const uint4*>(src + lower);
      hi = *reinterpret_cast<const uint4*>(src + upper);
    }
  };
  load(first);  // nothing it needs depends on the position

  // where the row sits
  int p = 0;
  long long slot = -1;  // offset of (page, slot); -1: no place
  if constexpr (kAppend) {
    const int s = find_seq(a.batch, row, lane);
    if (s < 0 || s >= a.batch.seqs) return;  // behind the last sequence: left as it was
    const int q0 = a.batch.q_start[s], q1 = a.batch.q_start[s + 1], len = a.batch.kv_len[s];
    if (q0 < 0 || row >= q1 || q1 > a.rows) {
      if (lane == 0 && a.status) *a.status = 5u;
      return;
    }
    const long long pl = (long long)len - (q1 - q0) + (row - q0);
    if (pl < 0 || len > (long long)a.batch.table_stride * a.pg.page_size) {  // pl < len
      if (lane == 0 && a.status) *a.status = 5u;
      return;
    }
    p = (int)pl;
    const int pi = p / a.pg.page_size;
    const int page = a.batch.table[(long long)s * a.batch.table_stride + pi];
    if (page >= 0 && page < a.pg.num_pages)
      slot = page * a.pg.page_stride + (long long)(p - pi * a.pg.page_size) * a.pg.slot_stride;
    else if (lane == 0 && a.status)
      *a.status = 5u;
  } else if (a.pos) {
    p = a.pos[row];
    if (p < 0) return;  // a padding row
  }
  float cs[V], sn[V];
  if (a.cos_t) {
    if (p >= a.rope_rows) {
      if (lane == 0 && a.status) *a.status = 5u;
      return;
    }
    if (turned) {
      const float* c = a.cos_t + (long long)p * a.r + e;
      const float* s = a.sin_t + (long long)p * a.r + e;
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(c + i)), s4 = __ldg(reinterpret_cast<const float4*>(s + i));
        cs[i] = c4.x, cs[i + 1] = c4.y, cs[i + 2] = c4.z, cs[i + 3] = c4.w;
        sn[i] = s4.x, sn[i + 1] = s4.y, sn[i + 2] = s4.z, sn[i + 3] = s4.w;
      }
    }
  }

#pragma unroll 1
  for (int it = first; it < last; ++it) {
    const int h = it * kHeads + lane / kLanes;
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hk;
    float x[V], y[V];
    unpack(lo, x, T());
    unpack(hi, y, T());
    if (it + 1 < last) load(it + 1);
    const float* g = is_v ? nullptr : is_q ? a.q_gamma : a.k_gamma;
    if (a.q_gamma || a.k_gamma) {  // the same for the whole warp: the shuffles need every lane
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) ss = __fmaf_rn(x[i], x[i], __fmaf_rn(y[i], y[i], ss));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
      if (g && h < heads) {
        const float inv = rsqrtf(__fadd_rn(__fmul_rn(ss, 1.0f / D), a.eps));
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const float4 gl = __ldg(reinterpret_cast<const float4*>(g + lower + i));
          const float4 gu = __ldg(reinterpret_cast<const float4*>(g + upper + i));
          x[i] = __fmul_rn(__fmul_rn(x[i], inv), gl.x), x[i + 1] = __fmul_rn(__fmul_rn(x[i + 1], inv), gl.y);
          x[i + 2] = __fmul_rn(__fmul_rn(x[i + 2], inv), gl.z), x[i + 3] = __fmul_rn(__fmul_rn(x[i + 3], inv), gl.w);
          y[i] = __fmul_rn(__fmul_rn(y[i], inv), gu.x), y[i + 1] = __fmul_rn(__fmul_rn(y[i + 1], inv), gu.y);
          y[i + 2] = __fmul_rn(__fmul_rn(y[i + 2], inv), gu.z), y[i + 3] = __fmul_rn(__fmul_rn(y[i + 3], inv), gu.w);
        }
      }
    }
    if (a.cos_t && turned && !is_v) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = __fsub_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(y[i], sn[i]));
        y[i] = __fadd_rn(__fmul_rn(y[i], cs[i]), __fmul_rn(x[i], sn[i]));
        x[i] = u;
      }
    }
    if (h >= heads) continue;
    if (is_q) {
      T* dst = static_cast<T*>(a.q_out) + row * a.qo_stride + h * D;
      store_elems(dst + lower, x);
      store_elems(dst + upper, y);
    } else if constexpr (kAppend) {
      if (slot < 0) continue;
      C* dst = static_cast<C*>(is_v ? a.v_pages : a.k_pages) + slot +
               (long long)(is_v ? h - a.hq - a.hk : h - a.hq) * a.pg.head_stride;
      store_elems(dst + lower, x);
      store_elems(dst + upper, y);
    } else {
      C* dst = static_cast<C*>(a.k_out) + row * a.ko_stride + (h - a.hq) * D;
      store_elems(dst + lower, x);
      store_elems(dst + upper, y);
    }
  }
}

}  // namespace paged
}  // namespace qora
