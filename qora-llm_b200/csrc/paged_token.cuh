// paged_token.cuh — attention of a few rows per sequence (one new token, or a few) over its
// paged cache. The time is the K and V bytes of the attended positions, read once.
//
// Tile. A tile is one (sequence, kv head): its rows are the sequence's new tokens times the
// kv head's query heads, packed (row r: token r / group, head r % group), at most kRows of
// them (longer ones: several tiles that share the positions through L2). kRows is what one
// m16 matrix instruction holds: 16 rows of 16-bit q, or 8 rows of f32 q, whose binary16
// (tf32, for an f32 cache) upper and lower halves are the instruction's rows 0-7 and 8-15:
// the 22 bits cost no second instruction. An f32 cache is split likewise into two operands.
//
// Work split. The steps (kPos positions) of all tiles form one line, cut into gridDim.x
// equal runs: every CTA reads the same number of bytes whatever the lengths are, and one
// request with a long cache fills the GPU as a batch does. The lengths are in device
// memory, so each CTA finds its run itself (a scan of the sequences' step counts). A tile
// that is cut is written as partials (numerators, maximum, sum) and joined in CTA order by
// join_kernel, which is launched behind with its launch overlapped; every tile cut begins in
// a different CTA, so the workspace has a fixed size and needs no initial contents.
//
// Inside a CTA every warp takes every kWarps-th step of a segment with its own ring of
// cp.async stages, running maximum and sum; there is no barrier until the segment's end.
// The maximum is only raised (and the numerators rescaled) when it grows by more than
// 2^kSlack, so weights stay below 2^(kShift + kSlack) <= 2^15, within binary16.
//
// Values that are masked never count: masked scores become -inf, slots behind the last
// position are filled with zeros. What a weight of zero times an infinite value leaves (NaN)
// shows in the numerators; such a segment is run again with the non-finite elements of V
// taken out and added to the rows that do see them.
#pragma once

#include "paged_attention.cuh"

namespace qora {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kShift = 7.0f;  // weights are 2^(x - m + kShift): small ones stay normal in binary16
constexpr float kSlack = 8.0f;

QORA_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

QORA_DEV void cp_async_16(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
QORA_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
QORA_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

QORA_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
QORA_DEV void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

QORA_DEV void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
QORA_DEV void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
QORA_DEV void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

QORA_DEV uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
QORA_DEV uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// x rounded to the 11 bits of tf32, and what that leaves (exact, at most 2^-11 of x; the
// instruction cuts it to 11 bits: 2^-22 of x are lost)
QORA_DEV uint32_t tf32_hi(float x) { return (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u; }
QORA_DEV uint32_t tf32_lo(float x) { return __float_as_uint(__fsub_rn(x, __uint_as_float(tf32_hi(x)))); }

template <typename T, typename C, int D>
struct TokenCfg {
  static constexpr bool kWide = sizeof(C) == 4;     // f32 cache
  static constexpr bool kHalves = sizeof(T) == 4;   // f32 rows: upper and lower halves
  static constexpr int kRows = kHalves ? 8 : 16;
  static constexpr int kPos = kWide ? 8 : 16;       // positions of a step
  static constexpr int kChunks = D * (int)sizeof(C) / 16;  // 16-byte pieces of a K or V row
  static constexpr int kSide = kPos * kChunks * 16;        // bytes of a step's K (or V)
  static constexpr int kStages = 3;
  static constexpr int kWarps = 8;
  static constexpr int kRing = kStages * 2 * kSide;  // bytes of a warp's ring
  static constexpr int kStage_ = kRows * D * 4;      // a warp's numerators at a segment's end, in its ring
  static_assert(kStage_ <= kRing, "the ring holds the numerators");
  static constexpr int kSmem = kWarps * kRing;
};

constexpr int kTokenMaxCtas = 320;
constexpr int kTokenMaxRows = 16;

// Workspace: records [ctas], partial maxima and sums [2 ctas][16], numerators [2 ctas][16][D].
struct TokenWork {
  int4* rec;    // (sequence, tile of the sequence, contributors, slot of the first), contributors 0: none
  float2* ml;
  float* num;
};
__host__ __device__ inline TokenWork token_work(void* p, int ctas) {
  char* c = static_cast<char*>(p);
  TokenWork w;
  w.rec = reinterpret_cast<int4*>(c);
  w.ml = reinterpret_cast<float2*>(c + (size_t)kTokenMaxCtas * 16);
  w.num = reinterpret_cast<float*>(c + (size_t)kTokenMaxCtas * 16 + (size_t)2 * kTokenMaxCtas * kTokenMaxRows * 8);
  return w;
}

// One sequence's share of the line of steps.
struct SeqWork {
  int q0, n, len, first;  // first row, new rows, positions, first step's position
  int steps, tiles;       // steps of a tile; tiles (row tiles x kv heads)
};
template <int kPos>
QORA_DEV SeqWork seq_work(const AttnArgs& a, int s, int rows_per_tile) {
  SeqWork w;
  w.q0 = a.batch.q_start[s];
  const int q1 = a.batch.q_start[s + 1];
  w.len = a.batch.kv_len[s];
  w.n = q1 - w.q0;
  w.first = w.steps = w.tiles = 0;
  const long long cap = (long long)a.batch.table_stride * a.pg.page_size;
  if (w.q0 < 0 || q1 < w.q0 || q1 > a.batch.rows || w.n > a.max_q || w.len < 0 || w.len > cap) {
    if (a.status) *a.status = 5u;
    return w;
  }
  if (w.n == 0) return w;
  const int lo = a.window > 0 ? max(0, w.len - w.n + 1 - a.window) : 0;
  w.first = lo / kPos * kPos;
  w.steps = max(1, (w.len - w.first + kPos - 1) / kPos);
  w.tiles = (w.n * a.group + rows_per_tile - 1) / rows_per_tile * a.hk;
  return w;
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(32 * TokenCfg<T, C, D>::kWarps, 1) token_kernel(const AttnArgs a, void* work, int min_steps) {
  using Cfg = TokenCfg<T, C, D>;
  constexpr int kPos = Cfg::kPos, kRows = Cfg::kRows, kWarps = Cfg::kWarps, kChunks = Cfg::kChunks, kStages = Cfg::kStages;
  constexpr bool kWide = Cfg::kWide, kHalves = Cfg::kHalves;
  constexpr int kThr = 32 * kWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_scan[kWarps];
  __shared__ long long s_total, s_base;
  __shared__ int s_seq;
  __shared__ float2 s_ml[kWarps][kRows];
  __shared__ uint32_t s_bad[kWarps][kStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const TokenWork ws = token_work(work, gridDim.x);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run of the line
  long long mine = 0;
  for (int s = tid; s < a.batch.seqs; s += kThr) {
    const SeqWork w = seq_work<kPos>(a, s, kRows);
    mine += (long long)w.steps * w.tiles;
  }
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_scan[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    long long x = 0;
    for (int w = 0; w < kWarps; ++w) x += s_scan[w];
    s_total = x;
    s_seq = a.batch.seqs;
  }
  __syncthreads();
  const long long total = s_total;
  // no more CTAs than leave min_steps each: a smaller share costs more to join than it saves
  const long long ctas = max(1LL, min((long long)gridDim.x, (total + min_steps - 1) / min_steps));
  const long long c = blockIdx.x;
  if (tid == 0) ws.rec[c] = make_int4(0, 0, 0, 0);
  if (c >= ctas) return;
  long long cur = c * total / ctas;
  const long long end = (c + 1) * total / ctas;
  if (cur >= end) return;
  {  // the sequence that holds step `cur`: scan in chunks of the CTA's threads
    long long base = 0;
    for (int s0 = 0; s0 < a.batch.seqs; s0 += kThr) {
      const int s = s0 + tid;
      long long v = 0;
      if (s < a.batch.seqs) {
        const SeqWork w = seq_work<kPos>(a, s, kRows);
        v = (long long)w.steps * w.tiles;
      }
      long long x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      long long before = base;
      for (int w = 0; w < warp; ++w) before += s_scan[w];
      long long all = base;
      for (int w = 0; w < kWarps; ++w) all += s_scan[w];
      if (v > 0 && before + x - v <= cur && cur < before + x) {
        s_seq = s;
        s_base = before + x - v;
      }
      __syncthreads();
      base = all;
      if (cur < base) break;
    }
  }
  int seq = s_seq;
  long long base = s_base;
  SeqWork sw = seq_work<kPos>(a, seq, kRows);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * Cfg::kRing);
  const float scale2 = a.scale * kLog2e;
  const bool pow2 = (a.pg.page_size & (a.pg.page_size - 1)) == 0;
  const int shift = 31 - __clz(a.pg.page_size);
  bool first_seg = true;

  while (cur < end) {
    while (cur >= base + (long long)sw.steps * sw.tiles) {  // the next sequence with work
      base += (long long)sw.steps * sw.tiles;
      if (++seq >= a.batch.seqs) return;
      sw = seq_work<kPos>(a, seq, kRows);
    }
    const long long in = cur - base;
    const int tile = (int)(in / sw.steps), st0 = (int)(in % sw.steps);
    const int st1 = (int)min((long long)sw.steps, st0 + (end - cur));
    const int head = tile % a.hk, row0 = tile / a.hk * kRows;  // first packed row
    const int nrows = min(kRows, sw.n * a.group - row0);
    const int p0 = sw.len - sw.n;
    const int* table = a.batch.table + (long long)seq * a.batch.table_stride;
    const C* kbase = static_cast<const C*>(a.k_pages) + head * a.pg.head_stride;
    const C* vbase = static_cast<const C*>(a.v_pages) + head * a.pg.head_stride;

    // positions the thread's rows see
    int plast[2], pfirst[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i;
      const bool ok = (!kHalves || i == 0) && r < nrows;
      plast[i] = ok ? p0 + (row0 + r) / a.group : -1;
      pfirst[i] = a.window > 0 ? max(0, plast[i] + 1 - a.window) : 0;
    }
    const int seen_to = p0 + row0 / a.group;                       // every row sees up to here
    const int top = p0 + (row0 + nrows - 1) / a.group;
    const int seen_from = a.window > 0 ? max(0, top + 1 - a.window) : 0;  // and from here

    // offset of position `pos` in the pages; -1: nothing there
    auto page_of = [&](int pos) -> int {
      if (pos >= sw.len) return -1;
      return table[pow2 ? pos >> shift : pos / a.pg.page_size];
    };
    auto offset_of = [&](int pos, int page) -> long long {
      if (page < 0 || page >= a.pg.num_pages) return -1;
      const int slot = pow2 ? pos & (a.pg.page_size - 1) : pos % a.pg.page_size;
      return page * a.pg.page_stride + (long long)slot * a.pg.slot_stride;
    };
    auto issue = [&](int step, int stage, int page) {  // page: of position step * kPos + lane
      const int pos = sw.first + step * kPos + (lane & (kPos - 1));
      const long long off = offset_of(pos, page);
      const unsigned bad = __ballot_sync(0xffffffffu, off < 0 && lane < kPos);
      if (lane == 0) {
        s_bad[warp][stage] = bad;
        if (a.status)  // a page that does not exist, unlike a slot behind the last position
          for (unsigned b = bad; b; b &= b - 1)
            if (pos + __ffs(b) - 1 < sw.len) *a.status = 5u;
      }
      const uint32_t dk = ring + stage * 2 * Cfg::kSide, dv = dk + Cfg::kSide;
#pragma unroll
      for (int i = 0; i < kPos * kChunks / 32; ++i) {
        const int row = (i * 32) / kChunks + lane / kChunks, ch = lane % kChunks;
        const long long o = __shfl_sync(0xffffffffu, off, row);
        const long long at = (o < 0 ? 0 : o) + ch * (16 / (int)sizeof(C));
        const int ck = kWide ? ch ^ ((row & 1) << 2) : ch ^ (row & 7);
        const int cv = kWide ? ch ^ (row & 6) : ch ^ (row & 7);
        cp_async_16(dk + (row * kChunks + ck) * 16, kbase + at, o >= 0);
        cp_async_16(dv + (row * kChunks + cv) * 16, vbase + at, o >= 0);
      }
    };

    // q in the instruction's layout. f32 rows: 2^e puts the row's largest value in [2^13, 2^14)
    float qscale[2] = {scale2, scale2};
    constexpr int kQ = kWide ? D / 8 : D / 16;
    uint32_t qa[kQ][4];
    auto load_q = [&]() {
      auto row_ptr = [&](int r) {
        const int pr = row0 + r;
        return static_cast<const T*>(a.q) + (long long)(sw.q0 + pr / a.group) * a.q_stride + (head * a.group + pr % a.group) * D;
      };
      if constexpr (!kHalves) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool ok = g + 8 * i < nrows;
          const T* q = row_ptr(ok ? g + 8 * i : 0);
#pragma unroll
          for (int k = 0; k < kQ; ++k) {
            qa[k][i] = ok ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t) : 0u;
            qa[k][2 + i] = ok ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8 + 2 * t) : 0u;
          }
        }
      } else {
        const bool ok = g < nrows;
        const float* q = reinterpret_cast<const float*>(row_ptr(ok ? g : 0));
        if constexpr (kWide) {  // tf32: the exponent range is f32's, no scale
#pragma unroll
          for (int b = 0; b < D / 16; ++b) {
            float4 x = *reinterpret_cast<const float4*>(q + 16 * b + 4 * t);
            if (!ok) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              qa[2 * b + (j >> 1)][2 * (j & 1)] = tf32_hi(e[j]);
              qa[2 * b + (j >> 1)][2 * (j & 1) + 1] = tf32_lo(e[j]);
            }
          }
        } else {
          float2 x[2 * kQ];
          float mx = 0.0f;
#pragma unroll
          for (int k = 0; k < 2 * kQ; ++k) {
            x[k] = *reinterpret_cast<const float2*>(q + 8 * k + 2 * t);
            if (!ok) x[k] = make_float2(0.0f, 0.0f);
            mx = fmaxf(mx, fmaxf(fabsf(x[k].x), fabsf(x[k].y)));
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // exponent of mx (0 for zeros and subnormals, 255 for non-finite rows: no scale)
          const int ex = (int)(__float_as_uint(mx) >> 23);
          const int up = ex == 0 || ex == 255 ? 0 : min(127, max(-126, 140 - ex));
          const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
          qscale[0] = scale2 * __uint_as_float((uint32_t)(127 - (up == 127 ? 126 : up)) << 23) * (up == 127 ? 0.5f : 1.0f);
#pragma unroll
          for (int k = 0; k < 2 * kQ; ++k) {
            const float u = x[k].x * mul, v = x[k].y * mul;
            const uint32_t hi = pack2(u, v, __half());
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            qa[k / 2][2 * (k & 1)] = hi;
            qa[k / 2][2 * (k & 1) + 1] = pack2(u - h.x, v - h.y, __half());
          }
        }
      }
    };

    constexpr int kO = D / 8;  // numerators: n8 tiles of 4 values
    float o[kO][4];
    float m[2], l[2];
    bool q_loaded = false;
    for (int careful = 0; careful < 2; ++careful) {
#pragma unroll
      for (int i = 0; i < kO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.0f;
      const int nst = st1 - st0 > warp ? (st1 - st0 - warp + kWarps - 1) / kWarps : 0;  // this warp's steps
      const int my0 = st0 + warp;
      auto next_page = [&](int i) { return i < nst ? page_of(sw.first + (my0 + i * kWarps) * kPos + (lane & (kPos - 1))) : -1; };
      int page = next_page(0);
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) {
        const int np = next_page(i + 1);
        if (i < nst) issue(my0 + i * kWarps, i, page);
        cp_async_commit();
        page = np;
      }
      if (!q_loaded) load_q();
      q_loaded = true;
      int stage = 0;
      for (int i = 0; i < nst; ++i) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        {  // refill the stage that the previous step left
          const int ns = stage == 0 ? kStages - 1 : stage - 1;
          const int np = next_page(i + kStages);
          if (i + kStages - 1 < nst) issue(my0 + (i + kStages - 1) * kWarps, ns, page);
          cp_async_commit();
          page = np;
        }
        const int pos0 = sw.first + (my0 + i * kWarps) * kPos;
        const uint32_t sk = ring + stage * 2 * Cfg::kSide, sv = sk + Cfg::kSide;
        const uint32_t bad = s_bad[warp][stage];
        if (careful) {  // non-finite elements of V become zero
          for (int x = lane; x < kPos * kChunks; x += 32) {
            uint4* p = reinterpret_cast<uint4*>(smem + warp * Cfg::kRing + stage * 2 * Cfg::kSide + Cfg::kSide) + x;
            uint4 v = *p;
            C* e = reinterpret_cast<C*>(&v);
            for (int y = 0; y < 16 / (int)sizeof(C); ++y)
              if (!isfinite(to_f32(e[y]))) e[y] = from_f32(0.0f, C());
            *p = v;
          }
          __syncwarp();
        }
        // scores
        constexpr int kN = kPos / 8;
        float s[kN][4];
        if constexpr (kWide) {
          float u[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int b = 0; b < D / 16; ++b) {
            const int ch = (4 * b + t) ^ ((g & 1) << 2);
            const float4 k = *reinterpret_cast<const float4*>(smem + warp * Cfg::kRing + stage * 2 * Cfg::kSide + (g * kChunks + ch) * 16);
            mma_tf32(u, qa[2 * b], tf32_hi(k.x), tf32_hi(k.y));
            mma_tf32(v, qa[2 * b], tf32_lo(k.x), tf32_lo(k.y));
            mma_tf32(u, qa[2 * b + 1], tf32_hi(k.z), tf32_hi(k.w));
            mma_tf32(v, qa[2 * b + 1], tf32_lo(k.z), tf32_lo(k.w));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) s[0][j] = u[j] + v[j];
        } else {
#pragma unroll
          for (int n = 0; n < kN; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
          const int mi = lane >> 3, row = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
          for (int k = 0; k < kQ; ++k) {
            uint32_t b[4];
            ldsm4(b, sk + (row * kChunks + ((2 * k + (mi & 1)) ^ (row & 7))) * 16);
            mma16(s[0], qa[k], b[0], b[1], C());
            mma16(s[1], qa[k], b[2], b[3], C());
          }
        }
        constexpr int kR = kHalves ? 1 : 2;
        if constexpr (kHalves) {
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            s[n][0] += s[n][2];
            s[n][1] += s[n][3];
          }
        }
        const bool plain = pos0 >= seen_from && pos0 + kPos - 1 <= seen_to && bad == 0;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int r = 0; r < kR; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float x = s[n][2 * r + j] * qscale[kHalves ? 0 : r];
              if (!plain) {
                const int w = 8 * n + 2 * t + j, pos = pos0 + w;
                if (pos > plast[r] || pos < pfirst[r] || ((bad >> w) & 1)) x = -INFINITY;
              }
              s[n][2 * r + j] = x;
              mx[r] = fmaxf(mx[r], x);
            }
        bool raise = false;
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
          mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
          raise |= mx[r] > m[r] + kSlack || (m[r] == -INFINITY && mx[r] > m[r]);
        }
        if (__any_sync(0xffffffffu, raise)) {
          float f[2] = {1.0f, 1.0f};
#pragma unroll
          for (int r = 0; r < kR; ++r) {
            const float mn = fmaxf(m[r], mx[r]);
            f[r] = mn == -INFINITY ? 1.0f : exp2_approx(m[r] - mn);
            m[r] = mn;
            l[r] *= f[r];
          }
          if (kHalves) f[1] = f[0];
#pragma unroll
          for (int x = 0; x < kO; ++x) {
            o[x][0] *= f[0];
            o[x][1] *= f[0];
            o[x][2] *= f[1];
            o[x][3] *= f[1];
          }
        }
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const float mm = (m[r] == -INFINITY ? 0.0f : m[r]) - kShift;
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float w = exp2_approx(s[n][2 * r + j] - mm);
              s[n][2 * r + j] = w;
              l[r] += w;
            }
        }
        // numerators
        if constexpr (kWide) {
          const uint32_t pa[4] = {tf32_hi(s[0][0]), tf32_lo(s[0][0]), tf32_hi(s[0][1]), tf32_lo(s[0][1])};
#pragma unroll
          for (int b = 0; b < D / 32; ++b) {
            const uint8_t* vp = smem + warp * Cfg::kRing + stage * 2 * Cfg::kSide + Cfg::kSide;
            const int ch = 8 * b + g;
            const float4 v0 = *reinterpret_cast<const float4*>(vp + ((2 * t) * kChunks + (ch ^ ((2 * t) & 6))) * 16);
            const float4 v1 = *reinterpret_cast<const float4*>(vp + ((2 * t + 1) * kChunks + (ch ^ ((2 * t + 1) & 6))) * 16);
            const float e0[4] = {v0.x, v0.y, v0.z, v0.w}, e1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // summed in registers: the instruction's own sum truncates
              mma_tf32(acc, pa, tf32_lo(e0[j]), tf32_lo(e1[j]));
              mma_tf32(acc, pa, tf32_hi(e0[j]), tf32_hi(e1[j]));
#pragma unroll
              for (int x = 0; x < 4; ++x) o[4 * b + j][x] += acc[x];
            }
          }
        } else {
          uint32_t pa[4];
          if constexpr (kHalves) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const uint32_t hi = pack2(s[n][0], s[n][1], __half());
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              pa[2 * n] = hi;
              pa[2 * n + 1] = pack2(s[n][0] - h.x, s[n][1] - h.y, __half());
            }
          } else {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              pa[2 * n] = pack2(s[n][0], s[n][1], C());
              pa[2 * n + 1] = pack2(s[n][2], s[n][3], C());
            }
          }
          const int mi = lane >> 3, row = (mi & 1) * 8 + (lane & 7);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t b[4];
            ldsm4_t(b, sv + (row * kChunks + ((2 * d + (mi >> 1)) ^ (row & 7))) * 16);
            if constexpr (kHalves) {
              float acc[2][4] = {};
              mma16(acc[0], pa, b[0], b[1], C());
              mma16(acc[1], pa, b[2], b[3], C());
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                o[2 * d][x] += acc[0][x];
                o[2 * d + 1][x] += acc[1][x];
              }
            } else {
              mma16(o[2 * d], pa, b[0], b[1], C());
              mma16(o[2 * d + 1], pa, b[2], b[3], C());
            }
          }
        }
        __syncwarp();
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
      cp_async_wait<0>();
      __syncwarp();
      if (careful) {  // the non-finite elements, for the rows that see them
        for (int i = 0; i < nst; ++i)
          for (int w = 0; w < kPos; ++w) {
            const int pos = sw.first + (my0 + i * kWarps) * kPos + w;
            const long long off = offset_of(pos, page_of(pos));
            if (off < 0) continue;
#pragma unroll
            for (int x = 0; x < kO; ++x)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int dim = kWide ? 32 * (x >> 2) + 4 * (2 * t + j) + (x & 3) : 8 * x + 2 * t + j;
                const float v = to_f32(vbase[off + dim]);
                if (isfinite(v)) continue;
                if (pos <= plast[0] && pos >= pfirst[0]) o[x][j] += v;
                if (!kHalves && pos <= plast[1] && pos >= pfirst[1]) o[x][2 + j] += v;
              }
          }
        break;
      }
      float z = 0.0f;
#pragma unroll
      for (int x = 0; x < kO; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) z = __fmaf_rn(o[x][j], 0.0f, z);
      if (!__any_sync(0xffffffffu, z != 0.0f)) break;  // z is 0, or NaN where a numerator is not finite
    }

    // ---- the warps' shares of the segment, in warp order
#pragma unroll
    for (int r = 0; r < (kHalves ? 1 : 2); ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) s_ml[warp][g + 8 * r] = make_float2(m[r], l[r]);
    }
    {
      float* dst = reinterpret_cast<float*>(smem + warp * Cfg::kRing);
#pragma unroll
      for (int x = 0; x < kO; ++x)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int dim = kWide ? 32 * (x >> 2) + 4 * (2 * t + j) + (x & 3) : 8 * x + 2 * t + j;
          if constexpr (kHalves) {
            dst[g * D + dim] = o[x][j] + o[x][2 + j];
          } else {
            dst[g * D + dim] = o[x][j];
            dst[(g + 8) * D + dim] = o[x][2 + j];
          }
        }
    }
    __syncthreads();
    const bool whole = st0 == 0 && st1 == sw.steps;
    const int slot = 2 * (int)c + (first_seg ? 0 : 1);
    for (int x = tid; x < nrows * (D / 4); x += kThr) {
      const int r = x / (D / 4), d = x % (D / 4) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_ml[w][r].x);
      const float mu = mm == -INFINITY ? 0.0f : mm;
      float ll = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_approx(s_ml[w][r].x - mu);
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * Cfg::kRing) + r * D + d);
        ll = __fmaf_rn(s_ml[w][r].y, f, ll);
        v[0] = __fmaf_rn(y.x, f, v[0]);
        v[1] = __fmaf_rn(y.y, f, v[1]);
        v[2] = __fmaf_rn(y.z, f, v[2]);
        v[3] = __fmaf_rn(y.w, f, v[3]);
      }
      if (whole) {
        const float inv = ll == 0.0f ? 0.0f : __fdiv_rn(1.0f, ll);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= inv;
        const int pr = row0 + r, row = sw.q0 + pr / a.group, h = head * a.group + pr % a.group;
        store_elems(static_cast<T*>(a.out) + (long long)row * a.out_stride + h * D + d, v);
        if (a.lse && d == 0)
          a.lse[(long long)row * a.hq + h] = ll == 0.0f ? -INFINITY : (mm - kShift + log2f(ll)) * kLn2;
      } else {
        *reinterpret_cast<float4*>(ws.num + ((size_t)slot * kTokenMaxRows + r) * D + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) ws.ml[(size_t)slot * kTokenMaxRows + r] = make_float2(mm, ll);
      }
    }
    if (!whole && st0 == 0 && tid == 0) {  // a cut tile begins here: its last step's CTA is the last contributor
      const long long last = cur + sw.steps - 1;
      long long e = last * ctas / total;
      while ((e + 1) * total / ctas <= last) ++e;
      while (e * total / ctas > last) --e;
      ws.rec[c] = make_int4(seq, tile, (int)(e - c) + 1, slot);
    }
    __syncthreads();
    cur += st1 - st0;
    first_seg = false;
  }
}

// The cut tiles: block (c, r) joins row r of the tile whose first part CTA c holds, in CTA
// order. Four warps take every fourth contributor.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(128) token_join_kernel(const AttnArgs a, void* work, int ctas) {
  __shared__ float s_w[kTokenMaxCtas];
  __shared__ float s_o[4][D];
  __shared__ float s_red[4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const TokenWork ws = token_work(work, ctas);
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 rec = ws.rec[c];
  const int count = rec.z;
  if (count == 0) return;
  const int q0 = a.batch.q_start[rec.x], n = a.batch.q_start[rec.x + 1] - q0;
  const int head = rec.y % a.hk, pr = rec.y / a.hk * kRows + r;
  if (pr >= n * a.group) return;
  auto slot_of = [&](int i) -> size_t { return ((size_t)(i == 0 ? rec.w : 2 * (c + i)) * kTokenMaxRows + r); };
  float mm = -INFINITY;
  for (int i = tid; i < count; i += 128) mm = fmaxf(mm, ws.ml[slot_of(i)].x);
  mm = warp_max(mm);
  if (lane == 0) s_red[warp] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float mu = mm == -INFINITY ? 0.0f : mm;
  float ll = 0.0f;
  __syncthreads();
  for (int i = tid; i < count; i += 128) {
    const float2 x = ws.ml[slot_of(i)];
    const float f = exp2_approx(x.x - mu);
    s_w[i] = f;
    ll = __fmaf_rn(x.y, f, ll);
  }
  ll = warp_sum(ll);
  if (lane == 0) s_red[warp] = ll;
  __syncthreads();
  ll = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
  constexpr int E = D / 32;
  float v[E];
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] = 0.0f;
#pragma unroll 8
  for (int i = warp; i < count; i += 4) {
    const float* p = ws.num + slot_of(i) * D + lane * E;
    const float f = s_w[i];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = __fmaf_rn(p[j], f, v[j]);
  }
#pragma unroll
  for (int j = 0; j < E; ++j) s_o[warp][lane * E + j] = v[j];
  __syncthreads();
  const int row = q0 + pr / a.group, h = head * a.group + pr % a.group;
  if (tid < D) {
    const float x = ((s_o[0][tid] + s_o[1][tid]) + s_o[2][tid]) + s_o[3][tid];
    static_cast<T*>(a.out)[(long long)row * a.out_stride + h * D + tid] = from_f32(ll == 0.0f ? 0.0f : __fmul_rn(x, __fdiv_rn(1.0f, ll)), T());
  }
  if (a.lse && tid == 0) a.lse[(long long)row * a.hq + h] = ll == 0.0f ? -INFINITY : (mm - kShift + log2f(ll)) * kLn2;
}

}  // namespace paged
}  // namespace qora
