// paged_token.cuh — attention of a few rows per sequence (one new token, or a few) over its
// paged cache. The time is the K and V bytes of the attended positions, read once.
//
// Tile. A tile is one (sequence, kv head): its rows are the sequence's new tokens times the
// kv head's query heads, packed (row r: token r / group, head r % group), at most kRows of
// them. kRows is what one m16 matrix instruction holds: 16 rows of 16-bit q, or 8 rows of
// f32 q, whose binary16 (tf32, for an f32 cache) upper and lower halves are the
// instruction's rows 0-7 and 8-15: the 22 bits cost no second instruction. An f32 cache is
// split likewise into two operands.
//
// Work split. The steps (kPos positions) of all tiles form one line, cut into gridDim.x
// equal runs: every CTA reads the same number of bytes whatever the lengths are, and one
// request with a long cache fills the GPU as a batch does. The lengths are in device
// memory, so each CTA finds its run itself (a scan of the sequences' step counts). A tile
// that is cut is written as partials (numerators, maximum, sum) and joined in CTA order by
// token_join_kernel, which is launched behind with its launch overlapped; every tile cut begins in
// a different CTA, so the workspace has a fixed size and needs no initial contents.
//
// Inside a CTA every warp takes every kWarps-th step of a segment with its own ring of
// cp.async stages, running maximum and sum; there is no barrier until the segment's end.
// Weights of 16-bit rows are multiplied in two parts too, upper and lower (22 bits, 16 of bf16):
// 128 binary16 tokens are then as close to the exact result as rounding lets them be (rms
// error 1.36e-5; weights rounded to binary16: 1.85e-5). Up to 8 packed rows leave the
// instruction's rows 8-15 for the lower parts (189 us instead of 188 us, consecutive calls on
// changing inputs; as instructions of their own 203 us); more rows take a second instruction
// (64 sequences of 1 to 4 rows over 4,000 positions: 96 us instead of 94 us).
// The maximum is only raised (and the numerators rescaled) when it grows by more than
// 2^kSlack, so weights stay below 2^(kShift + kSlack) <= 2^15, within binary16.
//
// Values that are masked never count: masked scores become -inf, slots behind the last
// position are filled with zeros. What a weight of zero times an infinite value leaves (NaN)
// shows in the numerators; such a segment is run again with the non-finite elements of V
// taken out and added to the rows that do see them, and with NaN scores of f32 rows (an
// infinite key's product with halves of unlike sign) computed in f32.
//
// Measured, the call replayed in a graph (in brackets: consecutive calls on changing inputs):
// 128 tokens over 200 to 8,000 binary16 positions, 4,193 on average, 1.1 GB, 175 us = 6.3 TB/s
// (190 us); 32 tokens over f32 caches, 253 MB, 55 us = 4.6 TB/s (58 us); one token over 32,768
// binary16 positions, 67 MB, 16 us = 4.1 TB/s (21 us), of which some 4 us are the launch, the
// schedule and the join. What holds the f32 caches back is the warps' own instructions: the two
// warps of a scheduler issue in 46 % of its cycles and wait for memory in 7 % of theirs (DRAM 58
// %, tensor pipe 32 % busy).
#pragma once

#include "paged_attention.cuh"
#include "ptx.cuh"

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
  static constexpr int kRowBytes = D * (int)sizeof(C);
  static constexpr int kChunks = kRowBytes / 16;    // 16-byte pieces of a K or V row
  // Pieces are permuted within their 128 bytes so that the reads below touch every bank once:
  // ldmatrix reads one piece of 8 rows; a quarter-warp reads 4 pieces of 2 rows of an f32 K
  // and 2 pieces of rows 0, 2, 4, 6 of V. (Rows padded by 16 bytes instead: 225 us where
  // this took 185 us, 128 ragged tokens; the copies write whole lines.)
  QORA_DEV static int k_at(int row, int ch) { return row * kRowBytes + ((kWide ? ch ^ ((row & 1) << 2) : ch ^ (row & 7)) << 4); }
  QORA_DEV static int v_at(int row, int ch) { return row * kRowBytes + ((kWide ? ch ^ (row & 6) : ch ^ (row & 7)) << 4); }
  static constexpr int kSide = kPos * kRowBytes;  // bytes of a step's K (or V)
  static constexpr int kStep = 2 * kSide;
  // q's fragments lie in shared memory, each warp makes a part of them: in registers they are
  // 32 (f32 cache: 64) of a thread's, made by every warp for itself (32 tokens over f32
  // caches: 61.5 us against 55.3 us)
  static constexpr int kStages = 3;
  static constexpr int kWarps = 8;
  static constexpr int kQSteps = D / (kWide ? 8 : 16);  // k steps of a score
  static constexpr int kQBytes = kQSteps * 32 * 16;
  static constexpr int kRing = kStages * kStep;  // bytes of a warp's ring
  static constexpr int kNum = D + (kWide ? 4 : 8);  // floats from one row of numerators to the next, in the ring
  static_assert(kRows * kNum * 4 <= kRing, "the ring holds the numerators");
  static constexpr int kSmem = kWarps * kRing + kQBytes;
};

constexpr int kTokenMaxCtas = 320;
constexpr int kTokenMaxRows = 16;

// Workspace: records [ctas], partial maxima and sums [2 ctas][16], numerators [2 ctas][16][D].
struct TokenWork {
  int4* rec;    // (first row, packed rows, contributors, 2 * kv head + which slot of the first), contributors 0: none
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

// One sequence's share of the line of steps: hk tiles of `steps` steps.
struct SeqWork {
  int q0, n, len, lo, first;  // first row, new rows, positions, first attended one, first step's
  int steps;
};
template <int kPos>
QORA_DEV SeqWork seq_work(const AttnArgs& a, int s) {
  SeqWork w;
  w.q0 = a.batch.q_start[s];
  const int q1 = a.batch.q_start[s + 1];
  w.len = a.batch.kv_len[s];
  w.n = q1 - w.q0;
  w.lo = w.first = w.steps = 0;
  const long long cap = (long long)a.batch.table_stride * a.pg.page_size;
  if (w.q0 < 0 || q1 < w.q0 || q1 > a.batch.rows || w.n > a.max_q || w.len < 0 || w.len > cap) {
    if (a.status) *a.status = 5u;
    return w;
  }
  if (w.n == 0 || w.n > a.few) return w;
  w.lo = first_seen(a, w.len - w.n);
  w.first = w.lo & ~(kPos - 1);
  w.steps = max(1, (w.len - w.first + kPos - 1) / kPos);
  return w;
}

// CTA c's run of `total` steps over `ctas` CTAs: equal shares, the first ones a step longer.
struct Share {
  unsigned quot, rem;
  QORA_DEV Share(unsigned total, unsigned ctas) : quot(total / ctas), rem(total % ctas) {}
  QORA_DEV unsigned begin(unsigned c) const { return c * quot + min(c, rem); }
  QORA_DEV unsigned owner(unsigned step) const {
    const unsigned big = rem * (quot + 1);
    return step < big ? step / (quot + 1) : rem + (step - big) / quot;
  }
};

template <typename T, typename C, int D>
__global__ void __launch_bounds__(32 * TokenCfg<T, C, D>::kWarps, 1) token_kernel(const AttnArgs a, void* work, int min_steps, int tile_cost) {
  using Cfg = TokenCfg<T, C, D>;
  constexpr int kPos = Cfg::kPos, kRows = Cfg::kRows, kWarps = Cfg::kWarps, kChunks = Cfg::kChunks, kStages = Cfg::kStages;
  constexpr bool kWide = Cfg::kWide, kHalves = Cfg::kHalves;
  static_assert(D / 16 <= kWarps, "a warp for each part of q");
  constexpr int kThr = 32 * kWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_ml[kWarps][kRows];
  __shared__ uint32_t s_bad[kWarps][kStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const TokenWork ws = token_work(work, gridDim.x);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run of the line. Every warp scans the sequences' steps for itself (a lane
  // holds a run of neighbouring sequences): no barrier, and the loads are in flight together
  const unsigned c = blockIdx.x;
  if (tid == 0) ws.rec[c] = make_int4(0, 0, 0, 0);
  const int per = (a.batch.seqs + 31) >> 5;
  unsigned mine = 0;
  bool fits = true;
#pragma unroll 4
  for (int j = 0; j < per; ++j) {
    const int s = lane * per + j;
    if (s < a.batch.seqs) {
      const SeqWork w = seq_work<kPos>(a, s);
      const unsigned long long v = w.steps ? (unsigned long long)(w.steps + tile_cost) * (unsigned)a.hk : 0ull;
      fits = fits && v < (1u << 26) && mine < (1u << 26);
      mine += (unsigned)v;
    }
  }
  fits = fits && mine < (1u << 26);  // 32 lanes: below 2^31
  unsigned x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  const unsigned total = __shfl_sync(0xffffffffu, x, 31);
  if (!__all_sync(0xffffffffu, fits)) {
    if (tid == 0 && a.status) *a.status = 5u;
    return;
  }
  if (total == 0) return;
  // no more CTAs than leave min_steps each: a smaller share costs more to join than it saves
  const unsigned ctas = min(gridDim.x, (total + min_steps - 1) / min_steps);
  if (c >= ctas) return;
  const Share share(total, ctas);
  unsigned cur = share.begin(c);
  const unsigned end = share.begin(c + 1);
  int seq = lane * per;
  unsigned base = x - mine;
  const bool here = base <= cur && cur < x;
  if (here) {
    for (; seq + 1 < min(a.batch.seqs, (lane + 1) * per); ++seq) {
      const SeqWork w = seq_work<kPos>(a, seq);
      const unsigned v = w.steps ? (unsigned)(w.steps + tile_cost) * a.hk : 0u;
      if (cur < base + v) break;
      base += v;
    }
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  seq = __shfl_sync(0xffffffffu, seq, src);
  base = __shfl_sync(0xffffffffu, base, src);
  SeqWork sw = seq_work<kPos>(a, seq);
  uint8_t* const ring = smem + warp * Cfg::kRing;
  const float scale2 = a.scale * kLog2e;
  const bool pow2 = (a.pg.page_size & (a.pg.page_size - 1)) == 0;
  const int shift = 31 - __clz(a.pg.page_size);
  bool first_seg = true;
  int careful = 0;

  while (cur < end) {
    for (unsigned v; cur - base >= (v = sw.steps ? (unsigned)(sw.steps + tile_cost) * a.hk : 0u);) {  // the next sequence with work
      base += v;
      if (++seq >= a.batch.seqs) return;
      sw = seq_work<kPos>(a, seq);
    }
    // units of the tile: tile_cost for the segment's fixed time, then its steps
    const unsigned units = (unsigned)(sw.steps + tile_cost);
    const int head = (int)((cur - base) / units);
    const unsigned u0 = cur - base - (unsigned)head * units, u1 = min(units, u0 + (end - cur));
    const int st0 = max(0, (int)u0 - tile_cost), st1 = max(0, (int)u1 - tile_cost);
    if (st1 <= st0) {
      cur += u1 - u0;
      continue;
    }
    const int nrows = sw.n * a.group;
    const bool spare = !kHalves && nrows <= 8;  // the instruction's rows 8-15 take the weights' lower parts
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
      plast[i] = ok ? p0 + token_of(a, r) : -1;
      pfirst[i] = first_seen(a, plast[i]);
    }
    // every row sees the positions from seen_from to p0
    const int seen_from = first_seen(a, sw.len - 1);

    // offset of position `pos` in the pages; -1: nothing there. Entries before the first
    // attended position may be those of released pages: not read
    auto page_of = [&](int pos) -> int {
      if (pos >= sw.len || pos < sw.lo) return -1;
      return table[pow2 ? pos >> shift : pos / a.pg.page_size];
    };
    auto offset_of = [&](int pos, int page) -> long long {
      if (page < 0 || page >= a.pg.num_pages) return -1;
      const int slot = pow2 ? pos & (a.pg.page_size - 1) : pos % a.pg.page_size;
      return page * a.pg.page_stride + (long long)slot * a.pg.slot_stride;
    };
    const int crow = lane / kChunks, cch = lane % kChunks;  // the lane copies rows crow + i * (32 / kChunks), piece cch
    auto issue = [&](int step, int stage, int page) {  // page: of position step * kPos + lane
      constexpr int kHop = 32 / kChunks;
      const int pos = sw.first + step * kPos;
      const uint32_t dk = ptx::smem_addr(ring + stage * Cfg::kStep), dv = dk + Cfg::kSide;
      const int mine = pos + (lane & (kPos - 1));
      const long long off = offset_of(mine, page);
      const unsigned bad = __ballot_sync(0xffffffffu, off < 0) & ((1u << kPos) - 1);
#pragma unroll
      for (int i = 0; i < kPos / kHop; ++i) {
        const long long o = __shfl_sync(0xffffffffu, off, crow + i * kHop);
        const long long at = (o < 0 ? 0 : o) + cch * (16 / (int)sizeof(C));
        cp_async_16(dk + Cfg::k_at(crow + i * kHop, cch), kbase + at, o >= 0);
        cp_async_16(dv + Cfg::v_at(crow + i * kHop, cch), vbase + at, o >= 0);
      }
      if (lane == 0) s_bad[warp][stage] = bad;
      if (bad && a.status && off < 0 && mine >= sw.lo && mine < sw.len) *a.status = 5u;  // a page that does not exist
    };

    // q in the instruction's layout. f32 rows: 2^e puts the row's largest value in [2^13, 2^14)
    float qscale[2] = {scale2, scale2};
    uint4* const s_q = reinterpret_cast<uint4*>(smem + kWarps * Cfg::kRing);  // [k step][lane]
    auto row_ptr = [&](int r) {
      const int tok = token_of(a, r);
      return static_cast<const T*>(a.q) + (long long)(sw.q0 + tok) * a.q_stride + (head * a.group + r - tok * a.group) * D;
    };
    // the loads are under way while the first copies are issued
    uint32_t qw[4];        // 16-bit rows: the warp's k step; f32 rows: the thread's dims of it
    float mx = 0.0f;       // f32 rows, 16-bit cache: the row's largest value
    if constexpr (!kHalves) {
      if (warp < Cfg::kQSteps) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool ok = g + 8 * i < nrows;
          const T* q = row_ptr(ok ? g + 8 * i : 0) + 16 * warp + 2 * t;
          qw[i] = ok ? *reinterpret_cast<const uint32_t*>(q) : 0u;
          qw[2 + i] = ok ? *reinterpret_cast<const uint32_t*>(q + 8) : 0u;
        }
      }
    } else {
      const bool ok = g < nrows;
      const float* q = reinterpret_cast<const float*>(row_ptr(ok ? g : 0));
      if (warp < D / 16) {
        // two k steps of 8: dims 16 b + 4 t ..; one of 16: 16 k + 2 t .. and 8 on
        const float2 u = *reinterpret_cast<const float2*>(q + 16 * warp + (kWide ? 4 : 2) * t);
        const float2 v = *reinterpret_cast<const float2*>(q + 16 * warp + (kWide ? 4 * t + 2 : 2 * t + 8));
        qw[0] = ok ? __float_as_uint(u.x) : 0u;
        qw[1] = ok ? __float_as_uint(u.y) : 0u;
        qw[2] = ok ? __float_as_uint(v.x) : 0u;
        qw[3] = ok ? __float_as_uint(v.y) : 0u;
      }
      if constexpr (!kWide) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const float4 u = *reinterpret_cast<const float4*>(q + 16 * k + 4 * t);
          mx = fmaxf(mx, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))));
        }
        if (!ok) mx = 0.0f;
      }
    }
    auto make_q = [&]() {
      if constexpr (!kHalves) {
        if (warp < Cfg::kQSteps) s_q[warp * 32 + lane] = make_uint4(qw[0], qw[1], qw[2], qw[3]);
      } else {
        const float x[4] = {__uint_as_float(qw[0]), __uint_as_float(qw[1]), __uint_as_float(qw[2]), __uint_as_float(qw[3])};
        if constexpr (kWide) {  // tf32: the exponent range is f32's, no scale
          if (warp < D / 16) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              s_q[(2 * warp + k) * 32 + lane] = make_uint4(tf32_hi(x[2 * k]), tf32_lo(x[2 * k]), tf32_hi(x[2 * k + 1]), tf32_lo(x[2 * k + 1]));
          }
        } else {
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // exponent of mx (0 for zeros and subnormals, 255 for non-finite rows: no scale)
          const int ex = (int)(__float_as_uint(mx) >> 23);
          const int up = ex == 0 || ex == 255 ? 0 : min(126, 140 - ex);
          const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
          qscale[0] = scale2 * __uint_as_float((uint32_t)(127 - up) << 23);
          if (warp < D / 16) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float u = x[2 * k] * mul, v = x[2 * k + 1] * mul;
              w[2 * k] = pack2(u, v, __half());
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * k]));
              w[2 * k + 1] = pack2(u - h.x, v - h.y, __half());
            }
            s_q[warp * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      __syncthreads();
    };

    // f32 rows: q . k in f32, of the thread's row and position `w` of a step. An infinite value
    // leaves NaN in the sum of products of halves, where q . k may be infinite.
    auto plain_score = [&](const uint8_t* pk, int w) {
      const float* q = reinterpret_cast<const float*>(row_ptr(g < nrows ? g : 0));
      constexpr int kPiece = 16 / (int)sizeof(C);
      float d = 0.0f;
#pragma unroll 1
      for (int x = 0; x < D; ++x)
        d = __fmaf_rn(q[x], to_f32(reinterpret_cast<const C*>(pk + Cfg::k_at(w, x / kPiece))[x % kPiece]), d);
      return d;
    };

    constexpr int kO = D / 8;  // numerators: n8 tiles of 4 values
    float o[kO][4];
    float m[2], l[2];
    {
#pragma unroll
      for (int i = 0; i < kO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.0f;
      const int nst = st1 - st0 > warp ? (st1 - st0 - warp + kWarps - 1) / kWarps : 0;  // this warp's steps
      const int my0 = st0 + warp;
      auto next_page = [&](int i) { return i < nst ? page_of(sw.first + (my0 + i * kWarps) * kPos + (lane & (kPos - 1))) : -1; };
      int page = next_page(0), stage = 0, fill = 0;
#pragma unroll 1
      for (int i = 1 - kStages; i < nst; ++i) {
        if (i >= 0) cp_async_wait<kStages - 2>();
        __syncwarp();
        const int np = next_page(i + kStages);
        if (i + kStages - 1 < nst) issue(my0 + (i + kStages - 1) * kWarps, fill, page);  // into the stage that the previous step left
        cp_async_commit();
        page = np;
        fill = fill + 1 == kStages ? 0 : fill + 1;
        if (i < 0) {
          if (i == -1) make_q();
          continue;
        }
        const int pos0 = sw.first + (my0 + i * kWarps) * kPos;
        uint8_t* const pk = ring + stage * Cfg::kStep;
        uint8_t* const pv = pk + Cfg::kSide;
        const uint32_t sk = ptx::smem_addr(pk), sv = ptx::smem_addr(pv);
        const uint32_t bad = s_bad[warp][stage];
        if (careful) {  // non-finite elements of V become zero
#pragma unroll 1
          for (int x = lane; x < kPos * kChunks; x += 32) {
            uint4* p = reinterpret_cast<uint4*>(pv) + x;
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
          float u[4] = {}, v[4] = {}, u2[4] = {}, v2[4] = {};
#pragma unroll
          for (int b = 0; b < D / 16; ++b) {
            const float4 k = *reinterpret_cast<const float4*>(pk + Cfg::k_at(g, 4 * b + t));
            const uint4 q0 = s_q[(2 * b) * 32 + lane], q1 = s_q[(2 * b + 1) * 32 + lane];
            const uint32_t a0[4] = {q0.x, q0.y, q0.z, q0.w}, a1[4] = {q1.x, q1.y, q1.z, q1.w};
            mma_tf32(u, a0, tf32_hi(k.x), tf32_hi(k.y));
            mma_tf32(v, a0, tf32_lo(k.x), tf32_lo(k.y));
            mma_tf32(u2, a1, tf32_hi(k.z), tf32_hi(k.w));
            mma_tf32(v2, a1, tf32_lo(k.z), tf32_lo(k.w));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) s[0][j] = (u[j] + u2[j]) + (v[j] + v2[j]);
        } else {
#pragma unroll
          for (int n = 0; n < kN; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
          float s2[kN][4] = {};  // two sums each: shorter chains
          const int mi = lane >> 3, row = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
          for (int k = 0; k < Cfg::kQSteps; ++k) {
            uint32_t b[4];
            ldsm4(b, sk + Cfg::k_at(row, 2 * k + (mi & 1)));
            const uint4 q4 = s_q[k * 32 + lane];
            const uint32_t qa[4] = {q4.x, q4.y, q4.z, q4.w};
            mma16(k & 1 ? s2[0] : s[0], qa, b[0], b[1], C());
            mma16(k & 1 ? s2[1] : s[1], qa, b[2], b[3], C());
          }
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] += s2[n][j];
        }
        constexpr int kR = kHalves ? 1 : 2;
        if constexpr (kHalves) {
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            s[n][0] += s[n][2];
            s[n][1] += s[n][3];
          }
        }
        const bool plain = pos0 >= seen_from && pos0 + kPos - 1 <= p0 && bad == 0;
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
        if (kHalves && careful) {
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (s[n][j] != s[n][j]) {
                s[n][j] = plain_score(pk, 8 * n + 2 * t + j) * scale2;
                mx[0] = fmaxf(mx[0], s[n][j]);
              }
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
          if (kHalves || spare) f[1] = f[0];
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
            const float4 v0 = *reinterpret_cast<const float4*>(pv + Cfg::v_at(2 * t, 8 * b + g));
            const float4 v1 = *reinterpret_cast<const float4*>(pv + Cfg::v_at(2 * t + 1, 8 * b + g));
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
          const int mi = lane >> 3, row = (mi & 1) * 8 + (lane & 7);
          auto lower = [&](uint32_t hi, float x, float y) {  // what the upper parts `hi` of two weights leave
            const C* e = reinterpret_cast<const C*>(&hi);
            return pack2(x - to_f32(e[0]), y - to_f32(e[1]), C());
          };
          uint32_t pa[4];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            pa[2 * n] = pack2(s[n][0], s[n][1], C());
            pa[2 * n + 1] = kHalves || spare ? lower(pa[2 * n], s[n][0], s[n][1]) : pack2(s[n][2], s[n][3], C());
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t b[4];
            ldsm4_t(b, sv + Cfg::v_at(row, 2 * d + (mi >> 1)));
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
          if (!kHalves && !spare) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              pa[2 * n] = lower(pa[2 * n], s[n][0], s[n][1]);
              pa[2 * n + 1] = lower(pa[2 * n + 1], s[n][2], s[n][3]);
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              uint32_t b[4];
              ldsm4_t(b, sv + Cfg::v_at(row, 2 * d + (mi >> 1)));
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
#pragma unroll 1
        for (int i = 0; i < nst; ++i)
#pragma unroll 1
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
      }
    }

    // ---- the warps' shares of the segment, in warp order
#pragma unroll
    for (int r = 0; r < (kHalves ? 1 : 2); ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) s_ml[warp][g + 8 * r] = make_float2(m[r], l[r]);
    }
    {
      float* dst = reinterpret_cast<float*>(ring) + g * Cfg::kNum;
      if constexpr (kWide) {
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            *reinterpret_cast<float4*>(dst + 32 * b + 4 * (2 * t + j)) =
                make_float4(o[4 * b][j] + o[4 * b][2 + j], o[4 * b + 1][j] + o[4 * b + 1][2 + j],
                            o[4 * b + 2][j] + o[4 * b + 2][2 + j], o[4 * b + 3][j] + o[4 * b + 3][2 + j]);
      } else {
#pragma unroll
        for (int x = 0; x < kO; ++x) {
          if constexpr (kHalves) {
            *reinterpret_cast<float2*>(dst + 8 * x + 2 * t) = make_float2(o[x][0] + o[x][2], o[x][1] + o[x][3]);
          } else if (spare) {
            *reinterpret_cast<float2*>(dst + 8 * x + 2 * t) = make_float2(o[x][0] + o[x][2], o[x][1] + o[x][3]);
          } else {
            *reinterpret_cast<float2*>(dst + 8 * x + 2 * t) = make_float2(o[x][0], o[x][1]);
            *reinterpret_cast<float2*>(dst + 8 * Cfg::kNum + 8 * x + 2 * t) = make_float2(o[x][2], o[x][3]);
          }
        }
      }
    }
    float z = 0.0f;  // 0, or NaN where a numerator is not finite
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j) z = __fmaf_rn(o[x][j], 0.0f, z);
    if (__syncthreads_or(z != 0.0f) && !careful) {
      careful = 1;
      continue;
    }
    careful = 0;
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
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * Cfg::kRing) + r * Cfg::kNum + d);
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
        const int tok = token_of(a, r), row = sw.q0 + tok, h = head * a.group + r - tok * a.group;
        store_elems(static_cast<T*>(a.out) + (long long)row * a.out_stride + h * D + d, v);
        if (a.lse && d == 0)
          a.lse[(long long)row * a.hq + h] = ll == 0.0f ? -INFINITY : (mm - kShift + log2f(ll)) * kLn2;
      } else {
        *reinterpret_cast<float4*>(ws.num + ((size_t)slot * kTokenMaxRows + r) * D + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) ws.ml[(size_t)slot * kTokenMaxRows + r] = make_float2(mm, ll);
      }
    }
    if (!whole && st0 == 0 && tid == 0) {  // a cut tile begins here: its last step's CTA is the last contributor
      const unsigned e = share.owner(base + (unsigned)(head + 1) * units - 1);
      ws.rec[c] = make_int4(sw.q0, sw.n * a.group, (int)(e - c) + 1, 2 * head + (first_seg ? 0 : 1));
    }
    __syncthreads();
    cur += u1 - u0;
    first_seg = false;
  }
}

// The cut tiles: block (c, r) joins row r of the tile whose first part CTA c holds, in CTA
// order. Four warps take every fourth contributor.
template <typename T, int D>
__global__ void __launch_bounds__(128) token_join_kernel(const AttnArgs a, void* work, int ctas) {
  __shared__ float s_w[kTokenMaxCtas];
  __shared__ float s_o[4][D];
  __shared__ float s_red[4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const TokenWork ws = token_work(work, ctas);
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 rec = ws.rec[c];
  const int count = rec.z;
  if (r >= rec.y || count == 0) return;
  const int head = rec.w >> 1;
  auto slot_of = [&](int i) -> size_t { return (size_t)(2 * (c + i) + (i == 0 ? rec.w & 1 : 0)) * kTokenMaxRows + r; };
  // the first contributors' numerators are on their way while the weights are found
  constexpr int E = D / 32, kAhead = 10;
  float y[kAhead][E];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int i = warp + 4 * k;
    const float* p = ws.num + slot_of(i < count ? i : 0) * D + lane * E;
#pragma unroll
    for (int j = 0; j < E; j += 2) {
      const float2 v = *reinterpret_cast<const float2*>(p + j);
      y[k][j] = v.x;
      y[k][j + 1] = v.y;
    }
  }
  float2 ml[(kTokenMaxCtas + 127) / 128];
  float mm = -INFINITY;
#pragma unroll
  for (int k = 0; k < (kTokenMaxCtas + 127) / 128; ++k) {
    const int i = tid + 128 * k;
    ml[k] = i < count ? ws.ml[slot_of(i)] : make_float2(-INFINITY, 0.0f);
    mm = fmaxf(mm, ml[k].x);
  }
  mm = warp_max(mm);
  if (lane == 0) s_red[warp] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float mu = mm == -INFINITY ? 0.0f : mm;
  float ll = 0.0f;
#pragma unroll
  for (int k = 0; k < (kTokenMaxCtas + 127) / 128; ++k) {
    const int i = tid + 128 * k;
    const float f = exp2_approx(ml[k].x - mu);
    if (i < count) s_w[i] = f;
    ll = __fmaf_rn(ml[k].y, f, ll);
  }
  ll = warp_sum(ll);
  __syncthreads();  // s_red is read by all before it is written again
  if (lane == 0) s_red[warp] = ll;
  __syncthreads();
  ll = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
  float v[E];
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] = 0.0f;
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (warp + 4 * k < count) {
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = __fmaf_rn(y[k][j], s_w[warp + 4 * k], v[j]);
    }
#pragma unroll 4
  for (int i = warp + 4 * kAhead; i < count; i += 4) {
    const float* p = ws.num + slot_of(i) * D + lane * E;
    const float f = s_w[i];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = __fmaf_rn(p[j], f, v[j]);
  }
#pragma unroll
  for (int j = 0; j < E; ++j) s_o[warp][lane * E + j] = v[j];
  __syncthreads();
  const int tok = token_of(a, r), row = rec.x + tok, h = head * a.group + r - tok * a.group;
  if (tid < D) {
    const float x = ((s_o[0][tid] + s_o[1][tid]) + s_o[2][tid]) + s_o[3][tid];
    static_cast<T*>(a.out)[(long long)row * a.out_stride + h * D + tid] = from_f32(ll == 0.0f ? 0.0f : __fmul_rn(x, __fdiv_rn(1.0f, ll)), T());
  }
  if (a.lse && tid == 0) a.lse[(long long)row * a.hq + h] = ll == 0.0f ? -INFINITY : (mm - kShift + log2f(ll)) * kLn2;
}

}  // namespace paged
}  // namespace qora
