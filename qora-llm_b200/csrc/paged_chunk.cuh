// paged_chunk.cuh — attention of chunks of new rows over their paged caches on the tensor
// cores (tcgen05, TMEM). The time is the two products, 4 D operations per (query head, row,
// position).
//
// Item. 256 packed rows of one (sequence, kv head): tokens times the kv head's query heads
// (row r: token r / group, head r % group), so that grouped heads share every K and V tile.
// They are two blocks of 128 rows (X = 0, 1), each with its scores (128 columns) and its
// numerators (D columns) in TMEM; K and V tiles of 128 positions feed both. Where there are
// fewer items than CTAs, the positions of an item are split evenly and join_kernel adds the
// parts in order. Items are taken from the last rows (the longest runs of positions) on, in
// alternating direction, so the CTAs end together.
//
// Roles (384 threads, one CTA per SM: a softmax thread keeps its row's 128 scores in registers):
//   warps 0-3, 4-7   softmax of block 0, 1: a thread owns a row, reads its 128 scores from
//                    TMEM, writes the weights back over them as the next product's operand
//   warp 8           issues the products: S_X = Q_X K^T; O_X += P_X V with P_X from TMEM
//   warps 9, 10      load K and V into the 128-byte-swizzled tiles that the products read. A
//                    tile whose 128 positions all exist comes by TMA, a page (or 128 rows of
//                    one) per copy, where the page size divides 128 or is a multiple of it;
//                    other tiles are copied by cp.async in 16-byte pieces, the page looked up
//                    per position (slots past the end become zeros)
//   warp 11          loads q (f32 rows: warps 9-11, which split it)
// While one block's weights are computed the other block's products run. S_X(j + 1) is
// issued behind O_X(j), which still reads P_X(j) from the columns it overwrites: one
// thread's products execute in order.
//
// f32 rows (f16 cache): q is split into binary16 upper and lower halves (22 bits, the row
// scaled by a power of two) and so are the weights; both halves are multiplied, which
// doubles the products.
//
// The running maximum is raised only when it grows by more than 2^kSlack: then the
// numerators in TMEM are scaled, which is rare after the first tiles. Masked scores become
// -inf before the maximum; a row that meets a non-finite value (a weight of zero times an
// infinite value of V, or a row whose own scores are) is computed again by one warp, one
// position at a time (row_attend).
#pragma once

#include <cuda.h>

#include <type_traits>

#include "paged_attention.cuh"
#include "paged_token.cuh"
#include "tcgen05.cuh"

namespace qora {
namespace paged {

template <typename T, typename C, int D>
struct ChunkCfg {
  static constexpr bool kHalves = sizeof(T) == 4;
  static constexpr int kParts = kHalves ? 2 : 1;
  static constexpr int kBlock = 128;            // rows of a block
  static constexpr int kRows = 2 * kBlock;      // rows of an item
  static constexpr int kPos = 128;              // positions of a tile
  static constexpr int kQTile = kBlock * D * 2;
  static constexpr int kQBytes = 2 * kParts * kQTile;  // [block][part]
  static constexpr int kStage = kPos * D * 2;
  static constexpr int kOther = 1024 /* offsets */ + 512 /* row scales */ + 512 /* barriers, flags */;
  static constexpr int kLimit = 227 * 1024 - 1024 - kOther;
  static constexpr int kStages = (kLimit - kQBytes) / kStage < 6 ? (kLimit - kQBytes) / kStage : 6;
  static_assert(kStages >= 3, "a K tile, a V tile and the next K tile");
  static constexpr int kLag = kStages >= 4 ? 2 : 1;  // copies in flight behind the newest: at most kStages - 2
  static constexpr int kSmem = kQBytes + kStages * kStage + kOther + 1024;
  static constexpr int kThreads = 384;
  static constexpr int kLoaders = 64;
};
constexpr int kChunkMaxCtas = 160;
constexpr unsigned long long kWaitNs = 2000000000ull;

// Workspace of split items: [item] (maximum, sum) of 256 rows, then numerators [item][256][D].
__host__ __device__ inline float2* chunk_ml(void* p) { return static_cast<float2*>(p); }
__host__ __device__ inline float* chunk_num(void* p) {
  return reinterpret_cast<float*>(static_cast<char*>(p) + (size_t)kChunkMaxCtas * 256 * 8);
}

// ---------------------------------------------------------------- instructions
QORA_DEV void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
QORA_DEV void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
// box at (x, slot, head, page) of the pages to shared memory, completing on `bar`
QORA_DEV void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(ptx::smem_addr(bar))
      : "memory");
}
QORA_DEV void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
QORA_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
QORA_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Tiles are [rows][64 elements] halves of 128-byte rows, 16-byte pieces permuted by the row
// (128-byte swizzle; 8-row groups 1024 bytes apart), the second half `rows * 128` bytes on.
// Read K-major (k along the row): a k step of 16 is 32 bytes on. Read MN-major (k down the
// rows): groups of 8 k are 1024 bytes apart, groups of 64 columns `rows * 128`.
// A matrix descriptor's upper word is the same for all; in the lower one the address counts
// 16 bytes, so a step is one addition: the issuing thread has 64 cycles per product.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
QORA_DEV uint32_t desc_k(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
QORA_DEV uint32_t desc_mn(uint32_t addr, uint32_t half) { return ((addr >> 4) & 0x3FFFu) | ((half >> 4) << 16); }

// D[tmem] (+)= A[smem] . B[smem], kind::f16
QORA_DEV void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem], kind::f16
QORA_DEV void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n mov.b64 db, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
// f32 accumulators, M = 128, N = n; b_mn: B is MN-major
template <typename C>
__host__ __device__ constexpr uint32_t chunk_idesc(int n, bool b_mn) {
  return (1u << 4) | (sizeof(C) == 2 && std::is_same<C, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) |
         (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// ---------------------------------------------------------------- items
struct ItemRange {
  int seq, q0, n, len, head, tok0, rows;  // sequence, its first row, new rows, positions; kv head, first token, packed rows here
  int first;                          // first position of the first tile
  int tiles;                          // tiles of this split
  int slot;                           // partial slot, or -1: the item is whole
};

// The sequences' row tiles as a warp holds them: a lane sums a run of neighbouring sequences.
struct ItemMap {
  int per, mine, upto, total;  // sequences of a lane; its row tiles; those up to it; all
};
QORA_DEV int seq_tiles(const AttnArgs& a, int s, int tokens) {
  const int q0 = a.batch.q_start[s], q1 = a.batch.q_start[s + 1], len = a.batch.kv_len[s];
  const long long cap = (long long)a.batch.table_stride * a.pg.page_size;
  if (q0 < 0 || q1 < q0 || q1 > a.batch.rows || q1 - q0 > a.max_q || len < 0 || len > cap) {
    if (a.status) *a.status = 5u;
    return 0;
  }
  return (q1 - q0 + tokens - 1) / tokens;
}
QORA_DEV ItemMap item_map(const AttnArgs& a, int tokens, int lane) {
  ItemMap m;
  m.per = (a.batch.seqs + 31) >> 5;
  m.mine = 0;
#pragma unroll 4
  for (int j = 0; j < m.per; ++j) {
    const int s = lane * m.per + j;
    if (s < a.batch.seqs) m.mine += seq_tiles(a, s, tokens);
  }
  m.upto = m.mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, m.upto, o);
    if (lane >= o) m.upto += y;
  }
  m.total = __shfl_sync(0xffffffffu, m.upto, 31);
  return m;
}
// Item idx, of m.total * hk * splits; by a whole warp.
template <int kPos, int kRows>
QORA_DEV ItemRange item_at(const AttnArgs& a, const ItemMap& m, int tokens, int splits, int idx, int lane) {
  const int split = idx % splits, head = idx / splits % a.hk;
  const int tile = m.total - 1 - idx / splits / a.hk;  // the longest runs of positions first
  const bool here = m.upto - m.mine <= tile && tile < m.upto;
  int s = lane * m.per, base = m.upto - m.mine;
  if (here) {
    for (; s + 1 < min(a.batch.seqs, (lane + 1) * m.per); ++s) {
      const int v = seq_tiles(a, s, tokens);
      if (tile < base + v) break;
      base += v;
    }
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  s = __shfl_sync(0xffffffffu, s, src);
  base = __shfl_sync(0xffffffffu, base, src);
  ItemRange r;
  r.seq = s;
  r.q0 = a.batch.q_start[s];
  r.n = a.batch.q_start[s + 1] - r.q0;
  r.len = a.batch.kv_len[s];
  r.head = head;
  r.tok0 = (tile - base) * tokens;
  const int toks = min(tokens, r.n - r.tok0);
  r.rows = toks * a.group;
  const int p0 = r.len - r.n + r.tok0;              // position of the first row
  const int hi = min(r.len, p0 + toks);             // positions [lo, hi) are attended to
  const int lo = a.window > 0 ? max(0, p0 + 1 - a.window) : 0;
  const int t0 = lo / kPos, nt = max(0, (hi + kPos - 1) / kPos - t0);
  const int b = (int)((long long)split * nt / splits), e = (int)((long long)(split + 1) * nt / splits);
  r.first = (t0 + b) * kPos;
  r.tiles = e - b;
  r.slot = splits > 1 ? idx : -1;
  return r;
}

// A row by one warp, over positions [from, to]: lane's elements lane + 32 i.
template <typename T, typename C, int D>
QORA_DEV void row_attend(const AttnArgs& a, const T* q, const int* table, int head, int from, int to, float scale2,
                         float (&o)[D / 32], float& m, float& l) {
  const int lane = threadIdx.x & 31;
  float qv[D / 32];
  for (int i = 0; i < D / 32; ++i) {
    qv[i] = to_f32(q[lane + 32 * i]);
    o[i] = 0.0f;
  }
  m = -INFINITY;
  l = 0.0f;
#pragma unroll 1
  for (int j = from; j <= to; ++j) {
    const int pi = j / a.pg.page_size, page = table[pi];
    if (page < 0 || page >= a.pg.num_pages) continue;
    const long long off = page * a.pg.page_stride + (long long)(j - pi * a.pg.page_size) * a.pg.slot_stride +
                          (long long)head * a.pg.head_stride;
    const C* k = static_cast<const C*>(a.k_pages) + off;
    const C* v = static_cast<const C*>(a.v_pages) + off;
    float d = 0.0f;
    for (int i = 0; i < D / 32; ++i) d = __fmaf_rn(qv[i], to_f32(k[lane + 32 * i]), d);
    d = __fmul_rn(warp_sum(d), scale2);
    const float mn = fmaxf(m, d);
    const float mu = mn == -INFINITY ? 0.0f : mn;  // a NaN score does not raise the maximum: its weight is NaN
    const float w = exp2f(d - mu + kShift), c = exp2f(m - mu);
    l = __fmaf_rn(l, c, w);
    for (int i = 0; i < D / 32; ++i) o[i] = __fmaf_rn(o[i], c, w == 0.0f ? 0.0f : __fmul_rn(w, to_f32(v[lane + 32 * i])));
    m = mn;
  }
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(384, 1) chunk_kernel(const AttnArgs a, void* work, int tokens, int splits, int max_items, int box_rows,
                                                       const __grid_constant__ CUtensorMap kmap,
                                                       const __grid_constant__ CUtensorMap vmap) {
  using Cfg = ChunkCfg<T, C, D>;
  constexpr bool kHalves = Cfg::kHalves;
  constexpr int kPos = Cfg::kPos, kParts = Cfg::kParts, kStages = Cfg::kStages, kLag = Cfg::kLag;
  constexpr int kHalfQ = Cfg::kBlock * 128, kHalfKV = kPos * 128;  // bytes from one 64-element half to the next
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (ptx::smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* const sq = smem;
  uint8_t* const ring = smem + Cfg::kQBytes;
  long long* const s_off = reinterpret_cast<long long*>(ring + kStages * Cfg::kStage);  // [128]
  int8_t* const s_up = reinterpret_cast<int8_t*>(s_off + 128);  // [2 turns][256] exponents of the row scales
  uint64_t* const bars = reinterpret_cast<uint64_t*>(s_up + 512);
  uint64_t *const full = bars, *const empty = bars + 8, *const q_full = bars + 16, *const q_empty = bars + 17,
           *const s_full = bars + 18, *const p_ready = bars + 20, *const o_full = bars + 22, *const done = bars + 24;
  uint32_t* const s_bad = reinterpret_cast<uint32_t*>(bars + 26);  // [8 tiles][4] positions that there are not
  uint32_t* const s_tmem = s_bad + 32;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(s_bad + 33);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full + i, 1);
      ptx::mbar_init(empty + i, 1);
    }
    ptx::mbar_init(q_full, kHalves ? 96 : 32);
    ptx::mbar_init(q_empty, 1);
    for (int x = 0; x < 2; ++x) {
      ptx::mbar_init(s_full + x, 1);
      ptx::mbar_init(p_ready + x, 128);
      ptx::mbar_init(o_full + x, 1);
    }
    ptx::mbar_init(done, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 8) umma::tmem_alloc(s_tmem, 512);
  umma::tc_fence_before();
  __syncthreads();
  umma::tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const uint32_t t_s[2] = {tmem, tmem + 128};
  const uint32_t t_o[2] = {tmem + 256, tmem + 256 + D};
  const ItemMap map = item_map(a, tokens, lane);
  // more row tiles than the rows can hold: the sequences' row ranges overlap
  const bool too_many = (long long)map.total * a.hk * splits > max_items;
  if (too_many && tid == 0 && a.status) *a.status = 5u;
  const int items = too_many ? 0 : map.total * a.hk * splits;
  const int ctas = (int)gridDim.x, cta = (int)blockIdx.x;
  // item of turn w: alternating direction, so that long and short items pair up
  auto item_of = [&](int w) { return w * ctas + (w & 1 ? ctas - 1 - cta : cta); };
  auto wait = [&](uint64_t* bar, uint32_t parity) { return umma::wait_bar(bar, parity, kWaitNs, abort_flag); };

  if (warp == 8) {
    {
      // ---------------------------------------------------------------- products
      uint32_t tile = 0, turn = 0, ns_done[2] = {0, 0};
      bool ok = true;
      const uint32_t q_k = desc_k(ptx::smem_addr(sq)), ring_k = desc_k(ptx::smem_addr(ring)),
                     ring_mn = desc_mn(ptx::smem_addr(ring), kHalfKV);
      constexpr uint32_t id_s = chunk_idesc<C>(kPos, false), id_o = chunk_idesc<C>(D, true);
      for (int w = 0; ok && w * ctas < items; ++w) {
        const int idx = item_of(w);
        if (idx >= items) continue;
        const ItemRange it = item_at<kPos, Cfg::kRows>(a, map, tokens, splits, idx, lane);
        if (it.tiles == 0) continue;
        const int blocks = it.rows > Cfg::kBlock ? 2 : 1;
        if (lane == 0) {
          // ring entries alternate K, V: entry e lies in stage e % kStages
          auto entry = [&](uint32_t e) { return wait(full + e % kStages, (e / kStages) & 1); };
          auto scores = [&](int x, uint32_t e) {
            const uint32_t kb = ring_k + (e % kStages) * (Cfg::kStage >> 4);
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint32_t qb = q_k + (x * kParts + part) * (Cfg::kQTile >> 4);
#pragma unroll
              for (int k = 0; k < D / 16; ++k)
                mma_ss(t_s[x], qb + (k / 4) * (kHalfQ >> 4) + (k % 4) * 2, kb + (k / 4) * (kHalfKV >> 4) + (k % 4) * 2, id_s,
                       part || k);
            }
            umma::mma_commit(s_full + x);
          };
          ok = wait(q_full, turn & 1) && entry(tile * 2);
          umma::tc_fence_after();
          if (ok) {
            for (int x = 0; x < blocks; ++x) scores(x, tile * 2);
            umma::mma_commit(empty + (tile * 2) % kStages);
            for (int j = 0; ok && j < it.tiles; ++j) {
              const uint32_t ev = (tile + j) * 2 + 1, ek = ev + 1;
              const bool last = j + 1 == it.tiles;
              ok = entry(ev);
              const uint32_t vb = ring_mn + (ev % kStages) * (Cfg::kStage >> 4);
              for (int x = 0; ok && x < blocks; ++x) {
                ok = wait(p_ready + x, ns_done[x] & 1);
                ++ns_done[x];
                umma::tc_fence_after();
                if (!ok) break;
#pragma unroll
                for (int part = 0; part < kParts; ++part)
#pragma unroll
                  for (int k = 0; k < kPos / 16; ++k)
                    mma_ts(t_o[x], t_s[x] + kParts * 32 * (k / 4) + part * 32 + (k % 4) * 8, vb + k * (2048 >> 4), id_o, part || k ? 1u : (uint32_t)(j > 0));
                if (last) {
                  umma::mma_commit(o_full + x);
                } else {
                  if (x == 0) {
                    ok = entry(ek);
                    umma::tc_fence_after();
                  }
                  if (ok) scores(x, ek);
                }
              }
              if (!ok) break;
              umma::mma_commit(empty + ev % kStages);
              if (!last) umma::mma_commit(empty + ek % kStages);
            }
            umma::mma_commit(q_empty);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        tile += it.tiles;
        ++turn;
      }
      // every product has completed before the TMEM goes
      if (lane == 0) {
        umma::mma_commit(done);
        umma::wait_bar(done, 0, kWaitNs, abort_flag);
      }
      __syncwarp();
    }
  } else if (warp > 8) {
    // ------------------------------------------------------------------ loads
    const int lw = warp - 9, lt = tid - 9 * 32;  // lw 0, 1: K and V; 2: q
    uint32_t entry = 0, turn = 0, tiles = 0;
    bool ok = true, stop = false;  // this thread's waits ended in time; the role's threads agree to stop
    uint64_t* pend[kLag];  // barriers of the copies still in flight
    int np = 0;
    // one arrival for the loaders' 64 threads, each of which has fenced its own copies
    auto arrive = [&](uint64_t* bar) {
      ptx::named_bar(1, Cfg::kLoaders);
      if (lt == 0) ptx::mbar_arrive(bar);
    };
    auto flush = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      ptx::fence_proxy_async();
#pragma unroll
      for (int i = 0; i < kLag; ++i)
        if (i < np) arrive(pend[i]);
      np = 0;
    };
    auto landed = [&](uint64_t* bar) {  // the newest group is bar's; the one kLag before it is done
      cp_async_commit();
      if (np == kLag) {
        cp_async_wait<kLag>();
        ptx::fence_proxy_async();
        arrive(pend[0]);
#pragma unroll
        for (int i = 0; i + 1 < kLag; ++i) pend[i] = pend[i + 1];
        pend[kLag - 1] = bar;
      } else {
#pragma unroll
        for (int i = 0; i < kLag; ++i)
          if (i == np) pend[i] = bar;
        ++np;
      }
    };
    // a wait that has to last announces what has landed first
    auto wait_free = [&](uint64_t* bar, uint32_t parity) {
      if (np && ptx::named_bar_or(1, Cfg::kLoaders, !ptx::mbar_try_wait(bar, parity))) flush();
      return wait(bar, parity);
    };
    constexpr int kPieces = D * 2 / 16;                 // 16-byte pieces of a 16-bit row
    constexpr int kHop = Cfg::kLoaders / kPieces;       // rows that the loaders copy at once
    const int pr = lt / kPieces, pc = lt % kPieces;
    // byte offset of (row, piece) in a tile whose halves are `half` bytes apart
    auto at = [](int row, int piece, int half) { return (piece >> 3) * half + row * 128 + (((piece & 7) ^ (row & 7)) << 4); };
    for (int w = 0; !stop && w * ctas < items; ++w) {
      const int idx = item_of(w);
      if (idx >= items) continue;
      const ItemRange it = item_at<kPos, Cfg::kRows>(a, map, tokens, splits, idx, lane);
      if (it.tiles == 0) continue;
      const int blocks = it.rows > Cfg::kBlock ? 2 : 1;
      if constexpr (!kHalves) {
        if (lw == 2) {
          ok = __all_sync(0xffffffffu, wait(q_empty, (turn & 1) ^ 1)) != 0;
          stop = !ok;
          if (stop) break;
          constexpr int kQHop = 32 / kPieces;
          const int qr = lane / kPieces, qc = lane % kPieces;
#pragma unroll 8
          for (int r = qr; r < blocks * Cfg::kBlock; r += kQHop) {
            const int tok = r / a.group;
            const bool live = r < it.rows;
            const T* src = static_cast<const T*>(a.q) + (long long)(it.q0 + (live ? it.tok0 + tok : 0)) * a.q_stride +
                           (live ? it.head * a.group + r - tok * a.group : 0) * D + qc * 8;
            cp_async_16(ptx::smem_addr(sq + (r / Cfg::kBlock) * Cfg::kQTile + at(r % Cfg::kBlock, qc, kHalfQ)), src, live);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          ptx::fence_proxy_async();
          ptx::mbar_arrive(q_full);
        }
      } else {
        if (lw < 2) flush();
        ok = ok && wait(q_empty, (turn & 1) ^ 1);
        // four lanes a row, every fourth float4 each; 2^up puts the row's largest in [2^13, 2^14)
        constexpr int kF4 = D / 16;  // float4s of a lane
        const int sub = lane & 3;
#pragma unroll 1
        for (int r0 = lw * 8; r0 < blocks * Cfg::kBlock; r0 += 24) {
          const int r = r0 + (lane >> 2), tok = r / a.group;
          const bool live = r < it.rows;
          const float* src = reinterpret_cast<const float*>(a.q) + (long long)(it.q0 + (live ? it.tok0 + tok : 0)) * a.q_stride +
                             (live ? it.head * a.group + r - tok * a.group : 0) * D + sub * 4;
          float4 x[kF4];
          float mx = 0.0f;
#pragma unroll
          for (int k = 0; k < kF4; ++k) x[k] = *reinterpret_cast<const float4*>(src + 16 * k);
#pragma unroll
          for (int k = 0; k < kF4; ++k) {
            if (!live) x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const int ex = (int)(__float_as_uint(mx) >> 23);
          const int up = ex == 0 || ex == 255 ? 0 : min(126, 140 - ex);
          const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
          if (r < blocks * Cfg::kBlock) {
            if (sub == 0) s_up[(turn & 1) * 256 + r] = (int8_t)up;
#pragma unroll
            for (int k = 0; k < kF4; ++k) {
              const float4 y = make_float4(x[k].x * mul, x[k].y * mul, x[k].z * mul, x[k].w * mul);
              uint2 hi, lo;
              hi.x = pack2(y.x, y.y, __half());
              hi.y = pack2(y.z, y.w, __half());
              const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
              const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
              lo.x = pack2(y.x - h0.x, y.y - h0.y, __half());
              lo.y = pack2(y.z - h1.x, y.w - h1.y, __half());
              const int f4 = 4 * k + sub;  // float4 of the row: half a piece
              uint8_t* dst = sq + (r / Cfg::kBlock) * kParts * Cfg::kQTile + at(r % Cfg::kBlock, f4 >> 1, kHalfQ) + (f4 & 1) * 8;
              *reinterpret_cast<uint2*>(dst) = hi;
              *reinterpret_cast<uint2*>(dst + Cfg::kQTile) = lo;
            }
          }
        }
        ptx::fence_proxy_async();
        ptx::mbar_arrive(q_full);
        if (lw == 2) {
          stop = !__all_sync(0xffffffffu, ok);
          if (stop) break;
        }
      }
      if (lw < 2) {
        const int* table = a.batch.table + (long long)it.seq * a.batch.table_stride;
        const C* kbase = static_cast<const C*>(a.k_pages) + it.head * a.pg.head_stride + pc * 8;
        const C* vbase = static_cast<const C*>(a.v_pages) + it.head * a.pg.head_stride + pc * 8;
        constexpr int kLook = kPos / Cfg::kLoaders;  // positions that a thread looks up
        // a tile's boxes: lane i holds the page of box i, looked up a tile ahead
        const int boxes = box_rows ? kPos / box_rows : 0;
        auto box_page = [&](int j) {
          const int pos = it.first + j * kPos + lane * box_rows;
          return lane < boxes && j < it.tiles && pos < it.len ? table[pos / a.pg.page_size] : -1;
        };
        int bpage = box_page(0);
        for (int j = 0; j < it.tiles; ++j) {
          const int tile0 = it.first + j * kPos;
          if (boxes && tile0 + kPos <= it.len &&
              __all_sync(0xffffffffu, lane >= boxes || (bpage >= 0 && bpage < a.pg.num_pages))) {
            if (np) flush();
            ok = __all_sync(0xffffffffu, ok) != 0;
            if (lw == 0) {
              if (lane == 0) *reinterpret_cast<uint4*>(s_bad + ((tiles + j) & 7) * 4) = make_uint4(0, 0, 0, 0);
#pragma unroll 1
              for (int kv = 0; kv < 2; ++kv, ++entry) {
                const uint32_t st = entry % kStages;
                ok = ok && __all_sync(0xffffffffu, wait(empty + st, ((entry / kStages) & 1) ^ 1));
                if (!ok) continue;
                if (lane == 0) ptx::mbar_arrive_expect_tx(full + st, Cfg::kStage);
                __syncwarp();
                if (lane < boxes) {
                  const int slot = (tile0 + lane * box_rows) % a.pg.page_size;
                  const uint32_t dst = ptx::smem_addr(ring + st * Cfg::kStage) + lane * box_rows * 128;
#pragma unroll
                  for (int h = 0; h < D / 64; ++h)
                    tma_4d(dst + h * kHalfKV, kv ? &vmap : &kmap, 64 * h, slot, it.head, bpage, full + st);
                }
              }
            } else {
              entry += 2;
            }
            bpage = box_page(j + 1);
            continue;
          }
          bpage = box_page(j + 1);
          stop = ptx::named_bar_or(1, Cfg::kLoaders, !ok);  // the previous tile's offsets have been read
          if (stop) break;
#pragma unroll
          for (int i = 0; i < kLook; ++i) {
            const int pos = tile0 + i * Cfg::kLoaders + lt;
            long long off = -1;
            if (pos < it.len) {
              const int page = table[pos / a.pg.page_size];
              if (page >= 0 && page < a.pg.num_pages)
                off = page * a.pg.page_stride + (long long)(pos % a.pg.page_size) * a.pg.slot_stride;
              else if (a.status)
                *a.status = 5u;
            }
            const unsigned bad = __ballot_sync(0xffffffffu, off < 0);
            s_off[i * Cfg::kLoaders + lt] = off;
            if (lane == 0) s_bad[((tiles + j) & 7) * 4 + i * (Cfg::kLoaders / 32) + lw] = bad;
          }
          ptx::named_bar(1, Cfg::kLoaders);
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            const uint32_t st = entry % kStages;
            const bool free = wait_free(empty + st, ((entry / kStages) & 1) ^ 1);
            ok = ok && free;
            const uint32_t dst = ptx::smem_addr(ring + st * Cfg::kStage);
            const C* basep = kv ? vbase : kbase;
#pragma unroll 8
            for (int r = pr; ok && r < kPos; r += kHop) {
              const long long o = s_off[r];
              cp_async_16(dst + at(r, pc, kHalfKV), basep + (o < 0 ? 0 : o), o >= 0);
            }
            landed(full + st);
            ++entry;
          }
        }
      }
      tiles += it.tiles;
      ++turn;
    }
    flush();
  } else {
    // ------------------------------------------------------------------ softmax
    const int x = warp >> 2, r = (warp & 3) * 32 + lane, rr = x * Cfg::kBlock + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = t_s[x] + lanes, to = t_o[x] + lanes;
    const float scale2 = a.scale * kLog2e;
    uint32_t seen = 0, o_turn = 0, tiles = 0, turn = 0;
    bool ok = true;  // the same for the whole warp
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    for (int w = 0; ok && w * ctas < items; ++w) {
      const int idx = item_of(w);
      if (idx >= items) continue;
      const ItemRange it = item_at<kPos, Cfg::kRows>(a, map, tokens, splits, idx, lane);
      const int block_rows = it.rows - x * Cfg::kBlock;  // of this block, if positive
      const bool live = r < block_rows;
      const int tok = rr / a.group, p0 = it.len - it.n + it.tok0;
      const int plast = live ? p0 + tok : -1;
      const int pfirst = a.window > 0 ? max(0, plast + 1 - a.window) : 0;
      // every row of the block sees the positions from seen_from to seen_to
      const int seen_to = p0 + x * Cfg::kBlock / a.group;
      const int top = p0 + (min(it.rows, (x + 1) * Cfg::kBlock) - 1) / a.group;
      const int seen_from = a.window > 0 ? max(0, top + 1 - a.window) : 0;
      const bool busy = block_rows > 0 && it.tiles > 0;
      float m = -INFINITY, l = 0.0f;
      if (busy) {
        float c = scale2;
        for (int j = 0; j < it.tiles; ++j) {
          ok = wait_all(s_full + x, seen & 1);
          ++seen;
          if (!ok) break;
          umma::tc_fence_after();
          if (kHalves && j == 0) c = scale2 * __uint_as_float((uint32_t)(127 - s_up[(turn & 1) * 256 + rr]) << 23);
          float s[kPos];
#pragma unroll
          for (int i = 0; i < kPos / 32; ++i) tmem_ld32(ts + 32 * i, s + 32 * i);
          umma::tmem_wait_ld();
          const int pos0 = it.first + j * kPos;
          const uint4 b4 = *reinterpret_cast<const uint4*>(s_bad + ((tiles + j) & 7) * 4);
          if (pos0 < seen_from || pos0 + kPos - 1 > seen_to || (b4.x | b4.y | b4.z | b4.w)) {
            const uint32_t bw[4] = {b4.x, b4.y, b4.z, b4.w};
            const int hi = plast - pos0, lo = pfirst - pos0;
#pragma unroll
            for (int i = 0; i < kPos; ++i)
              if (i > hi || i < lo || ((bw[i >> 5] >> (i & 31)) & 1)) s[i] = -INFINITY;
          }
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int i = 4; i + 7 < kPos; i += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], fmaxf(s[i + q], s[i + 4 + q]));
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], s[kPos - 4 + q]);
          const float top_x = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
          const bool raise = top_x > m + kSlack || (m == -INFINITY && top_x > m);
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = fmaxf(m, top_x);
            const float f = mn == -INFINITY ? 1.0f : exp2_approx(m - mn);
            m = mn;
            l *= f;
            if (j > 0) {
#pragma unroll 1
              for (int i = 0; i < D / 16; ++i) {
                float o[16];
                tmem_ld16(to + 16 * i, o);
                umma::tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] *= f;
                tmem_st16(to + 16 * i, reinterpret_cast<const uint32_t*>(o));
              }
            }
          }
          const float sub = (m == -INFINITY ? 0.0f : m) - kShift;
          const float2 c2 = make_float2(c, c), sub2 = make_float2(-sub, -sub);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int b = 0; b < kPos / 64; ++b) {  // 64 scores become 32 columns of weights (and 32 of lower halves)
            uint32_t hi[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float2 y = __ffma2_rn(make_float2(s[64 * b + 2 * i], s[64 * b + 2 * i + 1]), c2, sub2);
              const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
              sum[i & 1] = __fadd2_rn(sum[i & 1], e);
              hi[i] = pack2(e.x, e.y, C());
              if constexpr (kHalves) {
                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
                s[64 * b + i] = __uint_as_float(pack2(e.x - h.x, e.y - h.y, __half()));
              }
            }
            tmem_st32(ts + kParts * 32 * b, hi);
            if constexpr (kHalves) tmem_st32(ts + 64 * b + 32, reinterpret_cast<const uint32_t*>(s + 64 * b));
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tmem_wait_st();
          umma::tc_fence_before();
          ptx::mbar_arrive(p_ready + x);
        }
        if (ok) {
          ok = wait_all(o_full + x, o_turn & 1);
          ++o_turn;
          umma::tc_fence_after();
        }
      }
      if (!ok) break;
      tiles += it.tiles;
      turn += it.tiles > 0;
      if (block_rows <= 0) continue;
      // ---- the rows' results
      const int row = it.q0 + it.tok0 + tok, h = it.head * a.group + rr - tok * a.group;
      bool again = false;
      const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
      T* out = static_cast<T*>(a.out) + (long long)row * a.out_stride + h * D;
      float* num = it.slot < 0 ? nullptr : chunk_num(work) + ((size_t)it.slot * Cfg::kRows + rr) * D;
      for (int i = 0; i < D / 32; ++i) {
        float o[32];
        if (busy) {
          tmem_ld32(to + 32 * i, o);
          umma::tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.0f;
        }
        float z = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) z = __fmaf_rn(o[k], 0.0f, z);
        again |= z != 0.0f;  // 0, or NaN where a numerator is not finite
        if (live) {
          if (it.slot < 0) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              float y[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) y[q] = o[k + q] * inv;
              store_elems(out + 32 * i + k, y);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(num + 32 * i + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
      }
      again |= !(l * 0.0f == 0.0f);
      // rows with non-finite numerators, one after the other by the whole warp
      unsigned redo = __ballot_sync(0xffffffffu, live && again);
      if (redo) {
        const int* table = a.batch.table + (long long)it.seq * a.batch.table_stride;
        for (; redo; redo &= redo - 1) {
          const int src = __ffs(redo) - 1;
          const int r2 = rr - lane + src, tok2 = r2 / a.group;
          const int last2 = __shfl_sync(0xffffffffu, plast, src), first2 = __shfl_sync(0xffffffffu, pfirst, src);
          const long long row2 = it.q0 + it.tok0 + tok2;
          const int h2 = it.head * a.group + r2 - tok2 * a.group;
          float o2[D / 32], m2, l2;
          row_attend<T, C, D>(a, static_cast<const T*>(a.q) + row2 * a.q_stride + h2 * D, table, it.head, max(first2, it.first),
                              min(last2, it.first + it.tiles * kPos - 1), scale2, o2, m2, l2);
          if (lane == src) {
            m = m2;
            l = l2;
          }
          const float inv2 = l2 == 0.0f ? 0.0f : __fdiv_rn(1.0f, l2);
          for (int i = 0; i < D / 32; ++i) {
            if (it.slot < 0)
              static_cast<T*>(a.out)[row2 * a.out_stride + h2 * D + lane + 32 * i] = from_f32(__fmul_rn(o2[i], inv2), T());
            else
              chunk_num(work)[((size_t)it.slot * Cfg::kRows + r2) * D + lane + 32 * i] = o2[i];
          }
        }
      }
      if (live) {
        if (it.slot >= 0)
          chunk_ml(work)[(size_t)it.slot * Cfg::kRows + rr] = make_float2(m, l);
        else if (a.lse)
          a.lse[(long long)row * a.hq + h] = l == 0.0f ? -INFINITY : (m - kShift + log2f(l)) * kLn2;
      }
    }
  }
  // ---- end: every role has left its loop
  umma::tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag && a.status) *a.status = 6u;
  if (warp == 8) {
    umma::tc_fence_after();
    umma::tmem_relinquish();
    umma::tmem_dealloc(tmem, 512);
  }
}

// Split items: block (tile and head, group of 8 rows) adds an item's parts in order, a warp a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const AttnArgs a, void* work, int tokens, int splits) {
  constexpr int kRows = 256, E = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  const ItemMap map = item_map(a, tokens, lane);
  const int idx = blockIdx.x * splits;
  if ((long long)map.total * a.hk > (long long)gridDim.x || idx >= map.total * a.hk * splits) return;
  const ItemRange it = item_at<128, kRows>(a, map, tokens, splits, idx, lane);
  if (r >= it.rows) return;
  float mm = -INFINITY;
  for (int s = 0; s < splits; ++s) mm = fmaxf(mm, chunk_ml(work)[(size_t)(idx + s) * kRows + r].x);
  const float mu = mm == -INFINITY ? 0.0f : mm;
  float v[E], l = 0.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] = 0.0f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float2 ml = chunk_ml(work)[(size_t)(idx + s) * kRows + r];
    const float f = exp2_approx(ml.x - mu);
    l = __fmaf_rn(ml.y, f, l);
    const float* p = chunk_num(work) + ((size_t)(idx + s) * kRows + r) * D + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = __fmaf_rn(p[j], f, v[j]);
  }
  const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
  const int tok = r / a.group;
  const long long row = it.q0 + it.tok0 + tok;
  const int h = it.head * a.group + r - tok * a.group;
  T* out = static_cast<T*>(a.out) + row * a.out_stride + h * D + lane * E;
#pragma unroll
  for (int j = 0; j < E; ++j) out[j] = from_f32(v[j] * inv, T());
  if (a.lse && lane == 0) a.lse[row * a.hq + h] = l == 0.0f ? -INFINITY : (mm - kShift + log2f(l)) * kLn2;
}

}  // namespace paged
}  // namespace qora
