// paged_chunk.cuh — attention of chunks of new rows over their paged caches on the tensor
// cores (tcgen05, TMEM). The time is the two products, 4 D operations per (query head, row,
// position).
//
// Item. Two blocks (X = 0, 1) of up to 128 packed rows of one (sequence, kv head): tokens
// times the kv head's query heads (row r: token r / group, head r % group), so that grouped
// heads share every K and V tile. Each block has its scores and its numerators (D columns)
// in TMEM; K and V tiles of 128 positions (64 of an f32 cache) feed both. Where the items
// leave half of the CTAs idle, the positions of each are split evenly and chunk_join_kernel
// adds the parts in order; a part has one tile at least (8 short prompts in 18.5 us, with
// empty parts 20.6 us; parts of two tiles or more: 14 prompts over 500 positions in 23.7 us
// instead of 20.6 us). Items are taken from the last rows (the longest runs of positions
// of one prompt) on, in alternating direction. Equal shares of one line of tiles, as the token
// kernel has, cost more in items begun twice than they even out (8,192 rows in 314 us instead
// of 264 us; 240 items of a mixed batch in 126 us instead of 99 us).
//
// Roles (one CTA per SM):
//   warps 0-3, 4-7   softmax of block 0, 1: a thread owns a row, keeps its scores in
//                    registers, writes the weights back over them in TMEM as the next
//                    product's operand
//   warp 8           issues the products: S_X = Q_X K^T; O_X += P_X V with P_X from TMEM
//   warps 9, 10      16-bit caches: load K and V into the 128-byte-swizzled tiles that the
//                    products read. A tile whose 128 positions all exist comes by TMA, a page
//                    (or 128 rows of one) per copy, where the page size divides 128 or is a
//                    multiple of it; other tiles are copied by cp.async in 16-byte pieces,
//                    the page looked up per position (slots past the end become zeros)
//   warp 11          16-bit rows: loads q by TMA, the rows packed by its box (f32 rows are
//                    loaded and split by the softmax warps)
//   warps 9-12, 13-16   f32 caches: load K, V, and split them
// While one block's weights are computed the other block's products run. S_X(j + 1) is
// issued behind O_X(j), which still reads P_X(j) from the columns it overwrites: one
// thread's products execute in order.
//
// f32 operands are split into binary16 upper and lower halves (22 bits) after scaling by a
// power of two: q by row, K and V by tile (largest value in [2^13, 2^14); a value less than
// 2^-15 of that has fewer bits, its error stays within 2^-38 of the largest). The weights are
// split too. Upper x upper, lower x upper and upper x lower are multiplied: two products
// instead of one for an f16 cache, three for an f32 cache. The scale of K goes into the
// scores' scale. 16-bit rows' weights are rounded to the rows' type, which adds about as much
// error as the rounding of the result: a lower part as well would take 8,192 binary16 rows from
// 258 to 351 us (rms error 2.14e-5; 1.64e-5 with it), mixed bf16 chunks from 98 to 126 us. V's
// scales differ from tile to tile; the numerators count in the smallest so far (the largest
// values) and the weights of other tiles are scaled down to it.
//
// The running maximum is raised only when it grows by more than 2^kSlack: then the
// numerators in TMEM are scaled, which is rare after the first tiles. Masked scores become
// -inf before the maximum. Rows that meet a non-finite value (a weight of zero times an
// infinite value of V, or a row whose own scores are) are computed again in f32 when the CTA's
// roles have ended (rows_attend). So are rows of an f32 cache that meet a tile of K or V whose
// rows differ by more than 2^14 in size, a tile of V 2^12 below the largest before it, or
// growth of V by more than 2^60. This is for correctness alone, and 15 to 90 times as slow:
// where every row is concerned, 1,021 f32 rows take 0.84 ms instead of 58 us, 512 f32 rows
// over 8,192 binary16 positions 4.4 ms instead of 86 us, 2,048 binary16 rows 4.2 ms instead of
// 47 us (one row and one position at a time, between the tiles, took 10, 41 and 40 ms).
//
// Measured, 16 query heads over 4 kv heads of 128, short runs of the same call (in brackets:
// consecutive calls on changing inputs, under the power cap): a prompt of 8,192 binary16 rows,
// 275 GFLOP, in 257 to 273 us = 1.01 to 1.07 PFLOP/s (301 us); 512 f32 rows over 8,192 binary16 positions in
// 83 us (89 us); a prompt of 1,021 rows, all f32, in 56 us (61 us).
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
  static constexpr bool kHalves = sizeof(T) == 4;  // f32 rows: q and the weights in two halves
  static constexpr bool kWide = sizeof(C) == 4;    // f32 cache: K and V in two halves
  using M = typename std::conditional<kWide, __half, C>::type;  // what the tensor cores multiply
  static constexpr int kQParts = kHalves ? 2 : 1, kParts = kWide ? 2 : 1;
  static constexpr int kBlock = 128;            // rows of a block
  static constexpr int kPos = kWide ? 64 : 128;  // positions of a tile
  static constexpr int kQTile = kBlock * D * 2;
  static constexpr int kQBytes = 2 * kQParts * kQTile;  // [block][part]
  static constexpr int kTile = kPos * D * 2;            // one part of a K or V tile
  static constexpr int kStage = kParts * kTile;
  static constexpr int kOther = 1024 /* offsets */ + 1024 /* barriers, masks, scales */;
  static constexpr int kLimit = 227 * 1024 - 1024 - kOther;
  static constexpr int kFit = (kLimit - kQBytes) / kStage;
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static_assert(kStages >= 3, "a K tile, a V tile and the next K tile");
  static constexpr int kLag = kStages >= 4 ? 2 : 1;  // copies in flight behind the newest: at most kStages - 2
  static constexpr int kSmem = kQBytes + kStages * kStage + kOther + 1024;
  static constexpr int kLoaders = kWide ? 128 : 64;  // threads that load (f32 cache: each of K and V)
  static constexpr int kThreads = kWide ? 544 : 384;
  // Scores that a softmax thread holds at once. 16-bit rows: the whole tile's (8,192 rows in
  // 267 us; 32 at a time, read twice: 300 us, each read waits). f32 rows: 32, in small loops
  // (512 rows over 8K positions in 85 us; the whole tile's: 92 us, registers spill).
  static constexpr int kCols = kHalves ? 32 : kPos;
  // f32 rows: after so many tiles the numerators are added to those of the tiles before them
  // in registers, rounded to nearest. The tensor cores' own sums are cut: 16 tiles in a row
  // were off by 5.8e-6 of the result, where f32 sums are off by 1.8e-6.
  static constexpr int kFlush = 4;
};
constexpr int kChunkMaxCtas = 160;
// Turns of a CTA whose marks for recomputing are told apart; one more turn shares the mark of the
// first, and the rows of both are computed again.
constexpr int kRedoTurns = 512;
// Longest wait on a barrier; only a fault reaches it. (Rows are recomputed, which takes as long
// as the rows are long, when the CTA's roles have ended and nothing waits.)
constexpr unsigned long long kWaitNs = 2000000000ull;

constexpr int kChunkMaxParts = kChunkMaxCtas;  // parts of split items in one call: no more than CTAs
constexpr int kChunkMaxSplit = kChunkMaxCtas / 2;  // split items, of two turns at least
// Workspace of split items: [tile and head] (first row, tokens, kv head,
// slots << 16 | parts), [part] (maximum,
// sum) of 256 rows, numerators [part][256][D].
__host__ __device__ inline int4* chunk_rec(void* p) { return static_cast<int4*>(p); }
__host__ __device__ inline float2* chunk_ml(void* p) {
  return reinterpret_cast<float2*>(static_cast<char*>(p) + kChunkMaxParts * 16);
}
__host__ __device__ inline float* chunk_num(void* p) {
  return reinterpret_cast<float*>(static_cast<char*>(p) + kChunkMaxParts * 16 + (size_t)kChunkMaxParts * 256 * 8);
}

// f32 rows: a CTA's numerators so far, float4s [D / 4][256 rows]
template <int D>
__host__ __device__ inline float4* chunk_acc(void* p, int cta) {
  return reinterpret_cast<float4*>(chunk_num(p) + (size_t)kChunkMaxParts * 256 * D) + (size_t)cta * 64 * D;
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
// 16 lanes x 32 columns: v[4 n + 0, 1] lane (thread / 4), columns 8 n + 2 (thread % 4) + 0, 1;
// v[4 n + 2, 3] eight lanes on
QORA_DEV void tmem_ld_frag(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// box at (x, head, row) of q
QORA_DEV void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(head), "r"(row), "r"(ptx::smem_addr(bar))
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
  int seq, q0, n, len, head, tok0, toks;  // sequence, its first row, new rows, positions; kv head, first token, tokens
  int lo, first;                          // first attended position, first position of the first tile
  int tiles;                              // tiles of this part
  int part, parts;                        // partial slot, or -1: the item is whole; the item's parts
};

// The sequences' row tiles as a warp holds them: a lane sums a run of neighbouring sequences.
// Rows that no two sequences share make at most 2^24 / tokens + 2^20 tiles, below kManyTiles; a
// lane that counts more (overlapping ranges) stays there, so that the warp's sum cannot wrap
// and the batch is refused as having too many.
constexpr int kManyTiles = 1 << 25;
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
  return q1 - q0 <= a.few ? 0 : (q1 - q0 + tokens - 1) / tokens;
}
QORA_DEV ItemMap item_map(const AttnArgs& a, int tokens, int lane) {
  ItemMap m;
  m.per = (a.batch.seqs + 31) >> 5;
  m.mine = 0;
#pragma unroll 4
  for (int j = 0; j < m.per; ++j) {
    const int s = lane * m.per + j;
    if (s < a.batch.seqs) m.mine = min(kManyTiles, m.mine + seq_tiles(a, s, tokens));
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
template <int kPos>
QORA_DEV ItemRange item_at(const AttnArgs& a, const ItemMap& m, int tokens, int splits, int idx, int lane) {
  const unsigned th = (unsigned)idx / (unsigned)splits, split = (unsigned)idx - th * splits;
  const int back = (int)(th / (unsigned)a.hk);
  const int tile = m.total - 1 - back;  // the longest runs of positions first
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
  r.head = (int)th - back * a.hk;
  r.tok0 = (tile - base) * tokens;
  r.toks = min(tokens, r.n - r.tok0);
  const int p0 = r.len - r.n + r.tok0;              // position of the first row
  const int hi = min(r.len, p0 + r.toks);           // positions [lo, hi) are attended to
  const int lo = first_seen(a, p0);
  r.lo = lo;
  const int t0 = lo / kPos, nt = hi > lo ? (hi - 1) / kPos + 1 - t0 : 0;
  r.parts = max(1, min(splits, nt));
  if (split >= (unsigned)r.parts) {  // a turn that the item has no use for
    r.toks = r.tiles = 0;
    r.part = -1;
    return r;
  }
  const int b = (int)((long long)split * nt / r.parts), e = (int)((long long)(split + 1) * nt / r.parts);
  r.first = (t0 + b) * kPos;
  r.tiles = e - b;
  r.part = r.parts > 1 ? idx : -1;
  return r;
}

// Up to four rows of one kv head by a warp, in f32: row r over positions [from[r], to[r]], all
// within [lo, hi]; o[r]: lane's elements lane * D / 32 + i. Four positions at a time: K and V
// are read once for the four rows, and the 16 dot products are added up over the lanes
// together (lane / 8: row, lane / 2 % 4: position).
template <typename T, int E>
struct alignas(E * sizeof(T)) Piece {
  T v[E];
};
template <typename T, typename C, int D>
QORA_DEV void rows_attend(const AttnArgs& a, const T* const (&q)[4], const int (&from)[4], const int (&to)[4],
                          int lo, int hi, const int* table, int head, float scale2,
                          float (&o)[4][D / 32], float& m, float& l) {
  constexpr int E = D / 32, R = 4, P = 4;
  const int lane = threadIdx.x & 31, mine = lane >> 3, which = (lane >> 1) & 3;
  float qv[R][E];
  int first = from[0], last = to[0];  // of the lane's row
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const Piece<T, E> x = *reinterpret_cast<const Piece<T, E>*>(q[r] + lane * E);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      qv[r][e] = to_f32(x.v[e]);
      o[r][e] = 0.0f;
    }
    if (mine == r) first = from[r], last = to[r];
  }
  m = -INFINITY;
  l = 0.0f;
#pragma unroll 1
  for (int base = lo; base <= hi; base += min(32, hi - base + 1)) {
    long long off = -1;
    if (lane <= hi - base) {
      const int pos = base + lane, pi = pos / a.pg.page_size, page = table[pi];
      if (page >= 0 && page < a.pg.num_pages)
        off = page * a.pg.page_stride + (long long)(pos - pi * a.pg.page_size) * a.pg.slot_stride + (long long)head * a.pg.head_stride;
    }
    const unsigned there = __ballot_sync(0xffffffffu, off >= 0);
#pragma unroll 1
    for (int j = 0; j < 32 && j <= hi - base; j += P) {
      Piece<C, E> k[P], v[P];
      float s[R * P];
#pragma unroll
      for (int x = 0; x < P; ++x) {
        const long long at = __shfl_sync(0xffffffffu, off, j + x);
        k[x] = v[x] = Piece<C, E>{};
        if (at >= 0) {
          k[x] = *reinterpret_cast<const Piece<C, E>*>(static_cast<const C*>(a.k_pages) + at + lane * E);
          v[x] = *reinterpret_cast<const Piece<C, E>*>(static_cast<const C*>(a.v_pages) + at + lane * E);
        }
      }
#pragma unroll
      for (int x = 0; x < P; ++x)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float d = 0.0f;
#pragma unroll
          for (int e = 0; e < E; ++e) d = __fmaf_rn(qv[r][e], to_f32(k[x].v[e]), d);
          s[P * r + x] = d;
        }
      // halving the number of sums while doubling the lanes that each of them covers
#pragma unroll
      for (int n = 8; n > 0; n >>= 1) {
        const bool up = lane & (2 * n);
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float give = up ? s[i] : s[i + n], keep = up ? s[i + n] : s[i];
          s[i] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, 2 * n));
        }
      }
      float d = __fmul_rn(__fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], 1)), scale2);
      const int pos = base + j + which;
      if (!((there >> (j + which)) & 1) || pos < first || pos > last) d = -INFINITY;
      float top = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 2));
      top = fmaxf(m, fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4)));
      const float mu = top == -INFINITY ? 0.0f : top;  // a NaN score does not raise the maximum: its weight is NaN
      const float w = exp2f(d - mu + kShift), c = exp2f(m - mu);
      m = top;
      l = __fmaf_rn(l, c, w);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float cr = __shfl_sync(0xffffffffu, c, 8 * r);
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] *= cr;
#pragma unroll
        for (int x = 0; x < P; ++x) {
          const float wx = __shfl_sync(0xffffffffu, w, 8 * r + 2 * x);
          if (wx != 0.0f) {  // the same for the whole warp
#pragma unroll
            for (int e = 0; e < E; ++e) o[r][e] = __fmaf_rn(wx, to_f32(v[x].v[e]), o[r][e]);
          }
        }
      }
    }
  }
  l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 2));
  l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 4));
}

// Four consecutive f32 values, scaled, as binary16 upper and lower halves.
QORA_DEV void split4(const float4& x, float mul, uint2& hi, uint2& lo) {
  const float4 y = make_float4(x.x * mul, x.y * mul, x.z * mul, x.w * mul);
  hi.x = pack2(y.x, y.y, __half());
  hi.y = pack2(y.z, y.w, __half());
  const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
  const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
  lo.x = pack2(y.x - h0.x, y.y - h0.y, __half());
  lo.y = pack2(y.z - h1.x, y.w - h1.y, __half());
}
// e such that 2^e brings a largest magnitude (its bits) to [2^13, 2^14); 2^e and 2^-e are normal
QORA_DEV int scale_up(uint32_t bits) { return min(126, 140 - (int)(bits >> 23)); }
QORA_DEV float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
constexpr int kNoScale = 127;  // a tile of zeros
// Two halves of a value 2^-kMaxSpread of the tile's largest still have 22 bits; weights that
// are scaled down by 2^kMaxLift have 20 or more. Numerators that were scaled down by
// 2^kMaxDrop are still far from f32's subnormals. Beyond that the rows are computed again.
constexpr int kMaxSpread = 14, kMaxLift = 12, kMaxDrop = 60, kSpreadMark = 1024;

// byte offset of 16-byte piece `piece` of a row in a tile whose 64-element halves are `half` bytes apart
QORA_DEV int tile_at(int row, int piece, int half) { return (piece >> 3) * half + row * 128 + (((piece & 7) ^ (row & 7)) << 4); }

template <typename T, typename C, int D>
__global__ void __launch_bounds__(ChunkCfg<T, C, D>::kThreads, 1)
    chunk_kernel(const AttnArgs a, void* work, bool split, int max_tiles, int box_rows,
                 const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap) {
  using Cfg = ChunkCfg<T, C, D>;
  using M = typename Cfg::M;
  constexpr bool kHalves = Cfg::kHalves, kWide = Cfg::kWide;
  constexpr int kCols = Cfg::kCols;
  constexpr int kPos = Cfg::kPos, kStages = Cfg::kStages, kLag = Cfg::kLag, kLoaders = Cfg::kLoaders;
  constexpr int kHalfQ = Cfg::kBlock * 128, kHalfKV = kPos * 128;  // bytes from one 64-element half to the next
  constexpr int kProducts = kWide ? 3 : kHalves ? 2 : 1;           // (part of the left, of the right operand)
  // the small products first: the tensor cores cut every sum of f32 accumulators short
  constexpr int kLeft[3] = {kProducts > 1 ? 1 : 0, 0, 0}, kRight[3] = {0, kProducts > 2 ? 1 : 0, 0};
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (ptx::smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* const sq = smem;
  uint8_t* const ring = smem + Cfg::kQBytes;
  long long* const s_off = reinterpret_cast<long long*>(ring + kStages * Cfg::kStage);  // [128], or [K, V][64]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(s_off + 128);
  uint64_t *const full = bars, *const empty = bars + 8, *const q_full = bars + 16, *const s_full = bars + 18,
           *const p_ready = bars + 20, *const o_full = bars + 22, *const q_empty = bars + 24, *const done = bars + 25;
  uint32_t* const s_bad = reinterpret_cast<uint32_t*>(bars + 26);  // [8 tiles][4] positions that there are not
  int* const s_exp = reinterpret_cast<int*>(s_bad + 32);           // [8 tiles][K, V] scales of the tiles
  uint32_t* const s_max = reinterpret_cast<uint32_t*>(s_exp + 16);  // [K, V][4 warps]
  uint32_t* const s_low = s_max + 8;                                // [K, V][4 warps]
  uint32_t* const s_tmem = s_low + 8;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(s_tmem + 1);
  uint32_t* const s_redo = s_tmem + 2;  // [kRedoTurns / 4] softmax warps whose rows are computed again, a byte per turn

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int block_toks = Cfg::kBlock / a.group, tokens = 2 * block_toks;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full + i, 1);
      ptx::mbar_init(empty + i, 1);
    }
    ptx::mbar_init(q_empty, 1);
    for (int x = 0; x < 2; ++x) {
      ptx::mbar_init(q_full + x, kHalves ? 128 : 1);
      ptx::mbar_init(s_full + x, 1);
      ptx::mbar_init(p_ready + x, 128);
      ptx::mbar_init(o_full + x, 1);
    }
    ptx::mbar_init(done, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  for (int i = tid; i < kRedoTurns / 4; i += Cfg::kThreads) s_redo[i] = 0u;
  if (warp == 8) umma::tmem_alloc(s_tmem, 512);
  const ItemMap map = item_map(a, tokens, lane);
  umma::tc_fence_before();
  __syncthreads();
  umma::tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int ctas = (int)gridDim.x, cta = (int)blockIdx.x;
  // more row tiles than the rows can hold: the sequences' row ranges overlap
  const bool too_many = (long long)map.total * a.hk > max_tiles;
  if (too_many && tid == 0 && a.status) *a.status = 5u;
  const int whole = too_many ? 0 : map.total * a.hk;
  const int splits = split && whole ? max(1, ctas / whole) : 1, items = whole * splits;
  if (split && cta == 0) {  // no rows for the join where there is nothing to join
    for (int i = (splits > 1 ? whole : 0) + tid; i < min(max_tiles, kChunkMaxSplit); i += Cfg::kThreads)
      chunk_rec(work)[i] = make_int4(0, 0, 0, 0);
  }
  // item of turn w: alternating direction, so that long and short items pair up
  auto item_of = [&](int w) { return w * ctas + (w & 1 ? ctas - 1 - cta : cta); };
  // whether a block's numerators begin anew with tile j
  auto fresh = [&](int j) { return j == 0 || (kHalves && j % Cfg::kFlush == 0); };
  auto wait = [&](uint64_t* bar, uint32_t parity) { return umma::wait_bar(bar, parity, kWaitNs, abort_flag); };

  if (warp == 8) {
    // -------------------------------------------------------------------- products
    uint32_t tile = 0, q_turn[2] = {0, 0}, taken[2] = {0, 0};
    bool ok = true;
    const uint32_t q_k = desc_k(ptx::smem_addr(sq)), ring_k = desc_k(ptx::smem_addr(ring)),
                   ring_mn = desc_mn(ptx::smem_addr(ring), kHalfKV);
    constexpr uint32_t id_s = chunk_idesc<M>(kPos, false), id_o = chunk_idesc<M>(D, true);
    for (int w = 0; ok && w * ctas < items; ++w) {
      const int idx = item_of(w);
      if (idx >= items) continue;
      const ItemRange it = item_at<kPos>(a, map, tokens, splits, idx, lane);
      if (it.tiles == 0) continue;
      const int blocks = it.toks > block_toks ? 2 : 1;
      if (lane == 0) {
        // ring entries alternate K, V: entry e lies in stage e % kStages
        auto entry = [&](uint32_t e) { return wait(full + e % kStages, (e / kStages) & 1); };
        auto scores = [&](int x, uint32_t e) {
          const uint32_t kb = ring_k + (e % kStages) * (Cfg::kStage >> 4), qb = q_k + x * Cfg::kQParts * (Cfg::kQTile >> 4);
#pragma unroll
          for (int p = 0; p < kProducts; ++p)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_ss(tmem + x * 128, qb + kLeft[p] * (Cfg::kQTile >> 4) + (k / 4) * (kHalfQ >> 4) + (k % 4) * 2,
                     kb + kRight[p] * (Cfg::kTile >> 4) + (k / 4) * (kHalfKV >> 4) + (k % 4) * 2, id_s, p || k);
          umma::mma_commit(s_full + x);
        };
        ok = entry(tile * 2);
        for (int x = 0; ok && x < blocks; ++x) {
          ok = wait(q_full + x, q_turn[x] & 1);
          ++q_turn[x];
          umma::tc_fence_after();
          if (ok) scores(x, tile * 2);
        }
        if (ok) {
          umma::mma_commit(empty + (tile * 2) % kStages);
          for (int j = 0; ok && j < it.tiles; ++j) {
            const uint32_t ev = (tile + j) * 2 + 1, ek = ev + 1;
            const bool last = j + 1 == it.tiles;
            ok = entry(ev);
            const uint32_t vb = ring_mn + (ev % kStages) * (Cfg::kStage >> 4);
            for (int x = 0; ok && x < blocks; ++x) {
              ok = wait(p_ready + x, taken[x] & 1);
              ++taken[x];
              umma::tc_fence_after();
              if (!ok) break;
              // 32 weights are 16 columns, their lower halves the next 16
#pragma unroll
              for (int p = 0; p < kProducts; ++p)
#pragma unroll
                for (int k = 0; k < kPos / 16; ++k)
                  mma_ts(tmem + 256 + x * D, tmem + x * 128 + Cfg::kQParts * 16 * (k / 2) + kLeft[p] * 16 + (k % 2) * 8,
                         vb + kRight[p] * (Cfg::kTile >> 4) + k * (2048 >> 4), id_o,
                         p || k ? 1u : (uint32_t)!fresh(j));
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
    }
    // every product has completed before the TMEM and the tiles go
    if (lane == 0) {
      umma::mma_commit(done);
      umma::settle_bar(done, 0, kWaitNs);
    }
    __syncwarp();
  } else if (!kWide && warp == 11) {
    // -------------------------------------------------------------------- q of 16-bit rows
    if constexpr (!kHalves) {
      uint32_t turn = 0, loads[2] = {0, 0};
      for (int w = 0; w * ctas < items; ++w) {
        const int idx = item_of(w);
        if (idx >= items) continue;
        const ItemRange it = item_at<kPos>(a, map, tokens, splits, idx, lane);
        if (it.tiles == 0) continue;
        if (!__all_sync(0xffffffffu, wait(q_empty, (turn & 1) ^ 1))) break;
        const int blocks = it.toks > block_toks ? 2 : 1;
        if (lane == 0) {
          // a box is block_toks tokens x the group's heads x 64 elements: packed rows (rows
          // past the last token are other rows, or zeros: their results are not written)
          for (int x = 0; x < blocks; ++x) {
            ptx::mbar_arrive_expect_tx(q_full + x, block_toks * a.group * D * 2);
            for (int h = 0; h < D / 64; ++h)
              tma_3d(ptx::smem_addr(sq + x * Cfg::kQTile + h * kHalfQ), &qmap, 64 * h, it.head * a.group,
                     it.q0 + it.tok0 + x * block_toks, q_full + x);
            ++loads[x];
          }
        }
        __syncwarp();
        ++turn;
      }
      // every copy has landed before the shared memory goes
      if (lane == 0)
        for (int x = 0; x < 2; ++x)
          if (loads[x]) umma::settle_bar(q_full + x, (loads[x] - 1) & 1, kWaitNs);
    }
  } else if (warp > 8) {
    // -------------------------------------------------------------------- K and V
    const int team = kWide ? (warp - 9) >> 2 : 0;          // f32 cache: 0 loads K, 1 loads V
    const int lt = tid - 9 * 32 - team * 128, lw = lt >> 5;  // thread and warp of the team
    const int bar_id = 1 + team;
    uint32_t entry = kWide ? team : 0, tiles = 0;
    bool ok = true, stop = false;  // this thread's waits ended in time; the team's threads agree to stop
    uint64_t* pend[kLag];          // barriers of the copies still in flight
    int np = 0;
    uint32_t copied = 0, odd = 0;  // stages that TMA filled last, and the parity of that phase
    // one arrival for the team's threads, each of which has fenced its own writes; none on a
    // stage that did not come free (null)
    auto arrive = [&](uint64_t* bar) {
      ptx::named_bar(bar_id, kLoaders);
      if (lt == 0 && bar) ptx::mbar_arrive(bar);
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
      if (np && ptx::named_bar_or(bar_id, kLoaders, !ptx::mbar_try_wait(bar, parity))) flush();
      return wait(bar, parity);
    };
    for (int w = 0; !stop && w * ctas < items; ++w) {
      const int idx = item_of(w);
      if (idx >= items) continue;
      const ItemRange it = item_at<kPos>(a, map, tokens, splits, idx, lane);
      if (it.tiles == 0) continue;
      const int* table = a.batch.table + (long long)it.seq * a.batch.table_stride;
      const C* base = static_cast<const C*>(team ? a.v_pages : a.k_pages) + it.head * a.pg.head_stride;
      const C* vbase = static_cast<const C*>(a.v_pages) + it.head * a.pg.head_stride;
      // a tile's boxes: lane i holds the page of box i, looked up a tile ahead. Entries before
      // the first attended position may be those of released pages: where they name no page,
      // the tile is copied by position, and they are not looked at
      const int boxes = box_rows ? kPos / box_rows : 0;
      auto box_page = [&](int j) {
        const int pos = it.first + j * kPos + lane * box_rows;
        return lane < boxes && j < it.tiles && pos < it.len ? table[pos / a.pg.page_size] : -1;
      };
      int bpage = box_page(0);
      for (int j = 0; j < it.tiles; ++j) {
        const int tile0 = it.first + j * kPos, ring8 = (tiles + j) & 7;
        if constexpr (!kWide) {
          if (boxes && kPos <= it.len - tile0 &&
              __all_sync(0xffffffffu, lane >= boxes || (bpage >= 0 && bpage < a.pg.num_pages))) {
            if (np) flush();
            ok = __all_sync(0xffffffffu, ok) != 0;
            if (lw == 0) {
              if (lane == 0) *reinterpret_cast<uint4*>(s_bad + ring8 * 4) = make_uint4(0, 0, 0, 0);
#pragma unroll 1
              for (int kv = 0; kv < 2; ++kv, ++entry) {
                const uint32_t st = entry % kStages;
                ok = ok && __all_sync(0xffffffffu, wait(empty + st, ((entry / kStages) & 1) ^ 1));
                if (!ok) continue;
                if (lane == 0) ptx::mbar_arrive_expect_tx(full + st, Cfg::kStage);
                copied |= 1u << st;
                if ((entry / kStages) & 1)
                  odd |= 1u << st;
                else
                  odd &= ~(1u << st);
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
        }
        stop = ptx::named_bar_or(bar_id, kLoaders, !ok);  // the previous tile's offsets have been read
        if (stop) break;
        for (int i = lt; i < kPos; i += kLoaders) {
          const int pos = tile0 + i;
          long long off = -1;
          if (pos >= it.lo && pos < it.len) {
            const int page = table[pos / a.pg.page_size];
            if (page >= 0 && page < a.pg.num_pages)
              off = page * a.pg.page_stride + (long long)(pos % a.pg.page_size) * a.pg.slot_stride;
            else if (a.status)
              *a.status = 5u;
          }
          const unsigned bad = __ballot_sync(0xffffffffu, off < 0);
          s_off[team * kPos + i] = off;
          if (lane == 0 && team == 0) s_bad[ring8 * 4 + (i >> 5)] = bad;
        }
        if (kWide && team == 0 && lt == 127) s_bad[ring8 * 4 + 2] = s_bad[ring8 * 4 + 3] = 0u;
        ptx::named_bar(bar_id, kLoaders);
        if constexpr (!kWide) {
          constexpr int kPieces = D * 2 / 16;      // 16-byte pieces of a row
          constexpr int kHop = kLoaders / kPieces;  // rows that the team copies at once
          const int pr = lt / kPieces, pc = lt % kPieces;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv, ++entry) {
            const uint32_t st = entry % kStages;
            const bool free = wait_free(empty + st, ((entry / kStages) & 1) ^ 1);
            ok = ok && free;
            const uint32_t dst = ptx::smem_addr(ring + st * Cfg::kStage);
            const C* basep = (kv ? vbase : base) + pc * 8;
#pragma unroll 8
            for (int r = pr; ok && r < kPos; r += kHop) {
              const long long o = s_off[r];
              cp_async_16(dst + tile_at(r, pc, kHalfKV), basep + (o < 0 ? 0 : o), o >= 0);
            }
            if (free) copied &= ~(1u << st);
            landed(ok ? full + st : nullptr);
          }
        } else {
          constexpr int kF4 = D / 4;            // float4s of a row
          constexpr int kHop = kLoaders / kF4;  // rows at once
          constexpr int kN = kPos / kHop;
          const int f4 = lt % kF4, pr = lt / kF4;
          float4 x[kN];
          uint32_t mx = 0;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const long long o = s_off[team * kPos + pr + i * kHop];
            x[i] = o >= 0 ? *reinterpret_cast<const float4*>(base + o + 4 * f4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
          auto finite_bits = [](float v) {
            const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
            return b < 0x7F800000u ? b : 0u;
          };
          // the largest magnitude of the tile, and of its smallest row that is not zero
          uint32_t low = 0xffffffffu;
          const unsigned row_lanes = kF4 == 32 ? 0xffffffffu : lane < 16 ? 0xffffu : 0xffff0000u;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            uint32_t of_row = max(max(finite_bits(x[i].x), finite_bits(x[i].y)), max(finite_bits(x[i].z), finite_bits(x[i].w)));
            of_row = __reduce_max_sync(row_lanes, of_row);
            mx = max(mx, of_row);
            if (of_row) low = min(low, of_row);
          }
          mx = __reduce_max_sync(0xffffffffu, mx);
          low = __reduce_min_sync(0xffffffffu, low);
          if (lane == 0) s_max[team * 4 + lw] = mx;
          if (lane == 0) s_low[team * 4 + lw] = low;
          const uint32_t st = entry % kStages;
          const bool free = wait(empty + st, ((entry / kStages) & 1) ^ 1);
          ok = ok && free;
          ptx::named_bar(bar_id, kLoaders);
          const uint4 m4 = *reinterpret_cast<const uint4*>(s_max + team * 4);
          const uint4 l4 = *reinterpret_cast<const uint4*>(s_low + team * 4);
          mx = max(max(m4.x, m4.y), max(m4.z, m4.w));
          low = min(min(l4.x, l4.y), min(l4.z, l4.w));
          const int up = mx ? scale_up(mx) : kNoScale;
          const bool spread = mx && (int)(mx >> 23) - (int)(low >> 23) > kMaxSpread;
          const float mul = mx ? pow2(up) : 1.0f;
          if (lt == 0) s_exp[ring8 * 2 + team] = up + (spread ? kSpreadMark : 0);
          uint8_t* dst = ring + st * Cfg::kStage;
          if (ok) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
              uint2 hi, lo;
              split4(x[i], mul, hi, lo);
              const int o = tile_at(pr + i * kHop, f4 >> 1, kHalfKV) + (f4 & 1) * 8;
              *reinterpret_cast<uint2*>(dst + o) = hi;
              *reinterpret_cast<uint2*>(dst + Cfg::kTile + o) = lo;
            }
          }
          ptx::fence_proxy_async();
          arrive(ok ? full + st : nullptr);
          entry += 2;
        }
      }
      tiles += it.tiles;
    }
    flush();
    // every copy has landed before the shared memory goes
    if (!kWide && lw == 0 && lane == 0)
      for (int st = 0; st < kStages; ++st)
        if ((copied >> st) & 1) umma::settle_bar(full + st, (odd >> st) & 1, kWaitNs);
  } else {
    // -------------------------------------------------------------------- softmax
    const int x = warp >> 2, r0 = (warp & 3) * 32, r = r0 + lane;
    const uint32_t ts = tmem + x * 128 + ((uint32_t)r0 << 16), to = tmem + 256 + x * D + ((uint32_t)r0 << 16);
    const float scale2 = a.scale * kLog2e;
    const int rtok = token_of(a, r);  // token of the thread's row within the block
    uint32_t seen = 0, o_turn = 0, tiles = 0;
    bool ok = true;  // the same for the whole warp
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    for (int w = 0; ok && w * ctas < items; ++w) {
      const int idx = item_of(w);
      if (idx >= items) continue;
      const ItemRange it = item_at<kPos>(a, map, tokens, splits, idx, lane);
      const int toks = min(block_toks, it.toks - x * block_toks);  // of this block, if positive
      const bool live = rtok < toks;
      const int p0 = it.len - it.n + it.tok0 + x * block_toks;  // position of the block's first token
      const int plast = live ? p0 + rtok : -1;
      const int pfirst = first_seen(a, plast);
      // every row of the block sees the positions from seen_from to p0
      const int seen_from = first_seen(a, p0 + toks - 1);
      const bool busy = toks > 0 && it.tiles > 0;
      const long long row0 = it.q0 + it.tok0 + x * block_toks;  // the block's first row
      if (splits > 1 && idx % splits == 0 && tid == 0)
        chunk_rec(work)[idx / splits] = make_int4((int)row0, it.parts > 1 ? it.toks : 0, it.head, splits << 16 | it.parts);
      float c = scale2;
      if constexpr (kHalves) {
        // the warp's rows of q, eight at a time: four lanes a row, every fourth float4 each.
        // The previous item's products have completed (o_full)
        if (busy) {
          constexpr int kF4 = D / 16;
          const int sub = lane & 3;
          int ups[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = r0 + 8 * i + (lane >> 2), tok = token_of(a, rr);
            const bool there = tok < toks;
            const float* src = reinterpret_cast<const float*>(a.q) + (there ? (row0 + tok) * a.q_stride + (it.head * a.group + rr - tok * a.group) * D : 0) + sub * 4;
            float4 y[kF4];
            uint32_t mx = 0;
#pragma unroll
            for (int k = 0; k < kF4; ++k) y[k] = *reinterpret_cast<const float4*>(src + 16 * k);
#pragma unroll
            for (int k = 0; k < kF4; ++k) {
              if (!there) y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              mx = max(max(mx, max(__float_as_uint(y[k].x) << 1, __float_as_uint(y[k].y) << 1)),
                       max(__float_as_uint(y[k].z) << 1, __float_as_uint(y[k].w) << 1));
            }
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) >> 1;
            ups[i] = mx == 0 || mx >= 0x7F800000u ? 0 : scale_up(mx);
            const float mul = pow2(ups[i]);
#pragma unroll
            for (int k = 0; k < kF4; ++k) {
              uint2 hi, lo;
              split4(y[k], mul, hi, lo);
              const int f4 = 4 * k + sub;  // float4 of the row: half a piece
              uint8_t* dst = sq + x * 2 * Cfg::kQTile + tile_at(rr, f4 >> 1, kHalfQ) + (f4 & 1) * 8;
              *reinterpret_cast<uint2*>(dst) = hi;
              *reinterpret_cast<uint2*>(dst + Cfg::kQTile) = lo;
            }
          }
          ptx::fence_proxy_async();
          ptx::mbar_arrive(q_full + x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int up = __shfl_sync(0xffffffffu, ups[i], (lane & 7) * 4);
            if ((lane >> 3) == i) c = scale2 * pow2(-up);
          }
        }
      }
      float m = -INFINITY, l = 0.0f;
      int e_ref = kNoScale, e_first = kNoScale;  // f32 cache: the numerators count in 2^-e_ref
      bool wild = false;
      // f32 rows: numerators of earlier tiles, relative to m_acc and e_acc, in the workspace
      float m_acc = -INFINITY;
      int e_acc = kNoScale;
      float4* const acc = kHalves ? chunk_acc<D>(work, cta) + x * 128 + r : nullptr;
      bool some = false;
      auto add_up = [&](bool last) {
        float f = m_acc == -INFINITY ? 0.0f : exp2_approx(m_acc - m);
        if (kWide && e_acc != kNoScale) f *= pow2(max(-126, e_ref - e_acc));
#pragma unroll 1
        for (int i = 0; i < D / 32; ++i) {
          float o[32];
          tmem_ld32(to + 32 * i, o);
          umma::tmem_wait_ld();
          if (some) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 y = __ldcg(acc + (8 * i + k) * 256);
              o[4 * k] = __fmaf_rn(y.x, f, o[4 * k]);
              o[4 * k + 1] = __fmaf_rn(y.y, f, o[4 * k + 1]);
              o[4 * k + 2] = __fmaf_rn(y.z, f, o[4 * k + 2]);
              o[4 * k + 3] = __fmaf_rn(y.w, f, o[4 * k + 3]);
            }
          }
          if (last) {
            tmem_st32(to + 32 * i, reinterpret_cast<const uint32_t*>(o));
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              __stcg(acc + (8 * i + k) * 256, make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
          }
        }
        if (last) tmem_wait_st();
        some = true;
        m_acc = m;
        e_acc = e_ref;
      };
      if (busy) {
        for (int j = 0; j < it.tiles; ++j) {
          ok = wait_all(s_full + x, seen & 1);
          ++seen;
          if (!ok) break;
          umma::tc_fence_after();
          if (kHalves && j > 0 && fresh(j)) add_up(false);
          const int ring8 = (tiles + j) & 7;
          const int pos0 = it.first + j * kPos;
          const uint4 b4 = *reinterpret_cast<const uint4*>(s_bad + ring8 * 4);
          float ct = c, lift = 0.0f, o_scale = 1.0f, l_scale = 1.0f;
          if constexpr (kWide) {
            const uint32_t ev = (tiles + j) * 2 + 1;  // V's scale: its tile stays until this block's weights are used
            ok = wait_all(full + ev % kStages, (ev / kStages) & 1);
            if (!ok) break;
            int ek = s_exp[ring8 * 2], eV = s_exp[ring8 * 2 + 1];
            wild |= ek > kSpreadMark / 2 || eV > kSpreadMark / 2;
            if (ek > kSpreadMark / 2) ek -= kSpreadMark;
            if (eV > kSpreadMark / 2) eV -= kSpreadMark;
            if (ek != kNoScale) ct = c * pow2(-ek);
            if (eV != kNoScale) {
              if (eV < e_ref) {
                if (e_ref != kNoScale) o_scale = pow2(max(-126, eV - e_ref));
                else e_first = eV;
                e_ref = eV;
              }
              wild |= eV - e_ref > kMaxLift || e_first - e_ref > kMaxDrop;
              lift = (float)(e_ref - eV);
              l_scale = pow2(min(126, eV - e_ref));
            }
          }
          const bool masked = pos0 < seen_from || pos0 + kPos - 1 > p0 || (b4.x | b4.y | b4.z | b4.w);
          // kCols scores at a time, from TMEM for the maximum and, unless they are all, again
          // for the weights
          float s[kCols];
          auto load_scores = [&](int b) {
#pragma unroll
            for (int i = 0; i < kCols / 32; ++i) tmem_ld32(ts + kCols * b + 32 * i, s + 32 * i);
            umma::tmem_wait_ld();
            if (masked) {
              const int hi = plast - pos0 - kCols * b, lo = pfirst - pos0 - kCols * b;
#pragma unroll
              for (int i = 0; i < kCols / 32; ++i) {
                const uint32_t bw = s_bad[ring8 * 4 + (kCols / 32) * b + i];
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (32 * i + k > hi || 32 * i + k < lo || ((bw >> k) & 1)) s[32 * i + k] = -INFINITY;
              }
            }
          };
          float top_x = -INFINITY;
#pragma unroll 1
          for (int b = 0; b < kPos / kCols; ++b) {
            load_scores(b);
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int k = 4; k + 7 < kCols; k += 8)
#pragma unroll
              for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], fmaxf(s[k + q], s[k + 4 + q]));
#pragma unroll
            for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], s[kCols - 4 + q]);
            top_x = fmaxf(top_x, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          }
          top_x *= ct;
          const bool raise = top_x > m + kSlack || (m == -INFINITY && top_x > m);
          if (__any_sync(0xffffffffu, raise) || (kWide && o_scale != 1.0f)) {
            const float mn = raise ? fmaxf(m, top_x) : m;
            const float f = mn == -INFINITY ? 1.0f : exp2_approx(m - mn);
            m = mn;
            l *= f;
            const float fo = f * o_scale;
            if (!fresh(j)) {
#pragma unroll 1
              for (int i = 0; i < D / 16; ++i) {
                float o[16];
                tmem_ld16(to + 16 * i, o);
                umma::tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] *= fo;
                tmem_st16(to + 16 * i, reinterpret_cast<const uint32_t*>(o));
              }
            }
          }
          const float sub = (m == -INFINITY ? 0.0f : m) - kShift - lift;
          const float2 c2 = make_float2(ct, ct), sub2 = make_float2(-sub, -sub);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll 1
          for (int b = 0; b < kPos / kCols; ++b) {
            if constexpr (kCols < kPos) load_scores(b);
#pragma unroll
            for (int g = 0; g < kCols / 32; ++g) {  // 32 scores become 16 columns of weights (and 16 of lower halves)
              uint32_t hi[16], lo[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 y = __ffma2_rn(make_float2(s[32 * g + 2 * i], s[32 * g + 2 * i + 1]), c2, sub2);
                const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                sum[i & 1] = __fadd2_rn(sum[i & 1], e);
                hi[i] = pack2(e.x, e.y, M());
                if constexpr (kHalves) {
                  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
                  lo[i] = pack2(e.x - h.x, e.y - h.y, __half());
                }
              }
              const int col = kCols * b + 32 * g;
              tmem_st16(ts + Cfg::kQParts * (col / 2), hi);
              if constexpr (kHalves) tmem_st16(ts + col + 16, lo);
            }
          }
          const float add = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          l = kWide ? __fmaf_rn(add, l_scale, l) : l + add;
          tmem_wait_st();
          umma::tc_fence_before();
          ptx::mbar_arrive(p_ready + x);
        }
        if (ok) {
          ok = wait_all(o_full + x, o_turn & 1);
          umma::tc_fence_after();
          if (kHalves && ok && some) add_up(true);
          ++o_turn;
        }
      }
      if (!ok) break;
      tiles += it.tiles;
      if (toks <= 0) continue;
      // ---- the rows' results: 16 rows at a time, so that four threads write 32 bytes of a row
      const float back = kWide && e_ref != kNoScale ? pow2(-e_ref) : 1.0f;
      const float mul = it.part >= 0 ? 1.0f : l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
      const unsigned live_rows = __ballot_sync(0xffffffffu, live);
      unsigned redo = __ballot_sync(0xffffffffu, live && (wild || !(l * 0.0f == 0.0f)));
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const int ra = 16 * h + (lane >> 2), t = lane & 3;  // this thread's rows: ra and ra + 8 of the warp's
        const float mula = __shfl_sync(0xffffffffu, mul, ra), mulb = __shfl_sync(0xffffffffu, mul, ra + 8);
        const bool la = (live_rows >> ra) & 1, lb = (live_rows >> (ra + 8)) & 1;
        auto out_row = [&](int rr) {  // output of packed row rr of the block
          const int tok = token_of(a, rr);
          return static_cast<T*>(a.out) + (row0 + tok) * a.out_stride + (it.head * a.group + rr - tok * a.group) * D;
        };
        T* const oa = out_row(r0 + ra);
        T* const ob = out_row(r0 + ra + 8);
        float* const na = it.part < 0 ? nullptr : chunk_num(work) + ((size_t)it.part * 256 + x * 128 + r0 + ra) * D;
        float za = 0.0f, zb = 0.0f;  // 0, or NaN where a numerator is not finite
#pragma unroll 1
        for (int cb = 0; cb < D / 32; ++cb) {
          float v[16];
          if (busy) {
            tmem_ld_frag(to + ((uint32_t)(16 * h) << 16) + 32 * cb, v);
            umma::tmem_wait_ld();
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = 0.0f;
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            za = __fmaf_rn(v[4 * n], 0.0f, __fmaf_rn(v[4 * n + 1], 0.0f, za));
            zb = __fmaf_rn(v[4 * n + 2], 0.0f, __fmaf_rn(v[4 * n + 3], 0.0f, zb));
            v[4 * n] *= mula;
            v[4 * n + 1] *= mula;
            v[4 * n + 2] *= mulb;
            v[4 * n + 3] *= mulb;
            if constexpr (kWide) {  // apart from the quotient: their product may leave the normal range
#pragma unroll
              for (int k = 0; k < 4; ++k) v[4 * n + k] *= back;
            }
          }
          if (it.part >= 0 || kHalves) {
            float* const pa = it.part >= 0 ? na : reinterpret_cast<float*>(oa);
            float* const pb = it.part >= 0 ? na + 8 * D : reinterpret_cast<float*>(ob);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int d = 32 * cb + 8 * n + 2 * t;
              if (la) *reinterpret_cast<float2*>(pa + d) = make_float2(v[4 * n], v[4 * n + 1]);
              if (lb) *reinterpret_cast<float2*>(pb + d) = make_float2(v[4 * n + 2], v[4 * n + 3]);
            }
          } else {
            // neighbours trade, so that a thread has four consecutive elements of one n8 group
#pragma unroll
            for (int n = 0; n < 4; n += 2) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint32_t w0 = pack2(v[4 * n + 2 * q], v[4 * n + 2 * q + 1], M());
                const uint32_t w1 = pack2(v[4 * n + 4 + 2 * q], v[4 * n + 5 + 2 * q], M());
                const uint32_t got = __shfl_xor_sync(0xffffffffu, t & 1 ? w0 : w1, 1);
                const int d = 32 * cb + 8 * (n + (t & 1)) + 4 * (t >> 1);
                if (q ? lb : la) *reinterpret_cast<uint2*>((q ? ob : oa) + d) = t & 1 ? make_uint2(got, w1) : make_uint2(w0, got);
              }
            }
          }
        }
        const unsigned fa = __ballot_sync(0xffffffffu, za != 0.0f), fb = __ballot_sync(0xffffffffu, zb != 0.0f);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if ((fa >> (4 * q)) & 15u) redo |= 1u << (16 * h + q);
          if ((fb >> (4 * q)) & 15u) redo |= 1u << (16 * h + 8 + q);
        }
      }
      if ((redo & live_rows) && lane == 0) atomicOr(s_redo + w % kRedoTurns / 4, 1u << (w % 4 * 8 + warp));
      if (live) {
        if (it.part >= 0)
          chunk_ml(work)[(size_t)it.part * 256 + x * 128 + r] = make_float2(m, l);
        else if (a.lse)
          a.lse[(row0 + rtok) * a.hq + it.head * a.group + r - rtok * a.group] = l == 0.0f ? -INFINITY : (m - kShift + log2f(l)) * kLn2;
      }
    }
  }
  // ---- end: every role has left its loop
  umma::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    umma::tc_fence_after();
    umma::tmem_relinquish();
    umma::tmem_dealloc(tmem, 512);
  }
  if (*abort_flag) {
    if (tid == 0 && a.status) *a.status = 6u;
    // a part that was not finished makes its rows NaN, whatever the workspace held (split items
    // have one turn: the part is the CTA's number)
    if (splits > 1 && cta < items)
      for (int i = tid; i < 256; i += Cfg::kThreads) chunk_ml(work)[(size_t)cta * 256 + i] = make_float2(NAN, NAN);
    return;
  }
  // ---- rows to compute again: all of a softmax warp's 32, four at a time, by any warp
  for (int w = 0; w * ctas < items; ++w) {
    const uint32_t flags = (s_redo[w % kRedoTurns / 4] >> (w % 4 * 8)) & 0xffu;
    const int idx = item_of(w);
    if (!flags || idx >= items) continue;
    const ItemRange it = item_at<kPos>(a, map, tokens, splits, idx, lane);
    const int* table = a.batch.table + (long long)it.seq * a.batch.table_stride;
    const int end = it.first + (it.tiles * kPos - 1);  // the part's last position
    int turn = 0;
#pragma unroll 1
    for (int u = 0; u < 64; ++u) {
      if (!((flags >> (u >> 3)) & 1) || turn++ % (Cfg::kThreads / 32) != warp) continue;
      const int x = u >> 5, first_row = (u & 31) * 4;  // of block x
      const int toks = min(block_toks, it.toks - x * block_toks);
      const int p0 = it.len - it.n + it.tok0 + x * block_toks;
      const long long row0 = it.q0 + it.tok0 + x * block_toks;
      int from[4], to[4], lo = end, hi = -1;
      long long at[4];  // (row, query head) of the output, or -1
      const T* q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = token_of(a, first_row + i);
        const bool live = tok < toks;
        const long long row = row0 + (live ? tok : 0);
        const int h = it.head * a.group + (live ? first_row + i - tok * a.group : 0);
        q[i] = static_cast<const T*>(a.q) + row * a.q_stride + h * D;
        at[i] = live ? row * a.hq + h : -1;
        from[i] = max(first_seen(a, p0 + tok), it.first);
        to[i] = live ? min(p0 + tok, end) : -1;
        if (to[i] >= from[i]) lo = min(lo, from[i]), hi = max(hi, to[i]);
      }
      if (toks <= 0) continue;
      float o[4][D / 32], m, l;
      rows_attend<T, C, D>(a, q, from, to, lo, hi, table, it.head, a.scale * kLog2e, o, m, l);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mi = __shfl_sync(0xffffffffu, m, 8 * i), li = __shfl_sync(0xffffffffu, l, 8 * i);
        if (at[i] < 0) continue;
        const int h = it.head * a.group + first_row + i - token_of(a, first_row + i) * a.group;
        const long long row = row0 + token_of(a, first_row + i);
        const size_t part_row = (size_t)max(it.part, 0) * 256 + x * 128 + first_row + i;
        const float inv = li == 0.0f ? 0.0f : __fdiv_rn(1.0f, li);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const int d = lane * (D / 32) + e;
          if (it.part < 0)
            static_cast<T*>(a.out)[row * a.out_stride + h * D + d] = from_f32(__fmul_rn(o[i][e], inv), T());
          else
            chunk_num(work)[part_row * D + d] = o[i][e];
        }
        if (lane == 0) {
          if (it.part >= 0)
            chunk_ml(work)[part_row] = make_float2(mi, li);
          else if (a.lse)
            a.lse[at[i]] = li == 0.0f ? -INFINITY : (mi - kShift + log2f(li)) * kLn2;
        }
      }
    }
  }
}

// Split items: a warp adds the parts of a row in order; block (tile and head, group of 8 rows).
template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const AttnArgs a, void* work) {
  constexpr int E = D / 32, kAhead = 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 rec = chunk_rec(work)[blockIdx.x];  // (first row, tokens, kv head, slots and parts)
  const int splits = rec.w & 0xffff;
  const int lane = threadIdx.x & 31, rr = blockIdx.y * 8 + (threadIdx.x >> 5), x = rr >> 7, r = rr & 127;
  const int block_toks = 128 / a.group, rtok = token_of(a, r), tok = x * block_toks + rtok;
  if (rtok >= block_toks || tok >= rec.y) return;
  const size_t first = (size_t)blockIdx.x * (rec.w >> 16) * 256 + rr;
  float mm = -INFINITY;
  for (int s = lane; s < splits; s += 32) mm = fmaxf(mm, chunk_ml(work)[first + (size_t)s * 256].x);
  mm = warp_max(mm);
  const float mu = mm == -INFINITY ? 0.0f : mm;
  float v[E], l = 0.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] = 0.0f;
#pragma unroll 1
  for (int s0 = 0; s0 < splits; s0 += kAhead) {
    float2 ml[kAhead];
    float y[kAhead][E];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const size_t at = first + (size_t)min(s0 + k, splits - 1) * 256;
      ml[k] = s0 + k < splits ? chunk_ml(work)[at] : make_float2(-INFINITY, 0.0f);
      const float* p = chunk_num(work) + at * D + lane * E;
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const float2 z = *reinterpret_cast<const float2*>(p + j);
        y[k][j] = z.x;
        y[k][j + 1] = z.y;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (s0 + k >= splits) break;
      const float f = exp2_approx(ml[k].x - mu);
      l = __fmaf_rn(ml[k].y, f, l);
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = __fmaf_rn(y[k][j], f, v[j]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
  const long long row = rec.x + tok;
  const int h = rec.z * a.group + r - rtok * a.group;
  T* out = static_cast<T*>(a.out) + row * a.out_stride + h * D + lane * E;
#pragma unroll
  for (int j = 0; j < E; ++j) out[j] = from_f32(v[j] * inv, T());
  if (a.lse && lane == 0) a.lse[row * a.hq + h] = l == 0.0f ? -INFINITY : (mm - kShift + log2f(l)) * kLn2;
}

}  // namespace paged
}  // namespace qora
