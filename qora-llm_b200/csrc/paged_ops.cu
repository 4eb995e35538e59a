// paged_ops.cu — the kernel-level entry points for many requests over one paged cache:
// qora_qk_norm_rope, qora_paged_append, qora_paged_attention (include/qora_cuda.h). All
// checks that need no device data happen here; what lies in device memory (row ranges,
// lengths, page ids) is checked by the kernels, which skip what is out of range and set
// the caller's status word.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "host_util.h"
#include "paged_attention.cuh"
#include "paged_chunk.cuh"
#include "paged_rows.cuh"
#include "paged_token.cuh"

using namespace qora;

namespace {

typedef unsigned long long ull;

size_t elem_size(uint32_t dt) { return dt == QORA_DT_F32 ? 4 : 2; }

qora_status check_types(uint32_t dtype, uint32_t kv_dtype) {
  if (dtype > QORA_DT_BF16 || kv_dtype > QORA_DT_BF16)
    return fail(QORA_ERR_INVALID, "element types %u and %u", dtype, kv_dtype);
  if (dtype != kv_dtype && !(dtype == QORA_DT_F32 && kv_dtype == QORA_DT_F16))
    return fail(QORA_ERR_UNSUPPORTED, "rows of type %u with a cache of type %u (equal types, or f32 rows with an f16 cache)",
                dtype, kv_dtype);
  return QORA_OK;
}

qora_status check_heads(uint32_t rows, uint32_t hq, uint32_t hk, uint32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return fail(QORA_ERR_UNSUPPORTED, "head_dim %u: 64 or 128", head_dim);
  if (hq > 1024 || hk > 1024) return fail(QORA_ERR_INVALID, "%u query heads, %u kv heads", hq, hk);
  if (rows > (1u << 24)) return fail(QORA_ERR_INVALID, "%u rows in one call (at most 2^24)", rows);
  return QORA_OK;
}

qora_status check_rows(const char* what, const void* p, uint32_t rows, uint64_t stride, uint32_t heads, uint32_t head_dim, size_t esz) {
  if (!p && rows) return fail(QORA_ERR_INVALID, "%s is NULL", what);
  if (((uintptr_t)p | (stride * esz)) % 16)
    return fail(QORA_ERR_INVALID, "%s: rows must start on 16-byte boundaries (stride %llu)", what, (ull)stride);
  if (stride < (uint64_t)heads * head_dim || stride >= (1ull << 38))
    return fail(QORA_ERR_INVALID, "%s: row stride %llu for %u heads of %u", what, (ull)stride, heads, head_dim);
  return QORA_OK;
}

// Rows of `width` elements, `stride` apart: what an entry point reads or writes.
struct Rows {
  const void* p;
  uint64_t stride, width;
};
// Whether two sets of rows share a byte; those with unequal strides whose ranges meet count
// as sharing one.
bool meet(const Rows& a, const Rows& b, uint32_t rows, size_t esz) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  if (rows == 0 || x + ((rows - 1) * a.stride + a.width) * esz <= y || y + ((rows - 1) * b.stride + b.width) * esz <= x) return false;
  if (a.stride != b.stride) return true;
  const uint64_t step = a.stride * esz, off = x <= y ? (y - x) % step : (step - (x - y) % step) % step;  // b's row behind a's
  return off < a.width * esz || off + b.width * esz > step;
}
qora_status check_apart(const char* what, const Rows& a, const Rows& b, uint32_t rows, size_t esz) {
  if (meet(a, b, rows, esz)) return fail(QORA_ERR_INVALID, "%s overlap", what);
  return QORA_OK;
}

qora_status check_same(const char* what, const Rows& in, const Rows& out, uint32_t rows, size_t esz) {
  if (in.p == out.p && in.stride != out.stride)
    return fail(QORA_ERR_INVALID, "%s in place needs equal strides (%llu, %llu)", what, (ull)in.stride, (ull)out.stride);
  if (in.p != out.p && meet(in, out, rows, esz)) return fail(QORA_ERR_INVALID, "%s and its output overlap", what);
  return QORA_OK;
}

// Arrays of 32-bit words on the device
qora_status check_words(const char* what, const void* p) {
  if ((uintptr_t)p % 4) return fail(QORA_ERR_INVALID, "%s must be 4-byte aligned", what);
  return QORA_OK;
}

qora_status check_turn(const float* q_gamma, const float* k_gamma, float eps, const float* cos_t, const float* sin_t,
                       uint32_t rope_rows, uint32_t r, uint32_t head_dim) {
  if (((uintptr_t)q_gamma | (uintptr_t)k_gamma | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16)
    return fail(QORA_ERR_INVALID, "gains and rotation tables must be 16-byte aligned");
  if ((q_gamma || k_gamma) && !(eps >= 0.0f && std::isfinite(eps))) return fail(QORA_ERR_INVALID, "eps %g", (double)eps);
  if (!cos_t != !sin_t) return fail(QORA_ERR_INVALID, "cos and sin tables go together");
  if (cos_t) {
    if (r == 0 || 2 * (uint64_t)r > head_dim) return fail(QORA_ERR_INVALID, "rope_half_dim %u for head_dim %u", r, head_dim);
    if (r % 8) return fail(QORA_ERR_UNSUPPORTED, "rope_half_dim %u: a multiple of 8", r);
    if (rope_rows == 0 || rope_rows > 0x7fffffffu) return fail(QORA_ERR_INVALID, "rope_rows %u", rope_rows);
  }
  return QORA_OK;
}

qora_status check_pages(const void* k, const void* v, uint32_t hk, uint32_t head_dim, size_t esz, uint32_t num_pages,
                        uint32_t page_size, uint64_t page_stride, uint64_t head_stride, uint64_t slot_stride) {
  if (!k || !v) return fail(QORA_ERR_INVALID, "NULL pages");
  if (num_pages == 0 || num_pages > 0x7fffffffu || page_size == 0 || page_size > (1u << 20))
    return fail(QORA_ERR_INVALID, "%u pages of %u positions", num_pages, page_size);
  if (((uintptr_t)k | (uintptr_t)v | (page_stride * esz) | (head_stride * esz) | (slot_stride * esz)) % 16)
    return fail(QORA_ERR_INVALID, "pages and their strides must be multiples of 16 bytes");
  const uint64_t top = 1ull << 40;
  if (page_stride > top || head_stride > top || slot_stride > top) return fail(QORA_ERR_INVALID, "page strides beyond 2^40");
  const bool by_slot = slot_stride >= (uint64_t)(hk - 1) * head_stride + head_dim && (hk == 1 || head_stride >= head_dim);
  const bool by_head = head_stride >= (uint64_t)(page_size - 1) * slot_stride + head_dim && (page_size == 1 || slot_stride >= head_dim);
  if ((!by_slot && !by_head) ||
      (num_pages > 1 && page_stride < (uint64_t)(page_size - 1) * slot_stride + (uint64_t)(hk - 1) * head_stride + head_dim))
    return fail(QORA_ERR_INVALID, "page strides %llu, %llu, %llu overlap (page, head, slot)", (ull)page_stride,
                (ull)head_stride, (ull)slot_stride);
  return QORA_OK;
}

qora_status check_batch(const int32_t* q_start, const int32_t* kv_len, const int32_t* table, uint32_t table_stride,
                        uint32_t page_size, uint32_t seqs) {
  if (seqs && (!q_start || !kv_len || !table)) return fail(QORA_ERR_INVALID, "NULL batch arrays");
  QCHECK(check_words("batch arrays", (const void*)((uintptr_t)q_start | (uintptr_t)kv_len | (uintptr_t)table)));
  if (seqs > (1u << 20)) return fail(QORA_ERR_INVALID, "%u sequences", seqs);
  if (table_stride == 0 || (uint64_t)table_stride * page_size > 0x7fffffffull)
    return fail(QORA_ERR_INVALID, "table rows of %u pages of %u positions", table_stride, page_size);
  return QORA_OK;
}

// Groups of head rows that a warp walks over: all of a token's, fewer while there are not
// warps enough to fill the GPU (32 on every SM).
template <typename T, typename C, int D, bool kAppend>
qora_status launch_rows(paged::RowArgs a, cudaStream_t s) {
  constexpr int kHeads = 32 / (D / 2 / paged::Elem<T>::kVec);
  const int groups = (a.hq + a.hk + a.hv + kHeads - 1) / kHeads;
  int dev = 0;
  QCUDA(cudaGetDevice(&dev));
  const long long fill = 32LL * sm_count(dev);
  const int parts = (int)std::min<long long>(groups, (fill + a.rows - 1) / a.rows);
  a.per_warp = (groups + parts - 1) / parts;
  const long long units = (long long)a.rows * ((groups + a.per_warp - 1) / a.per_warp);
  if (units > 0x7fffffff) return fail(QORA_ERR_INVALID, "%d rows of %d head rows", a.rows, a.hq + a.hk + a.hv);
  paged::rows_kernel<T, C, D, kAppend><<<(unsigned)((units + paged::kRowWarps - 1) / paged::kRowWarps), 32 * paged::kRowWarps, 0, s>>>(a);
  QCUDA(cudaGetLastError());
  return QORA_OK;
}

template <typename T, typename C, bool kAppend>
qora_status launch_rows_d(uint32_t head_dim, const paged::RowArgs& a, cudaStream_t s) {
  return head_dim == 64 ? launch_rows<T, C, 64, kAppend>(a, s) : launch_rows<T, C, 128, kAppend>(a, s);
}

// A kernel's dynamic shared memory limit, set once per device and kernel.
template <auto* kKernel>
qora_status allow_smem(int dev, int bytes) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return QORA_OK;
  QCUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_release);
  return QORA_OK;
}

// Fewest units of work worth a CTA of their own, and what a tile's fixed time counts, in
// steps: 128 ragged tokens take 181 us at 16, 174 us at 32 and 176 us at 48.
constexpr int kTokenMinSteps = 16;
constexpr int kTokenTileCost = 32;

template <typename T, typename C, int D>
qora_status launch_token(const paged::AttnArgs& a, void* work, cudaStream_t s) {
  using Cfg = paged::TokenCfg<T, C, D>;
  int dev = 0;
  QCUDA(cudaGetDevice(&dev));
  QCHECK((allow_smem<&paged::token_kernel<T, C, D>>(dev, Cfg::kSmem)));
  QCHECK((allow_smem<&paged::token_join_kernel<T, D>>(dev, 0)));
  const int ctas = std::min(sm_count(dev), paged::kTokenMaxCtas);
  paged::token_kernel<T, C, D><<<ctas, 32 * Cfg::kWarps, Cfg::kSmem, s>>>(a, work, kTokenMinSteps, kTokenTileCost);
  QCUDA(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, std::min(a.max_q, a.few) * a.group);
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  QCUDA(cudaLaunchKernelEx(&cfg, paged::token_join_kernel<T, D>, a, work, ctas));
  return QORA_OK;
}

// Tensor map of 16-bit elements, 64 innermost elements per box, 128-byte swizzle. False
// where the map cannot describe them.
template <typename C>
bool encode_rows(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                 const cuuint32_t* box) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  for (int i = 0; i + 1 < rank; ++i)
    if (strides[i] >= (1ull << 40)) return false;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type =
      std::is_same<C, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(m, type, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// One layer's pages as [page][head][slot][D], boxes of box_rows slots.
template <typename C>
bool encode_pages(CUtensorMap* m, const void* base, const paged::AttnArgs& a, int D, int box_rows) {
  const cuuint64_t row = (cuuint64_t)D * sizeof(C);
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.pg.page_size, (cuuint64_t)a.hk, (cuuint64_t)a.pg.num_pages};
  // the stride of a dimension of one is free: any valid number does
  const cuuint64_t strides[3] = {(cuuint64_t)a.pg.slot_stride * sizeof(C), a.hk > 1 ? (cuuint64_t)a.pg.head_stride * sizeof(C) : row,
                                 a.pg.num_pages > 1 ? (cuuint64_t)a.pg.page_stride * sizeof(C) : row};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  return encode_rows<C>(m, base, 4, dims, strides, box);
}

template <typename T, typename C, int D>
qora_status launch_chunk(const paged::AttnArgs& a, void* work, cudaStream_t s) {
  using Cfg = paged::ChunkCfg<T, C, D>;
  int dev = 0;
  QCUDA(cudaGetDevice(&dev));
  QCHECK((allow_smem<&paged::chunk_kernel<T, C, D>>(dev, Cfg::kSmem)));
  const int sms = std::min(sm_count(dev), paged::kChunkMaxCtas);
  const int block_toks = Cfg::kBlock / a.group, tokens = 2 * block_toks;
  // Row tiles that sequences with disjoint rows can have, and that they are likely to have
  // (a half one behind each sequence). Where these leave half of the SMs idle, the kernel
  // splits the items by the number that there are (7 prompts of 45 to 181 rows over up to
  // 2,684 f32 positions: 74.5 us, split by the number that there can be 116 us).
  const long long most = ((long long)a.batch.rows + (long long)a.batch.seqs * (tokens - 1)) / tokens * a.hk;
  const int long_ones = a.few ? (a.batch.rows + a.max_q - 1) / a.max_q : a.batch.seqs;
  const long long likely = ((long long)a.batch.rows + (long long)long_ones * (tokens / 2)) / tokens * a.hk;
  if (most > 0x7fffffff) return fail(QORA_ERR_INVALID, "%d rows of %d sequences", a.batch.rows, a.batch.seqs);
  const bool split = 2 * likely <= sms;
  const int ctas = split ? sms : (int)std::min<long long>(sms, most);
  CUtensorMap qmap{}, kmap{}, vmap{};
  int box_rows = 0;
  if constexpr (!Cfg::kWide) {
    // boxes of a page, or of kPos rows of one: whole swizzle groups of 8 rows
    const int ps = a.pg.page_size;
    box_rows = ps % Cfg::kPos == 0 ? Cfg::kPos : Cfg::kPos % ps == 0 && ps >= 8 ? ps : 0;
    if (box_rows && !(encode_pages<C>(&kmap, a.k_pages, a, D, box_rows) && encode_pages<C>(&vmap, a.v_pages, a, D, box_rows)))
      box_rows = 0;
  }
  if constexpr (!Cfg::kHalves) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.hq, (cuuint64_t)a.batch.rows};
    const cuuint64_t strides[2] = {(cuuint64_t)D * sizeof(T), (cuuint64_t)a.q_stride * sizeof(T)};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)block_toks};
    if (!encode_rows<T>(&qmap, a.q, 3, dims, strides, box)) return fail(QORA_ERR_CUDA, "cuTensorMapEncodeTiled failed on q");
  }
  paged::chunk_kernel<T, C, D><<<ctas, Cfg::kThreads, Cfg::kSmem, s>>>(a, work, split, (int)most, box_rows, qmap, kmap, vmap);
  QCUDA(cudaGetLastError());
  if (!split) return QORA_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<long long>(most, paged::kChunkMaxSplit), a.max_q > block_toks ? 32 : 16);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  QCUDA(cudaLaunchKernelEx(&cfg, paged::chunk_join_kernel<T, D>, a, work));
  return QORA_OK;
}

// Sequences with at most `few` new rows are the token kernel's, which reads their pages nearly
// as fast as memory gives them (64 sequences over 4,000 positions, 4 query heads per kv head:
// 1 to 4 f16 rows 96 us, 1 to 2 f32 rows over f32 caches 181 us); longer ones the chunk
// kernel's (1 to 8 f16 rows 147 us, 1 to 5 rows 167 us; 1 to 4 f32 rows over f32 caches 533 us).
// Both run where short sequences are likely (the longest is far longer than the mean, or the
// others are short on average; the host does not know) and are more than the chunk kernel
// would have in one turn of its CTAs, half of that with an f32 cache: 60 tokens over 4,000
// positions with 4 chunks of 512 rows over 2,000 take 154 us (f16), 202 us (f32 over f16) and
// 380 us (f32) with both, 202, 321 and 724 us with the chunk kernel alone. 31 tokens over 2,000
// with a chunk of 256 rows would take 63, 67 and 93 us with both; alone 48, 66 and 148 us: that
// batch gets both for f32 caches only. A token kernel without work costs 4 to 10 us.
template <typename T, typename C, int D>
qora_status launch_attn(paged::AttnArgs a, void* work, cudaStream_t s) {
  a.few = paged::TokenCfg<T, C, D>::kRows / a.group;
  if (a.max_q <= a.few) return launch_token<T, C, D>(a, work, s);
  const long long rows = a.batch.rows, others = a.batch.seqs - 1;
  int dev = 0;
  QCUDA(cudaGetDevice(&dev));
  const bool many = (others + 1) * a.hk * (sizeof(C) == 4 ? 2 : 1) > sm_count(dev);
  const bool uneven = 2 * rows <= (others + 1) * a.max_q || rows - a.max_q <= others * a.few;
  if (!many || !uneven) a.few = 0;
  if (a.few) QCHECK((launch_token<T, C, D>(a, work, s)));
  return launch_chunk<T, C, D>(a, work, s);
}

template <typename T, typename C>
qora_status launch_attn_d(uint32_t head_dim, const paged::AttnArgs& a, void* work, cudaStream_t s) {
  return head_dim == 64 ? launch_attn<T, C, 64>(a, work, s) : launch_attn<T, C, 128>(a, work, s);
}

}  // namespace

extern "C" {

qora_status qora_qk_norm_rope(const void* d_q, uint64_t q_stride, const void* d_k, uint64_t k_stride, uint32_t dtype,
                              uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
                              const float* d_q_gamma, const float* d_k_gamma, float eps, const int32_t* d_pos,
                              const float* d_cos, const float* d_sin, uint32_t rope_rows, uint32_t rope_half_dim,
                              void* d_q_out, uint64_t q_out_stride, void* d_k_out, uint64_t k_out_stride,
                              uint32_t* d_status, void* stream) {
  QCHECK(check_types(dtype, dtype));
  QCHECK(check_heads(rows, q_heads, kv_heads, head_dim));
  if (q_heads + kv_heads == 0) return fail(QORA_ERR_INVALID, "no heads");
  const size_t esz = elem_size(dtype);
  if (q_heads) {
    QCHECK(check_rows("q", d_q, rows, q_stride, q_heads, head_dim, esz));
    QCHECK(check_rows("q_out", d_q_out, rows, q_out_stride, q_heads, head_dim, esz));
  }
  if (kv_heads) {
    QCHECK(check_rows("k", d_k, rows, k_stride, kv_heads, head_dim, esz));
    QCHECK(check_rows("k_out", d_k_out, rows, k_out_stride, kv_heads, head_dim, esz));
  }
  QCHECK(check_words("positions and status", (const void*)((uintptr_t)d_pos | (uintptr_t)d_status)));
  QCHECK(check_turn(d_q_gamma, d_k_gamma, eps, d_cos, d_sin, rope_rows, rope_half_dim, head_dim));
  if (d_cos && !d_pos && rows) return fail(QORA_ERR_INVALID, "a rotation needs positions");
  if (rows == 0) return QORA_OK;
  const Rows q{d_q, q_stride, (uint64_t)q_heads * head_dim}, qo{d_q_out, q_out_stride, q.width};
  const Rows k{d_k, k_stride, (uint64_t)kv_heads * head_dim}, ko{d_k_out, k_out_stride, k.width};
  if (q_heads) QCHECK(check_same("q", q, qo, rows, esz));
  if (kv_heads) QCHECK(check_same("k", k, ko, rows, esz));
  if (q_heads && kv_heads) {
    QCHECK(check_apart("q_out and k", qo, k, rows, esz));
    QCHECK(check_apart("k_out and q", ko, q, rows, esz));
    QCHECK(check_apart("q_out and k_out", qo, ko, rows, esz));
  }
  paged::RowArgs a{};
  a.q = d_q, a.k = d_k, a.q_stride = (long long)q_stride, a.k_stride = (long long)k_stride;
  a.rows = (int)rows, a.hq = (int)q_heads, a.hk = (int)kv_heads, a.hv = 0;
  a.q_gamma = d_q_gamma, a.k_gamma = d_k_gamma, a.eps = eps;
  a.pos = d_pos, a.cos_t = d_cos, a.sin_t = d_sin, a.rope_rows = (int)rope_rows;
  a.r = d_cos ? (int)rope_half_dim : (int)head_dim / 2;
  a.q_out = d_q_out, a.k_out = d_k_out, a.qo_stride = (long long)q_out_stride, a.ko_stride = (long long)k_out_stride;
  a.status = d_status;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == QORA_DT_F32) return launch_rows_d<float, float, false>(head_dim, a, s);
  if (dtype == QORA_DT_F16) return launch_rows_d<__half, __half, false>(head_dim, a, s);
  return launch_rows_d<__nv_bfloat16, __nv_bfloat16, false>(head_dim, a, s);
}

qora_status qora_paged_append(const void* d_q, uint64_t q_stride, const void* d_k, uint64_t k_stride, const void* d_v,
                              uint64_t v_stride, uint32_t dtype, uint32_t rows, uint32_t q_heads, uint32_t kv_heads,
                              uint32_t head_dim, const float* d_q_gamma, const float* d_k_gamma, float eps,
                              const float* d_cos, const float* d_sin, uint32_t rope_rows, uint32_t rope_half_dim,
                              void* d_q_out, uint64_t q_out_stride, void* d_k_pages, void* d_v_pages, uint32_t kv_dtype,
                              uint32_t num_pages, uint32_t page_size, uint64_t page_stride, uint64_t head_stride,
                              uint64_t slot_stride, const int32_t* d_q_start, const int32_t* d_kv_len,
                              const int32_t* d_table, uint32_t table_stride, uint32_t seqs, uint32_t* d_status,
                              void* stream) {
  QCHECK(check_types(dtype, kv_dtype));
  QCHECK(check_heads(rows, q_heads, kv_heads, head_dim));
  if (kv_heads == 0) return fail(QORA_ERR_INVALID, "no kv heads");
  const size_t esz = elem_size(dtype);
  if (q_heads) {
    QCHECK(check_rows("q", d_q, rows, q_stride, q_heads, head_dim, esz));
    QCHECK(check_rows("q_out", d_q_out, rows, q_out_stride, q_heads, head_dim, esz));
  }
  QCHECK(check_rows("k", d_k, rows, k_stride, kv_heads, head_dim, esz));
  QCHECK(check_rows("v", d_v, rows, v_stride, kv_heads, head_dim, esz));
  QCHECK(check_words("status", d_status));
  QCHECK(check_turn(d_q_gamma, d_k_gamma, eps, d_cos, d_sin, rope_rows, rope_half_dim, head_dim));
  QCHECK(check_pages(d_k_pages, d_v_pages, kv_heads, head_dim, elem_size(kv_dtype), num_pages, page_size, page_stride,
                     head_stride, slot_stride));
  QCHECK(check_batch(d_q_start, d_kv_len, d_table, table_stride, page_size, seqs));
  if (rows == 0 || seqs == 0) return QORA_OK;
  if (q_heads) {
    const Rows q{d_q, q_stride, (uint64_t)q_heads * head_dim}, qo{d_q_out, q_out_stride, q.width};
    QCHECK(check_same("q", q, qo, rows, esz));
    QCHECK(check_apart("q_out and k", qo, {d_k, k_stride, (uint64_t)kv_heads * head_dim}, rows, esz));
    QCHECK(check_apart("q_out and v", qo, {d_v, v_stride, (uint64_t)kv_heads * head_dim}, rows, esz));
  }
  paged::RowArgs a{};
  a.q = d_q, a.k = d_k, a.v = d_v;
  a.q_stride = (long long)q_stride, a.k_stride = (long long)k_stride, a.v_stride = (long long)v_stride;
  a.rows = (int)rows, a.hq = (int)q_heads, a.hk = a.hv = (int)kv_heads;
  a.q_gamma = q_heads ? d_q_gamma : nullptr, a.k_gamma = d_k_gamma, a.eps = eps;
  a.cos_t = d_cos, a.sin_t = d_sin, a.rope_rows = (int)rope_rows;
  a.r = d_cos ? (int)rope_half_dim : (int)head_dim / 2;
  a.q_out = d_q_out, a.qo_stride = (long long)q_out_stride;
  a.k_pages = d_k_pages, a.v_pages = d_v_pages;
  a.pg = {(int)num_pages, (int)page_size, (long long)page_stride, (long long)head_stride, (long long)slot_stride};
  a.batch = {d_q_start, d_kv_len, d_table, (int)table_stride, (int)seqs, (int)rows};
  a.status = d_status;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == QORA_DT_F32 && kv_dtype == QORA_DT_F32) return launch_rows_d<float, float, true>(head_dim, a, s);
  if (dtype == QORA_DT_F32) return launch_rows_d<float, __half, true>(head_dim, a, s);
  if (dtype == QORA_DT_F16) return launch_rows_d<__half, __half, true>(head_dim, a, s);
  return launch_rows_d<__nv_bfloat16, __nv_bfloat16, true>(head_dim, a, s);
}

qora_status qora_paged_attention(const void* d_q, uint64_t q_stride, uint32_t dtype, uint32_t rows, uint32_t q_heads,
                                 uint32_t kv_heads, uint32_t head_dim, float scale, uint32_t window,
                                 const void* d_k_pages, const void* d_v_pages, uint32_t kv_dtype, uint32_t num_pages,
                                 uint32_t page_size, uint64_t page_stride, uint64_t head_stride, uint64_t slot_stride,
                                 const int32_t* d_q_start, const int32_t* d_kv_len, const int32_t* d_table,
                                 uint32_t table_stride, uint32_t seqs, uint32_t max_q, void* d_out, uint64_t out_stride,
                                 float* d_lse, void* d_work, uint64_t work_bytes, uint32_t* d_status, void* stream) {
  QCHECK(check_types(dtype, kv_dtype));
  QCHECK(check_heads(rows, q_heads, kv_heads, head_dim));
  if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads || q_heads / kv_heads > 128)
    return fail(QORA_ERR_INVALID, "%u query heads over %u kv heads", q_heads, kv_heads);
  const size_t esz = elem_size(dtype);
  QCHECK(check_rows("q", d_q, rows, q_stride, q_heads, head_dim, esz));
  QCHECK(check_rows("out", d_out, rows, out_stride, q_heads, head_dim, esz));
  QCHECK(check_words("lse and status", (const void*)((uintptr_t)d_lse | (uintptr_t)d_status)));
  if (!(scale > 0.0f) || !std::isfinite(2.0f * scale)) return fail(QORA_ERR_INVALID, "scale %g", (double)scale);
  if (window > 0x7fffffffu) return fail(QORA_ERR_INVALID, "window %u", window);
  QCHECK(check_pages(d_k_pages, d_v_pages, kv_heads, head_dim, elem_size(kv_dtype), num_pages, page_size, page_stride,
                     head_stride, slot_stride));
  QCHECK(check_batch(d_q_start, d_kv_len, d_table, table_stride, page_size, seqs));
  if (!d_work || (uintptr_t)d_work % 256 || work_bytes < QORA_PAGED_WORK_BYTES)
    return fail(QORA_ERR_INVALID, "the workspace needs %u bytes on a 256-byte boundary", QORA_PAGED_WORK_BYTES);
  if (rows == 0 || seqs == 0) return QORA_OK;
  if (max_q == 0) return fail(QORA_ERR_INVALID, "max_q is 0");
  QCHECK(check_apart("q and out", {d_q, q_stride, (uint64_t)q_heads * head_dim}, {d_out, out_stride, (uint64_t)q_heads * head_dim}, rows, esz));
  paged::AttnArgs a{};
  a.q = d_q, a.q_stride = (long long)q_stride;
  a.out = d_out, a.out_stride = (long long)out_stride;
  a.lse = d_lse;
  a.k_pages = d_k_pages, a.v_pages = d_v_pages;
  a.pg = {(int)num_pages, (int)page_size, (long long)page_stride, (long long)head_stride, (long long)slot_stride};
  a.batch = {d_q_start, d_kv_len, d_table, (int)table_stride, (int)seqs, (int)rows};
  a.hq = (int)q_heads, a.hk = (int)kv_heads, a.group = (int)(q_heads / kv_heads);
  a.group_inv = (65535 + a.group) / a.group;
  a.window = (int)window, a.scale = scale;
  a.max_q = (int)(max_q < rows ? max_q : rows);
  a.status = d_status;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == QORA_DT_F32 && kv_dtype == QORA_DT_F32) return launch_attn_d<float, float>(head_dim, a, d_work, s);
  if (dtype == QORA_DT_F32) return launch_attn_d<float, __half>(head_dim, a, d_work, s);
  if (dtype == QORA_DT_F16) return launch_attn_d<__half, __half>(head_dim, a, d_work, s);
  return launch_attn_d<__nv_bfloat16, __nv_bfloat16>(head_dim, a, d_work, s);
}

}  // extern "C"
