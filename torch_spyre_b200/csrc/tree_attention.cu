// Attention of drafted tokens over the paged cache: sequence b's nodes
// t = q_indptr[b] .. q_indptr[b + 1] - 1 attend to its ctx_b committed tokens
// and to those of its own nodes (cached at positions ctx_b, ctx_b + 1, ...)
// that the tree mask shows:
//   out[t, h] = sum_p exp(s_p - m) v_p / sum_p exp(s_p - m),
//   s_p = scale * q[t, h] . k_p,  m = max_p s_p   over the visible p;
// a row that sees nothing is zero with lse = -inf.
//
// tree_mma.cuh has the kernels; here are the C entries, the masks and the
// tensor maps.
#include <cmath>

#include "decode_common.cuh"
#include "rows.cuh"
#include "tree_attention.h"

namespace b200kv {
namespace {

// ------------------------------------------------------------------- masks --
// A thread per node walks up to its root.  Latency: one dependent load per level
// (16 drafts of up to 64 nodes: 3 us).
__global__ void __launch_bounds__(128) tree_mask_kernel(const int32_t *parents, const int32_t *indptr, int batch,
                                                        int64_t total, int64_t words, uint64_t *mask,
                                                        int32_t *error_flag) {
  // (the attention that comes next sets itself up meanwhile; it waits for the mask)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= total) return;
  uint64_t *row = mask + i * words;
  for (int64_t w = 0; w < words; ++w) row[w] = 0;
  int lo = 0, hi = batch - 1;  // the last sequence that begins at or before i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(indptr + mid) <= i) lo = mid; else hi = mid - 1;
  }
  const int64_t first = __ldg(indptr + lo);
  int64_t j = i - first;
  if (first < 0 || j < 0 || j >= words * 64 || i >= __ldg(indptr + lo + 1)) {
    if (error_flag) atomicOr(error_flag, B200KV_DEVERR_BAD_LEN);
    return;
  }
  int parent = __ldg(parents + i);
  for (;;) {
    if (parent == -2) {  // pruned, itself or by an ancestor: sees nothing
      for (int64_t w = 0; w < words; ++w) row[w] = 0;
      return;
    }
    row[j >> 6] |= uint64_t{1} << (j & 63);
    if (parent == -1) return;
    if (parent < 0 || parent >= j) {  // parents come before their children
      if (error_flag) atomicOr(error_flag, B200KV_DEVERR_BAD_LEN);
      return;
    }
    j = parent;
    parent = __ldg(parents + first + j);
  }
}

// --------------------------------------------------------------------- maps --
constexpr int kBoxElems = 64;  // 16-bit elements of a 128-byte operand row

int encode(CUtensorMap *map, CUtensorMapDataType type, const void *base, const cuuint64_t (&dims)[3],
           const cuuint64_t (&strides)[2], const cuuint32_t (&box)[3]) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return set_error(B200KV_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, type, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(B200KV_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return B200KV_OK;
}

// Pages of a 16-bit pool, one box per page and 64-element stick column, into the
// 128-byte swizzle of an operand tile.  (8-bit pages come by plain bulk copies.)
int pool_map(CUtensorMap *map, const void *pool, int64_t pages, int64_t dim, CUtensorMapDataType type) {
  const cuuint64_t rows = dim / kBoxElems * kPageTokens;
  return encode(map, type, pool, {kBoxElems, rows, static_cast<cuuint64_t>(pages)}, {128, rows * 128},
                {kBoxElems, kPageTokens, 1});
}

struct Workspace {
  int64_t joins, ml, o, total;
};
// After the decode kernels' counters, which calls on a shared workspace find as
// they left them.
Workspace workspace_of(int64_t dim) {
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  Workspace w;
  w.joins = kMaxCounters * 4;
  w.ml = up(w.joins + tree::kMaxCtas * static_cast<int64_t>(sizeof(tree::Join)));
  w.o = up(w.ml + 2 * tree::kMaxCtas * 256 * 8);
  w.total = up(w.o + 2 * tree::kMaxCtas * 256 * dim * 4);
  return w;
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int64_t b200kv_tree_workspace_bytes(int64_t total_q, int64_t batch, int64_t num_q_heads,
                                               int64_t num_kv_heads, int64_t head_dim) {
  if (total_q < 0 || batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128))
    return -1;
  return workspace_of(head_dim).total;
}

extern "C" int b200kv_tree_mask(const int32_t *parents, const int32_t *q_indptr, int64_t batch, int64_t total_q,
                                int64_t mask_words, int64_t *mask, int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(batch >= 0 && batch < (int64_t{1} << 31) && total_q >= 0 && total_q < (int64_t{1} << 31),
                   "batch or total_q out of range");
  B200KV_CHECK_ARG(mask_words > 0 && mask_words <= (1 << 20), "mask_words %lld out of range", (long long)mask_words);
  if (total_q == 0) return B200KV_OK;
  B200KV_CHECK_ARG(batch > 0, "nodes without a sequence");
  B200KV_CHECK_ARG(parents && q_indptr && mask, "null pointer argument");
  tree_mask_kernel<<<static_cast<unsigned>((total_q + 127) / 128), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      parents, q_indptr, static_cast<int>(batch), total_q, mask_words, reinterpret_cast<uint64_t *>(mask), error_flag);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}

extern "C" int b200kv_tree_attention(const void *q, int32_t q_dtype, int64_t q_stride_t, int64_t q_stride_h,
                                     const void *k_pool, const void *v_pool, int32_t pool_dtype,
                                     const float *k_scales, const float *v_scales, const int32_t *block_table,
                                     int64_t block_table_stride, const int32_t *context_lens,
                                     const int32_t *q_indptr, const int64_t *tree_mask, int64_t mask_words, void *out,
                                     float *lse, int64_t total_q, int64_t batch, int64_t num_q_heads,
                                     int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks,
                                     int64_t max_blocks_per_seq, int64_t max_nodes, float scale, void *workspace,
                                     int64_t workspace_bytes, int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(q_dtype == B200KV_F16 || q_dtype == B200KV_BF16, "q dtype %d is not fp16 or bf16", q_dtype);
  const bool k8 = pool_dtype == B200KV_I8 || pool_dtype == B200KV_E4M3;
  B200KV_CHECK_ARG(k8 || pool_dtype == q_dtype, "a 16-bit pool must have q's dtype");
  if (head_dim != 128 && !(head_dim == 64 && !k8))
    return set_error(B200KV_ERR_UNSUPPORTED, "head_dim %lld unsupported (128, or 64 in 16-bit pools)",
                     (long long)head_dim);
  B200KV_CHECK_ARG(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
                   "num_q_heads (%lld) must be a positive multiple of num_kv_heads (%lld)", (long long)num_q_heads,
                   (long long)num_kv_heads);
  if (num_q_heads / num_kv_heads > 128)
    return set_error(B200KV_ERR_UNSUPPORTED, "GQA group size %lld unsupported (<= 128)",
                     (long long)(num_q_heads / num_kv_heads));
  B200KV_CHECK_ARG(batch >= 0 && total_q >= 0 && total_q * num_q_heads < (int64_t{1} << 31),
                   "batch or total_q * num_q_heads out of range");
  if (batch > 1024) return set_error(B200KV_ERR_UNSUPPORTED, "batch %lld > 1024 unsupported", (long long)batch);
  B200KV_CHECK_ARG(num_blocks > 0 && num_blocks * num_kv_heads < (int64_t{1} << 31) && max_blocks_per_seq > 0 &&
                       max_blocks_per_seq * kPageTokens < (int64_t{1} << 30),
                   "num_blocks or max_blocks_per_seq out of range");
  B200KV_CHECK_ARG(block_table_stride >= max_blocks_per_seq, "block_table_stride < max_blocks_per_seq");
  B200KV_CHECK_ARG(max_nodes > 0 && max_nodes < (int64_t{1} << 30), "max_nodes %lld out of range", (long long)max_nodes);
  B200KV_CHECK_ARG(!tree_mask || mask_words * 64 >= max_nodes, "mask_words (%lld) cover fewer than max_nodes (%lld)",
                   (long long)mask_words, (long long)max_nodes);
  B200KV_CHECK_ARG(std::isfinite(scale), "scale must be finite");
  // the kernel counts its units of work in 31 bits
  // (a block of one Q tile holds at least 65 of total_q * group rows, and 9 + 2 a tile units; of two 130, and 13 + 4)
  if ((batch + total_q * (num_q_heads / num_kv_heads) / 64 + 1) * num_kv_heads * (2 * max_blocks_per_seq + 17) >=
      (int64_t{1} << 31))
    return set_error(B200KV_ERR_UNSUPPORTED, "2^31 or more steps of rows and tokens");
  if (total_q == 0) return B200KV_OK;
  B200KV_CHECK_ARG(batch > 0, "nodes without a sequence");
  B200KV_CHECK_ARG(q && k_pool && v_pool && block_table && context_lens && q_indptr && out, "null pointer argument");
  B200KV_CHECK_ARG(!k8 || (k_scales && v_scales), "8-bit pools need k_scales and v_scales");
  B200KV_CHECK_ARG(!k8 || (aligned_to(k_scales, 16) && aligned_to(v_scales, 16)), "scales must be 16-byte aligned");
  B200KV_CHECK_ARG(aligned_to(q, 16) && (total_q == 1 || (q_stride_t % 8 == 0 && q_stride_t > 0)) &&
                       (num_q_heads == 1 || (q_stride_h % 8 == 0 && q_stride_h > 0)),
                   "q must be 16-byte aligned with positive strides that are multiples of 8 elements");
  B200KV_CHECK_ARG(aligned_to(k_pool, 16) && aligned_to(v_pool, 16) && aligned_to(out, 16), "pools and out must be 16-byte aligned");
  const int64_t need = b200kv_tree_workspace_bytes(total_q, batch, num_q_heads, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need)
    return set_error(B200KV_ERR_WORKSPACE, "workspace of %lld bytes required (got %lld)", (long long)need,
                     (long long)workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return set_error(B200KV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  int dev = 0, sms = 0;
  int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  const int group = static_cast<int>(num_q_heads / num_kv_heads);
  tree::Args a{};
  a.block_table = block_table, a.bt_stride = block_table_stride;
  a.ctx = context_lens, a.indptr = q_indptr;
  a.mask = reinterpret_cast<const uint64_t *>(tree_mask), a.words = mask_words;
  a.k_scales = k_scales, a.v_scales = v_scales, a.k_pool = k_pool, a.v_pool = v_pool;
  a.out = out, a.lse = lse;
  a.total_q = static_cast<int>(total_q), a.batch = static_cast<int>(batch);
  a.hq = static_cast<int>(num_q_heads), a.hkv = static_cast<int>(num_kv_heads), a.group = group;
  a.max_blocks = static_cast<int>(max_blocks_per_seq), a.max_nodes = static_cast<int>(max_nodes);
  a.num_blocks = static_cast<int>(num_blocks);
  a.tile_nodes = 128 / group;
  a.scale = scale;
  a.error_flag = error_flag;
  const Workspace ws = workspace_of(head_dim);
  uint8_t *base = static_cast<uint8_t *>(workspace);
  a.joins = reinterpret_cast<tree::Join *>(base + ws.joins);
  a.part_ml = reinterpret_cast<float2 *>(base + ws.ml);
  a.part_o = reinterpret_cast<float *>(base + ws.o);

  const CUtensorMapDataType type = q_dtype == B200KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // Q: 64 elements x the KV head's query heads x the nodes of a tile (no more
  // than a sequence can have), rows node-major
  a.small_boxes = k8 && 32 % group == 0;
  const int64_t box_nodes = a.small_boxes ? 32 / group : (max_nodes < a.tile_nodes ? max_nodes : a.tile_nodes);
  a.box_nodes = static_cast<int>(box_nodes);
  a.q_box_bytes = static_cast<uint32_t>(box_nodes * group * 128);
  CUtensorMap qm, km{}, vm{};
  // a dimension of one element may have any stride
  const int64_t qs_h = num_q_heads == 1 ? head_dim : q_stride_h, qs_t = total_q == 1 ? num_q_heads * head_dim : q_stride_t;
  st = encode(&qm, type, q,
              {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(num_q_heads), static_cast<cuuint64_t>(total_q)},
              {static_cast<cuuint64_t>(qs_h * 2), static_cast<cuuint64_t>(qs_t * 2)},
              {kBoxElems, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(box_nodes)});
  if (st != B200KV_OK) return st;
  if (!k8) {
    st = pool_map(&km, k_pool, num_blocks * num_kv_heads, head_dim, type);
    if (st != B200KV_OK) return st;
    st = pool_map(&vm, v_pool, num_blocks * num_kv_heads, head_dim, type);
    if (st != B200KV_OK) return st;
  }
  const int ctas = sms < tree::kMaxCtas ? sms : tree::kMaxCtas;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const WorkspaceLock lock(workspace);
  return q_dtype == B200KV_F16 ? tree::launch_f16(qm, km, vm, a, static_cast<int>(head_dim), pool_dtype, ctas, s)
                               : tree::launch_bf16(qm, km, vm, a, static_cast<int>(head_dim), pool_dtype, ctas, s);
}
