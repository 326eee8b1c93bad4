// Attention of drafted tokens over the paged cache: sequence b's nodes
// t = q_indptr[b] .. q_indptr[b + 1] - 1 attend to its ctx_b committed tokens
// and to those of its own nodes (cached at positions ctx_b, ctx_b + 1, ...)
// that the tree mask shows:
//   out[t, h] = sum_p exp(s_p - m) v_p / sum_p exp(s_p - m),
//   s_p = scale * q[t, h] . k_p,  m = max_p s_p   over the visible p;
// a row that sees nothing is zero with lse = -inf.
#include <cmath>

#include "rows.cuh"

namespace b200kv {
namespace {

constexpr float kLog2e = 1.44269504088896341f;

struct TreeArgs {
  const void *q;
  int64_t q_st, q_sh;
  const void *k_pool, *v_pool;
  const float *k_scales, *v_scales;
  const int32_t *block_table;
  int64_t bt_stride;
  const int32_t *ctx, *indptr;
  const uint64_t *mask;  // [N, words], null: a chain
  int64_t words;
  void *out;  // contiguous [N, Hq, D]
  float *lse;
  int64_t total_q, num_blocks;
  int batch, hq, hkv, max_blocks, max_nodes;
  float scale;
  int32_t *error_flag;
};

// ------------------------------------------------------------------- masks --
__global__ void __launch_bounds__(128) tree_mask_kernel(const int32_t *parents, const int32_t *indptr, int batch,
                                                        int64_t total, int64_t words, uint64_t *mask,
                                                        int32_t *error_flag) {
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
  if (parent == -2) return;  // pruned: sees nothing
  for (;;) {
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

// -------------------------------------------------------------- attention --
template <typename T, int kCache>
__device__ __forceinline__ float cache_value(const void *pool, int64_t at) {
  if constexpr (kCache == B200KV_I8) {
    return static_cast<float>(static_cast<const int8_t *>(pool)[at]);
  } else if constexpr (kCache == B200KV_E4M3) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t *>(pool)[at], __NV_E4M3)));
  } else {
    return to_float(static_cast<const T *>(pool)[at]);
  }
}

// One warp per (node, query head); lane l owns dims l, l + 32, ...
template <typename T, int D, int kCache>
__global__ void __launch_bounds__(256) tree_rows_kernel(const TreeArgs a) {
  constexpr int kStick = kCache == B200KV_F16 ? 64 : 128;
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= a.total_q * a.hq) return;
  const int64_t t = row / a.hq;
  const int h = static_cast<int>(row - t * a.hq), kvh = h / (a.hq / a.hkv);
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(a.indptr + mid) <= t) lo = mid; else hi = mid - 1;
  }
  const int b = lo;
  const int64_t first = __ldg(a.indptr + b);
  const int cap = a.max_blocks * kPageTokens;
  int ctx = __ldg(a.ctx + b);
  int nodes = static_cast<int>(__ldg(a.indptr + b + 1) - first);
  const int node = static_cast<int>(t - first);
  if (ctx < 0 || ctx > cap || nodes > a.max_nodes || ctx + nodes > cap || node < 0 || node >= nodes) {
    if (lane == 0 && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
    ctx = ctx < 0 ? 0 : min(ctx, cap);
    nodes = max(0, min(min(nodes, a.max_nodes), cap - ctx));
  }
  float q[kPer], o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    q[i] = to_float(static_cast<const T *>(a.q)[t * a.q_st + h * a.q_sh + lane + 32 * i]) * (a.scale * kLog2e);
    o[i] = 0.f;
  }
  float m = -CUDART_INF_F, l = 0.f;
  for (int p = 0; p < ctx + nodes; ++p) {
    if (p >= ctx) {
      const int j = p - ctx;
      const bool see = a.mask ? (j < a.words * 64 && ((__ldg(a.mask + t * a.words + (j >> 6)) >> (j & 63)) & 1)) : j <= node;
      if (!see) continue;
    }
    const int blk = __ldg(a.block_table + b * a.bt_stride + (p >> 6));
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0 && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_BLOCK);
      continue;
    }
    const int64_t page = int64_t(blk) * a.hkv + kvh;
    float s = 0.f;
    int64_t at[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 32 * i;
      at[i] = (page * (D / kStick) + d / kStick) * (64 * kStick) + int64_t(p & 63) * kStick + d % kStick;
      s += q[i] * cache_value<T, kCache>(a.k_pool, at[i]);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    float vs = 1.f;
    if (kCache != B200KV_F16) {
      s *= __ldg(a.k_scales + page * 64 + (p & 63));
      vs = __ldg(a.v_scales + page * 64 + (p & 63));
    }
    const float mn = fmaxf(m, s);
    const float keep = exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * keep + w * vs * cache_value<T, kCache>(a.v_pool, at[i]);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T *out = static_cast<T *>(a.out) + row * D;
#pragma unroll
  for (int i = 0; i < kPer; ++i) from_float(out[lane + 32 * i], l == 0.f ? 0.f : o[i] * inv);
  if (lane == 0 && a.lse) a.lse[row] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) / kLog2e;
}

template <typename T, int D, int kCache>
int launch_tree(const TreeArgs &a, cudaStream_t s) {
  const int64_t blocks = (a.total_q * a.hq + 7) / 8;
  tree_rows_kernel<T, D, kCache><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}
template <typename T>
int tree_cache(const TreeArgs &a, int64_t dim, int cache, cudaStream_t s) {
  if (cache == B200KV_I8) return launch_tree<T, 128, B200KV_I8>(a, s);
  if (cache == B200KV_E4M3) return launch_tree<T, 128, B200KV_E4M3>(a, s);
  return dim == 64 ? launch_tree<T, 64, B200KV_F16>(a, s) : launch_tree<T, 128, B200KV_F16>(a, s);
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int64_t b200kv_tree_workspace_bytes(int64_t total_q, int64_t batch, int64_t num_q_heads,
                                               int64_t num_kv_heads, int64_t head_dim) {
  if (total_q < 0 || batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128))
    return -1;
  return 256;
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
  if (total_q == 0) return B200KV_OK;
  B200KV_CHECK_ARG(batch > 0, "nodes without a sequence");
  B200KV_CHECK_ARG(q && k_pool && v_pool && block_table && context_lens && q_indptr && out, "null pointer argument");
  B200KV_CHECK_ARG(!k8 || (k_scales && v_scales), "8-bit pools need k_scales and v_scales");
  B200KV_CHECK_ARG(aligned_to(q, 16) && q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && q_stride_t > 0 && q_stride_h > 0,
                   "q must be 16-byte aligned with positive strides that are multiples of 8 elements");
  B200KV_CHECK_ARG(aligned_to(k_pool, 16) && aligned_to(v_pool, 16) && aligned_to(out, 16), "pools and out must be 16-byte aligned");
  const int64_t need = b200kv_tree_workspace_bytes(total_q, batch, num_q_heads, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need)
    return set_error(B200KV_ERR_WORKSPACE, "workspace of %lld bytes required (got %lld)", (long long)need,
                     (long long)workspace_bytes);
  TreeArgs a{};
  a.q = q, a.q_st = q_stride_t, a.q_sh = q_stride_h;
  a.k_pool = k_pool, a.v_pool = v_pool, a.k_scales = k_scales, a.v_scales = v_scales;
  a.block_table = block_table, a.bt_stride = block_table_stride;
  a.ctx = context_lens, a.indptr = q_indptr;
  a.mask = reinterpret_cast<const uint64_t *>(tree_mask), a.words = mask_words;
  a.out = out, a.lse = lse;
  a.total_q = total_q, a.num_blocks = num_blocks;
  a.batch = static_cast<int>(batch), a.hq = static_cast<int>(num_q_heads), a.hkv = static_cast<int>(num_kv_heads);
  a.max_blocks = static_cast<int>(max_blocks_per_seq), a.max_nodes = static_cast<int>(max_nodes);
  a.scale = scale;
  a.error_flag = error_flag;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return q_dtype == B200KV_F16 ? tree_cache<__half>(a, head_dim, pool_dtype, s)
                               : tree_cache<__nv_bfloat16>(a, head_dim, pool_dtype, s);
}
