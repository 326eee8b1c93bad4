// Latent attention, absorbed form: sequence b's nodes t attend to the cached rows
// c_p = (c'_p, r_p) of its committed tokens and of its own nodes that the mask shows,
//   s_p = scale * (q_latent[t, h] . c'_p + q_rope[t, h] . r_p),
//   out[t, h] = sum_p exp(s_p - m) c'_p / sum_p exp(s_p - m),  m = max_p s_p;
// a row that sees nothing is zero with lse = -inf.
//
// latent_mma.cuh and latent_pair.cuh have the kernels; here are the C entries, the
// tensor maps and the launches.
#include <cmath>

#include "decode_common.cuh"
#include "latent_pair.cuh"

namespace b200kv {
namespace {

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

struct Workspace {
  int64_t joins, ml, o, total;
};
// After the decode kernels' counters, which calls on a shared workspace find as they left them.
Workspace workspace_of() {
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  Workspace w;
  w.joins = kMaxCounters * 4;
  w.ml = up(w.joins + latent::kMaxCtas * static_cast<int64_t>(sizeof(latent::Join)));
  w.o = up(w.ml + 2 * latent::kMaxCtas * latent::kTileRows * 8);
  w.total = up(w.o + int64_t{2} * latent::kMaxCtas * latent::kTileRows * latent::kRank * 4);
  return w;
}

// The attention (on single SMs or on pairs) and the join behind it.
template <typename T>
int launch(const CUtensorMap &qm, const CUtensorMap &rm, const CUtensorMap &hm, const CUtensorMap &pm,
           const CUtensorMap &sm, const latent::Args &a, bool pairs, int ctas, cudaStream_t stream) {
  const auto kernel = pairs ? latent::pair::latent_pair_kernel<T> : latent::latent_kernel<T>;
  const int smem = pairs ? latent::pair::kSmem : latent::kSmem;
  static int configured[2][64] = {{0}};
  int dev = 0;
  B200KV_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return set_error(B200KV_ERR_UNSUPPORTED, "device ordinal %d", dev);
  if (!__atomic_load_n(&configured[pairs][dev], __ATOMIC_ACQUIRE)) {
    B200KV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    __atomic_store_n(&configured[pairs][dev], 1, __ATOMIC_RELEASE);
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(latent::kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pairs ? 2 : 1;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, qm, rm, hm, pm, sm, a));
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>((a.box_nodes * a.head_box + 3) / 4));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, pairs ? latent::latent_join_kernel<T, true> : latent::latent_join_kernel<T, false>, a));
  return B200KV_OK;
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int64_t b200kv_latent_workspace_bytes(int64_t total_q, int64_t batch, int64_t num_heads) {
  if (total_q < 0 || batch < 0 || num_heads <= 0 || num_heads > latent::kMaxHeads) return -1;
  return workspace_of().total;
}

extern "C" int b200kv_latent_attention(const void *q_latent, int64_t q_latent_stride_t, int64_t q_latent_stride_h,
                                       const void *q_rope, int64_t q_rope_stride_t, int64_t q_rope_stride_h,
                                       int32_t dtype, const void *pool, const int32_t *block_table,
                                       int64_t block_table_stride, const int32_t *context_lens, const int32_t *q_indptr,
                                       const int64_t *tree_mask, int64_t mask_words, void *out, float *lse,
                                       int64_t total_q, int64_t batch, int64_t num_heads, int64_t num_blocks,
                                       int64_t max_blocks_per_seq, int64_t max_nodes, float scale, void *workspace,
                                       int64_t workspace_bytes, int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(dtype == B200KV_F16 || dtype == B200KV_BF16, "dtype %d is not fp16 or bf16", dtype);
  B200KV_CHECK_ARG(num_heads > 0, "num_heads %lld out of range", (long long)num_heads);
  if (num_heads > latent::kMaxHeads)
    return set_error(B200KV_ERR_UNSUPPORTED, "%lld heads unsupported (<= 512)", (long long)num_heads);
  B200KV_CHECK_ARG(batch >= 0 && total_q >= 0 && total_q * num_heads < (int64_t{1} << 31),
                   "batch or total_q * num_heads out of range");
  if (batch > 1024) return set_error(B200KV_ERR_UNSUPPORTED, "batch %lld > 1024 unsupported", (long long)batch);
  B200KV_CHECK_ARG(num_blocks > 0 && num_blocks < (int64_t{1} << 31) && max_blocks_per_seq > 0 &&
                       max_blocks_per_seq * kPageTokens < (int64_t{1} << 30),
                   "num_blocks or max_blocks_per_seq out of range");
  B200KV_CHECK_ARG(block_table_stride >= max_blocks_per_seq, "block_table_stride < max_blocks_per_seq");
  B200KV_CHECK_ARG(max_nodes > 0 && max_nodes < (int64_t{1} << 30), "max_nodes %lld out of range", (long long)max_nodes);
  B200KV_CHECK_ARG(!tree_mask || mask_words * 64 >= max_nodes, "mask_words (%lld) cover fewer than max_nodes (%lld)",
                   (long long)mask_words, (long long)max_nodes);
  B200KV_CHECK_ARG(std::isfinite(scale), "scale must be finite");
  latent::Args a{};
  a.head_box = static_cast<int>(num_heads < 64 ? num_heads : 64);
  a.tile_nodes = 64 / a.head_box;
  // Blocks of more than 64 rows, as far as the host knows, go to pairs of SMs (when this was chosen: 32
  // sequences, 128 heads: 60 us, in a form for single SMs 78; 8 trees, 128 heads: 101 and 158; 16
  // chains of 4, 32 heads: 35 and 41), others to single ones (64 sequences, 16 heads: 67 us, on pairs 81;
  // 300 short ones: 37 and 48).  More than 64 heads have the pairs alone, whose second CTA may be nearly
  // empty: 32 sequences of 4000 tokens take 59 us with 65 heads, 61 with 128, 53 with 64 on single SMs.
  // The host knows sums: a batch with few rows on average stays on single SMs though it has a large tree,
  // whose blocks read its pages each.  63 single tokens over 4000 and a tree of 64 nodes over 8000, 16
  // heads: 94 us, on pairs 96; the singles over 1000 and the tree over 60000: 221 and 129.
  const bool pairs = num_heads > 64 || total_q > batch * a.tile_nodes;
  a.stride = pairs ? 2 * static_cast<int>((num_heads + 127) / 128) : 1;
  a.block_nodes = pairs && num_heads <= 64 ? 2 * a.tile_nodes : a.tile_nodes;
  // the kernel counts its units of work in 31 bits
  if ((batch + total_q / a.tile_nodes + 1) * (max_blocks_per_seq + latent::kBegin) >= (int64_t{1} << 31))
    return set_error(B200KV_ERR_UNSUPPORTED, "2^31 or more steps of rows and tokens");
  if (total_q == 0) return B200KV_OK;
  B200KV_CHECK_ARG(batch > 0, "nodes without a sequence");
  B200KV_CHECK_ARG(q_latent && q_rope && pool && block_table && context_lens && q_indptr && out, "null pointer argument");
  auto strides_ok = [&](int64_t t, int64_t h) {
    return (total_q == 1 || (t % 8 == 0 && t > 0)) && (num_heads == 1 || (h % 8 == 0 && h > 0));
  };
  B200KV_CHECK_ARG(aligned_to(q_latent, 16) && aligned_to(q_rope, 16) && strides_ok(q_latent_stride_t, q_latent_stride_h) &&
                       strides_ok(q_rope_stride_t, q_rope_stride_h),
                   "q must be 16-byte aligned with positive strides that are multiples of 8 elements");
  B200KV_CHECK_ARG(aligned_to(pool, 16) && aligned_to(out, 16), "pool and out must be 16-byte aligned");
  const Workspace ws = workspace_of();
  if (!workspace || workspace_bytes < ws.total)
    return set_error(B200KV_ERR_WORKSPACE, "workspace of %lld bytes required (got %lld)", (long long)ws.total,
                     (long long)workspace_bytes);
  if (!aligned_to(workspace, 256)) return set_error(B200KV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  int dev = 0, sms = 0;
  int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  a.block_table = block_table, a.bt_stride = block_table_stride;
  a.ctx = context_lens, a.indptr = q_indptr;
  a.mask = reinterpret_cast<const uint64_t *>(tree_mask), a.words = mask_words;
  a.pool = pool, a.out = out, a.lse = lse;
  a.total_q = static_cast<int>(total_q), a.batch = static_cast<int>(batch), a.heads = static_cast<int>(num_heads);
  a.max_blocks = static_cast<int>(max_blocks_per_seq), a.max_nodes = static_cast<int>(max_nodes);
  a.num_blocks = static_cast<int>(num_blocks);
  a.box_nodes = static_cast<int>(max_nodes < a.tile_nodes ? max_nodes : a.tile_nodes);
  a.scale = scale, a.error_flag = error_flag;
  uint8_t *base = static_cast<uint8_t *>(workspace);
  a.joins = reinterpret_cast<latent::Join *>(base + ws.joins);
  a.part_ml = reinterpret_cast<float2 *>(base + ws.ml);
  a.part_o = reinterpret_cast<float *>(base + ws.o);
  const CUtensorMapDataType type = dtype == B200KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap qm, rm, hm, pm, sm;
  auto q_map = [&](CUtensorMap *map, const void *q, int64_t stride_t, int64_t stride_h, int64_t width) {
    // a dimension of one element may have any stride
    const int64_t sh = num_heads == 1 ? width : stride_h, st = total_q == 1 ? num_heads * width : stride_t;
    return encode(map, type, q,
                  {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(num_heads), static_cast<cuuint64_t>(total_q)},
                  {static_cast<cuuint64_t>(sh * 2), static_cast<cuuint64_t>(st * 2)},
                  {64, static_cast<cuuint32_t>(a.head_box), static_cast<cuuint32_t>(a.box_nodes)});
  };
  auto pool_map = [&](CUtensorMap *map, int sticks) {
    return encode(map, type, pool, {64, latent::kSticks * kPageTokens, static_cast<cuuint64_t>(num_blocks)},
                  {128, latent::kSticks * kPageTokens * 128}, {64, static_cast<cuuint32_t>(sticks * kPageTokens), 1});
  };
  if ((st = q_map(&qm, q_latent, q_latent_stride_t, q_latent_stride_h, latent::kRank)) != B200KV_OK) return st;
  if ((st = q_map(&rm, q_rope, q_rope_stride_t, q_rope_stride_h, latent::kRope)) != B200KV_OK) return st;
  if ((st = pool_map(&hm, 4)) != B200KV_OK || (st = pool_map(&pm, 2)) != B200KV_OK || (st = pool_map(&sm, 1)) != B200KV_OK)
    return st;
  const int ctas = (sms < latent::kMaxCtas ? sms : latent::kMaxCtas) / a.stride * a.stride;
  if (ctas == 0) return set_error(B200KV_ERR_UNSUPPORTED, "a GPU of %d SMs", sms);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const WorkspaceLock lock(workspace);
  return dtype == B200KV_F16 ? launch<__half>(qm, rm, hm, pm, sm, a, pairs, ctas, s)
                             : launch<__nv_bfloat16>(qm, rm, hm, pm, sm, a, pairs, ctas, s);
}
