// Latent attention, expanded form, for prompts: row i of sequence b (of n_b, over
// m_b tokens) and head h attend to tokens p <= m_b - n_b + i (or all),
//   s_p = scale * (q[i, h, :128] . k_nope[p, h] + q[i, h, 128:] . k_rope[p]),
//   out[i, h] = sum_p exp(s_p - m) v[p, h] / sum_p exp(s_p - m),  m = max_p s_p;
// a row that sees nothing is zero with lse = -inf.
//
// prompt_mma.cuh has the kernels; here are the C entries and the tensor maps.
#include <cmath>

#include "decode_common.cuh"
#include "prompt_mma.cuh"

namespace b200kv {
namespace {

// Rows of `width` elements of `heads` heads and `rows` tokens, a box of 64 elements x `box_rows` tokens of a head.
int encode(CUtensorMap *map, CUtensorMapDataType type, const void *base, int64_t width, int64_t heads, int64_t rows,
           int64_t stride_h, int64_t stride_t, int box_rows) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return set_error(B200KV_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  // a dimension of one element may have any stride
  const int64_t sh = heads == 1 ? width : stride_h, st = rows == 1 ? heads * width : stride_t;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh * 2), static_cast<cuuint64_t>(st * 2)};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(box_rows)}, estr[3] = {1, 1, 1};
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
  w.ml = up(w.joins + prompt::kMaxCtas * static_cast<int64_t>(sizeof(prompt::Join)));
  w.o = up(w.ml + 2 * prompt::kMaxCtas * 256 * 8);
  w.total = up(w.o + int64_t{2} * prompt::kMaxCtas * 256 * prompt::kDim * 4);
  return w;
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int64_t b200kv_prompt_workspace_bytes(int64_t total_q, int64_t total_kv, int64_t batch, int64_t num_heads) {
  if (total_q < 0 || total_kv < 0 || batch < 0 || num_heads <= 0) return -1;
  return workspace_of().total;
}

extern "C" int b200kv_latent_prompt_attention(const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k_nope,
                                              int64_t k_stride_t, int64_t k_stride_h, const void *k_rope,
                                              int64_t k_rope_stride_t, const void *v, int64_t v_stride_t,
                                              int64_t v_stride_h, int32_t dtype, const int32_t *q_indptr,
                                              const int32_t *kv_indptr, void *out, float *lse, int64_t total_q,
                                              int64_t total_kv, int64_t batch, int64_t num_heads, float scale,
                                              int32_t causal, void *workspace, int64_t workspace_bytes,
                                              int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(dtype == B200KV_F16 || dtype == B200KV_BF16, "dtype %d is not fp16 or bf16", dtype);
  B200KV_CHECK_ARG(num_heads > 0 && num_heads <= 65536, "num_heads %lld out of range", (long long)num_heads);
  B200KV_CHECK_ARG(batch >= 0 && total_q >= 0 && total_kv >= 0 && total_q * num_heads < (int64_t{1} << 31) &&
                       total_kv < (int64_t{1} << 30),
                   "batch, total_q * num_heads or total_kv out of range");
  if (batch > 1024) return set_error(B200KV_ERR_UNSUPPORTED, "batch %lld > 1024 unsupported", (long long)batch);
  B200KV_CHECK_ARG(std::isfinite(scale), "scale must be finite");
  // The kernel counts a share's units of work, and one more block's, in 31 bits: kBegin + 4 a tile for a
  // block of 256 rows.  At most, that is: the rows of a batch meet their own sequences' tokens only.
  const int64_t blocks = total_q / 256 + batch, tiles = total_kv / prompt::kTok + 1;
  const int64_t units = (blocks * (prompt::kBegin2 + 4) + 4 * (total_q / 256 * tiles + tiles + batch)) * num_heads;
  auto countable = [&](int shares) { return units / shares + 4 * tiles + 64 < (int64_t{1} << 31); };
  if (!countable(prompt::kMaxCtas))
    return set_error(B200KV_ERR_UNSUPPORTED, "2^31 or more steps of rows and tokens for an SM");
  if (total_q == 0) return B200KV_OK;
  B200KV_CHECK_ARG(batch > 0, "rows without a sequence");
  B200KV_CHECK_ARG(q && q_indptr && kv_indptr && out && (total_kv == 0 || (k_nope && k_rope && v)), "null pointer argument");
  auto strides_ok = [&](int64_t rows, int64_t t, int64_t h) {
    return (rows <= 1 || (t % 8 == 0 && t > 0)) && (num_heads == 1 || (h % 8 == 0 && h > 0));
  };
  B200KV_CHECK_ARG(aligned_to(q, 16) && aligned_to(k_nope, 16) && aligned_to(k_rope, 16) && aligned_to(v, 16) &&
                       aligned_to(out, 16),
                   "buffers must be 16-byte aligned");
  B200KV_CHECK_ARG(strides_ok(total_q, q_stride_t, q_stride_h) && strides_ok(total_kv, k_stride_t, k_stride_h) &&
                       strides_ok(total_kv, v_stride_t, v_stride_h) &&
                       (total_kv <= 1 || (k_rope_stride_t % 8 == 0 && k_rope_stride_t > 0)),
                   "strides must be positive multiples of 8 elements");
  const Workspace ws = workspace_of();
  if (!workspace || workspace_bytes < ws.total)
    return set_error(B200KV_ERR_WORKSPACE, "workspace of %lld bytes required (got %lld)", (long long)ws.total,
                     (long long)workspace_bytes);
  if (!aligned_to(workspace, 256)) return set_error(B200KV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  int dev = 0, sms = 0;
  int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  const int ctas = sms < prompt::kMaxCtas ? sms : prompt::kMaxCtas;
  if (!countable(ctas)) return set_error(B200KV_ERR_UNSUPPORTED, "2^31 or more steps of rows and tokens for an SM");
  prompt::Args a{};
  a.q_indptr = q_indptr, a.kv_indptr = kv_indptr;
  a.v = v, a.v_st = v_stride_t, a.v_sh = v_stride_h;
  a.out = out, a.lse = lse;
  a.total_q = static_cast<int>(total_q), a.total_kv = static_cast<int>(total_kv);
  a.batch = static_cast<int>(batch), a.heads = static_cast<int>(num_heads), a.causal = causal != 0;
  a.scale = scale, a.error_flag = error_flag;
  uint8_t *base = static_cast<uint8_t *>(workspace);
  a.joins = reinterpret_cast<prompt::Join *>(base + ws.joins);
  a.part_ml = reinterpret_cast<float2 *>(base + ws.ml);
  a.part_o = reinterpret_cast<float *>(base + ws.o);
  const CUtensorMapDataType type = dtype == B200KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // no token at all: the maps are of q's rows, and every row is masked
  const bool none = total_kv == 0;
  const int64_t rows = none ? total_q : total_kv;
  CUtensorMap qm, km, rm, vm;
  st = encode(&qm, type, q, prompt::kNope + prompt::kRope, num_heads, total_q, q_stride_h, q_stride_t,
              prompt::kTile);
  if (st == B200KV_OK)
    st = encode(&km, type, none ? q : k_nope, prompt::kNope, num_heads, rows, none ? q_stride_h : k_stride_h,
                none ? q_stride_t : k_stride_t, prompt::kTok);
  if (st == B200KV_OK)
    st = encode(&rm, type, none ? q : k_rope, prompt::kRope, 1, rows, 0, none ? q_stride_t : k_rope_stride_t,
                prompt::kTok);
  if (st == B200KV_OK)
    st = encode(&vm, type, none ? q : v, prompt::kDim, num_heads, rows, none ? q_stride_h : v_stride_h,
                none ? q_stride_t : v_stride_t, prompt::kTok);
  if (st != B200KV_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const WorkspaceLock lock(workspace);
  return dtype == B200KV_F16 ? prompt::launch<__half>(qm, km, rm, vm, a, ctas, s)
                             : prompt::launch<__nv_bfloat16>(qm, km, rm, vm, a, ctas, s);
}
