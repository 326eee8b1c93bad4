// Rows of a latent cache: one row a token, 512 latent elements that all heads
// share as key and value, then 64 rotary key elements, 16-bit, in the paged
// stick layout with one "head" of nine sticks.
//   store   latent: y = x / sqrt(mean(x^2) + eps) * w  (or x as it is),
//           key: turned by its rotary position; the heads' 64 rotary query
//           elements turned beside them.  fp32, rounded once.
//   commit  the accepted path of a drafted tree moved (kv_rows.cu).
#include "rows.cuh"

namespace b200kv {
namespace {

constexpr int kRank = B200KV_LATENT_RANK, kRope = B200KV_LATENT_ROPE, kRow = kRank + kRope;

struct StoreArgs {
  const void *latent, *k_rope, *q_rope;
  int64_t latent_sn, rope_sn, q_sn, q_sh;
  const void *weight;
  float eps;
  void *pool, *q_out;  // q_out contiguous [N, H, 64]
  const int64_t *slots;
  const float2 *table;
  int64_t max_pos;
  const int32_t *positions;
  int64_t num_slots;
  int tokens, heads, parts;
  int32_t *error_flag;
};

// Offset, in elements, of element e (a multiple of 8) of the row at `slot`.
__device__ __forceinline__ int64_t row_at(int64_t slot, int e) {
  return ((slot / kPageTokens * (kRow / 64) + e / 64) * kPageTokens + slot % kPageTokens) * 64 + e % 64;
}

// A warp per token: part 0 the latent row (16 elements a lane) and the key, the
// others kHeads heads' queries each.  Four lanes turn a row of 64: lane l has pairs
// 8l .. 8l + 7, which are two 16-byte vectors in either layout, so that the eight
// rows of a step need one set of cosines and sines.
//
// Bound: bytes, and how many of them are asked for at a time: all that a warp loads but
// the angles, which wait for a position, is under way before it waits for any of it
// (one thing after the other: 32.0 instead of 27.8 us below).  16381 tokens, with an L2
// full of lines that have to be written back first: 16 heads 27.8 us (3.9 TB/s), 29.9
// with 32 heads to a warp; 128 heads 97.6 us with 32 (5.9 TB/s), 117 with 16.
template <typename T, int kTurn, int kHeads>  // kTurn: 0 none, 1 half, 2 interleaved
__global__ void __launch_bounds__(256, 4) latent_store_kernel(const StoreArgs a) {
  const int lane = threadIdx.x & 31;
  const uint32_t unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / a.parts), part = static_cast<int>(unit % a.parts);
  if (t >= a.tokens) return;
  const int l = lane & 3;
  const int e0 = kTurn == 2 ? 16 * l : 8 * l, e1 = kTurn == 2 ? e0 + 8 : e0 + 32;  // the lane's vectors
  float2 cs[8];
  const int p_in = kTurn != 0 ? __ldg(a.positions + t) : 0;
  auto angles = [&] {  // (called with the rows under way)
    if (kTurn == 0) return;
    const int64_t p = p_in < 0 ? 0 : (p_in >= a.max_pos ? a.max_pos - 1 : p_in);
    const float4 *row = reinterpret_cast<const float4 *>(a.table + p * (kRope / 2) + 8 * l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldg(row + i);
      cs[2 * i] = make_float2(v.x, v.y), cs[2 * i + 1] = make_float2(v.z, v.w);
    }
  };
  auto turn = [&](uint4 &u, uint4 &v) {
    if (kTurn == 0) return;
    float x[8], y[8];
    unpack8(u, x, T());
    unpack8(v, y, T());
    if (kTurn == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn_pair(x[i], y[i], cs[i].x, cs[i].y, x[i], y[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        turn_pair(x[2 * i], x[2 * i + 1], cs[i].x, cs[i].y, x[2 * i], x[2 * i + 1]);
        turn_pair(y[2 * i], y[2 * i + 1], cs[4 + i].x, cs[4 + i].y, y[2 * i], y[2 * i + 1]);
      }
    }
    u = pack8(x, T());
    v = pack8(y, T());
  };
  if (part > 0) {
    const int h0 = (part - 1) * kHeads + (lane >> 2);
    const T *q = static_cast<const T *>(a.q_rope) + t * a.q_sn;
    T *out = static_cast<T *>(a.q_out) + static_cast<int64_t>(t) * a.heads * kRope;
    uint4 u[kHeads / 8], v[kHeads / 8];
#pragma unroll
    for (int i = 0; i < kHeads / 8; ++i) {
      const int h = h0 + 8 * i;
      if (h >= a.heads) continue;
      u[i] = __ldg(reinterpret_cast<const uint4 *>(q + h * a.q_sh + e0));
      v[i] = __ldg(reinterpret_cast<const uint4 *>(q + h * a.q_sh + e1));
    }
    angles();
#pragma unroll
    for (int i = 0; i < kHeads / 8; ++i) {
      const int h = h0 + 8 * i;
      if (h >= a.heads) continue;
      turn(u[i], v[i]);
      *reinterpret_cast<uint4 *>(out + h * kRope + e0) = u[i];
      *reinterpret_cast<uint4 *>(out + h * kRope + e1) = v[i];
    }
    return;
  }
  const int64_t slot = __ldg(a.slots + t);
  const T *x = static_cast<const T *>(a.latent) + t * a.latent_sn;
  T *pool = static_cast<T *>(a.pool);
  uint4 raw[2], ku, kv;
#pragma unroll
  for (int i = 0; i < 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(x + 256 * i + 8 * lane));
  if (lane < 4) {
    const T *k = static_cast<const T *>(a.k_rope) + t * a.rope_sn;
    ku = __ldg(reinterpret_cast<const uint4 *>(k + e0));
    kv = __ldg(reinterpret_cast<const uint4 *>(k + e1));
  }
  // (all of it is under way before the first of it is waited for)
  if (kTurn != 0 && lane == 0 && (p_in < 0 || p_in >= a.max_pos) && a.error_flag)
    atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
  if (slot < 0 || slot >= a.num_slots) {
    if (slot >= 0 && lane == 0 && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_SLOT);
    return;
  }
  if (lane < 4) angles();
  if (a.weight) {
    uint4 weight[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      weight[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.weight) + 256 * i + 8 * lane));
    float f[2][8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unpack8(raw[i], f[i], T());
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(f[i][j], f[i][j], sum);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const float by = 1.f / sqrtf(sum * (1.f / kRank) + a.eps);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float w[8];
      unpack8(weight[i], w, T());
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = f[i][j] * by * w[j];
      raw[i] = pack8(f[i], T());
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) *reinterpret_cast<uint4 *>(pool + row_at(slot, 256 * i + 8 * lane)) = raw[i];
  if (lane < 4) {
    turn(ku, kv);
    *reinterpret_cast<uint4 *>(pool + row_at(slot, kRank + e0)) = ku;
    *reinterpret_cast<uint4 *>(pool + row_at(slot, kRank + e1)) = kv;
  }
}

template <typename T, int kHeads>
void launch(const StoreArgs &a, int turn, unsigned grid, cudaStream_t s) {
  if (turn == 0)
    latent_store_kernel<T, 0, kHeads><<<grid, 256, 0, s>>>(a);
  else if (turn == 1)
    latent_store_kernel<T, 1, kHeads><<<grid, 256, 0, s>>>(a);
  else
    latent_store_kernel<T, 2, kHeads><<<grid, 256, 0, s>>>(a);
}
template <typename T>
void launch(const StoreArgs &a, int turn, int heads, unsigned grid, cudaStream_t s) {
  if (heads == 16)
    launch<T, 16>(a, turn, grid, s);
  else
    launch<T, 32>(a, turn, grid, s);
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_latent_store(const void *latent, int64_t latent_stride_n, const void *k_rope,
                                   int64_t k_rope_stride_n, const void *q_rope, int64_t q_stride_n, int64_t q_stride_h,
                                   void *q_out, int32_t dtype, const void *norm_weight, float eps, void *pool,
                                   const int64_t *slots, const float *table, int64_t max_pos, const int32_t *positions,
                                   int32_t interleaved, int64_t num_tokens, int64_t num_q_heads, int64_t num_blocks,
                                   int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(dtype == B200KV_F16 || dtype == B200KV_BF16, "dtype %d is not fp16 or bf16", dtype);
  B200KV_CHECK_ARG(num_tokens >= 0 && num_q_heads >= 0 && num_q_heads <= 65536 && num_blocks > 0 &&
                       num_blocks < (int64_t{1} << 40),
                   "num_tokens, num_q_heads or num_blocks out of range");
  const int per = num_q_heads <= 16 ? 16 : 32;  // heads of a warp
  const int64_t parts = 1 + (num_q_heads + per - 1) / per;
  B200KV_CHECK_ARG(num_tokens * parts < (int64_t{1} << 31), "num_tokens %lld out of range", (long long)num_tokens);
  B200KV_CHECK_ARG(!table || max_pos > 0, "max_pos must be > 0");
  B200KV_CHECK_ARG(table || num_q_heads == 0, "q_rope is only taken to be turned: a table is needed");
  B200KV_CHECK_ARG(!norm_weight || eps >= 0.f, "eps must be >= 0");
  if (num_tokens == 0) return B200KV_OK;
  B200KV_CHECK_ARG(latent && k_rope && pool && slots && (num_q_heads == 0 || (q_rope && q_out)), "null pointer argument");
  B200KV_CHECK_ARG(!table || positions, "a table needs positions");
  B200KV_CHECK_ARG(aligned_to(latent, 16) && aligned_to(k_rope, 16) && aligned_to(pool, 16) && aligned_to(q_rope, 16) &&
                       aligned_to(q_out, 16) && aligned_to(table, 16) && aligned_to(norm_weight, 16),
                   "buffers must be 16-byte aligned");
  const bool many = num_tokens > 1;  // (a dimension of one element may have any stride)
  B200KV_CHECK_ARG((!many || (latent_stride_n % 8 == 0 && k_rope_stride_n % 8 == 0)) &&
                       (num_q_heads == 0 || ((!many || q_stride_n % 8 == 0) && (num_q_heads == 1 || q_stride_h % 8 == 0))),
                   "row strides must be multiples of 8 elements");
  StoreArgs a{};
  a.latent = latent, a.latent_sn = latent_stride_n, a.k_rope = k_rope, a.rope_sn = k_rope_stride_n;
  a.q_rope = q_rope, a.q_sn = q_stride_n, a.q_sh = q_stride_h, a.q_out = q_out;
  a.weight = norm_weight, a.eps = eps, a.pool = pool, a.slots = slots;
  a.table = reinterpret_cast<const float2 *>(table), a.max_pos = max_pos, a.positions = positions;
  a.num_slots = num_blocks * kPageTokens;
  a.tokens = static_cast<int>(num_tokens), a.heads = static_cast<int>(num_q_heads), a.parts = static_cast<int>(parts);
  a.error_flag = error_flag;
  const unsigned grid = static_cast<unsigned>((num_tokens * parts + 7) / 8);
  const int turn = !table ? 0 : (interleaved ? 2 : 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B200KV_F16)
    launch<__half>(a, turn, per, grid, s);
  else
    launch<__nv_bfloat16>(a, turn, per, grid, s);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}
