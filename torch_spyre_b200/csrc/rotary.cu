// Rotary positions of head rows x [T, H, D] from an fp32 table of (cos, sin)
// pairs: for pair i of the first rotary_dim elements (elements i and
// i + rotary_dim / 2 in the half layout, 2i and 2i + 1 interleaved)
//   a' = a cos - b sin,   b' = b cos + a sin,
// computed in fp32 and rounded once; the other elements are copied.  The map is
// linear in x with the transpose "turn by -angle", which is its gradient.
//
// Bound by HBM: 2 * D * sizeof(T) bytes per row against 3 operations per
// element.  A thread owns one 16-byte vector position of a token (two, a pair's
// halves, in the half layout), keeps its cos / sin in registers and walks up to
// four heads with it, so the table's 8 bytes per pair are fetched once per four
// heads and not once per head.  8192 tokens of 40 heads, 128 elements of which 64
// are turned, bf16 (168 MB): 29 us interleaved, 0.91 of the copy rate, 32 in the
// half layout.
#include "rows.cuh"

namespace b200kv {
namespace {

struct RotaryArgs {
  const void *x;
  int64_t xs_t, xs_h;
  void *out;  // contiguous [T, H, D]
  const float2 *table;
  int64_t max_pos;
  const int32_t *positions;
  int64_t tokens;
  int heads, dim, half;  // half = rotary_dim / 2
  float sign;            // +1, or -1 for the transpose
  int32_t *error_flag;
  int items;   // vector positions of a row
  int groups;  // head groups of a token
  int tpb;     // tokens of a block
};

__device__ __forceinline__ int64_t checked_pos(const RotaryArgs &a, int64_t t, bool report) {
  int64_t pos = __ldg(a.positions + t);
  if (pos < 0 || pos >= a.max_pos) {
    if (report && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
    pos = pos < 0 ? 0 : a.max_pos - 1;
  }
  return pos;
}

template <typename T>
struct Vec;  // kN elements of a 16-byte vector as fp32
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void load(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 store(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <typename T>
struct Vec {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void load(uint4 v, float (&f)[8]) { unpack8(v, f, T()); }
  static __device__ __forceinline__ uint4 store(const float (&f)[8]) { return pack8(f, T()); }
};

// kHeads heads per thread.  Half layout: item c < half / kN is the pair of
// vectors at c * kN and half + c * kN, a later item two copied neighbours.
// Interleaved: every item is one vector, its pairs before rotary_dim turned.
template <typename T, bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  constexpr int kN = Vec<T>::kN;
  constexpr int kPairs = kInterleaved ? kN / 2 : kN;
  const int per = a.groups * a.items;
  const int local = threadIdx.x;
  const int tl = local / per, r = local - tl * per;
  const int64_t t = int64_t(blockIdx.x) * a.tpb + tl;
  if (tl >= a.tpb || t >= a.tokens) return;
  // gridDim.y blocks share a token whose items do not fit one block
  const int unit = r + blockIdx.y * blockDim.x;
  if (unit >= per) return;
  const int g = unit / a.items, c = unit - g * a.items;
  const int h0 = g * kHeads;
  const T *x = static_cast<const T *>(a.x) + t * a.xs_t;
  T *out = static_cast<T *>(a.out) + t * a.heads * a.dim;
  const int pair_items = kInterleaved ? 0 : a.half / kN;
  const bool pair = !kInterleaved && c < pair_items;
  const int e = kInterleaved || pair ? c * kN : 2 * a.half + (c - pair_items) * 2 * kN;
  const int beside = pair ? a.half : kN;
  const bool second = pair || (!kInterleaved && e + kN < a.dim);
  const bool turn = kInterleaved ? e < 2 * a.half : pair;

  uint4 va[kHeads], vb[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (h0 + i < a.heads) {
      va[i] = __ldg(reinterpret_cast<const uint4 *>(x + (h0 + i) * a.xs_h + e));
      if (second) vb[i] = __ldg(reinterpret_cast<const uint4 *>(x + (h0 + i) * a.xs_h + beside + e));
    }
  }
  float cosv[kPairs], sinv[kPairs];
  if (turn) {
    const float2 *row = a.table + checked_pos(a, t, unit == 0) * a.half;
    const int p0 = kInterleaved ? e / 2 : e;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      // past rotary_dim (a vector cut by its end): the identity
      const float2 cs = p0 + i < a.half ? __ldg(row + p0 + i) : make_float2(1.f, 0.f);
      cosv[i] = cs.x;
      sinv[i] = a.sign * cs.y;
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (h0 + i >= a.heads) continue;
    T *o = out + (h0 + i) * a.dim + e;
    if (turn) {
      float f[kN];
      Vec<T>::load(va[i], f);
      if (kInterleaved) {
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
          // a pair past rotary_dim is copied, not multiplied (inf * 0 is NaN)
          if (e / 2 + j < a.half) turn_pair(f[2 * j], f[2 * j + 1], cosv[j], sinv[j], f[2 * j], f[2 * j + 1]);
        }
      } else {
        float s[kN];
        Vec<T>::load(vb[i], s);
#pragma unroll
        for (int j = 0; j < kN; ++j) turn_pair(f[j], s[j], cosv[j], sinv[j], f[j], s[j]);
        __stcs(reinterpret_cast<uint4 *>(o + a.half), Vec<T>::store(s));
      }
      __stcs(reinterpret_cast<uint4 *>(o), Vec<T>::store(f));
    } else {
      __stcs(reinterpret_cast<uint4 *>(o), va[i]);
      if (second) __stcs(reinterpret_cast<uint4 *>(o + beside), vb[i]);
    }
  }
}

// Rows whose pairs or strides do not fall on 16-byte vectors: one thread per
// pair or copied element.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(256) rotary_scalar_kernel(const RotaryArgs a) {
  const int64_t total = a.tokens * a.heads * a.items;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int c = static_cast<int>(i % a.items);
    const int64_t th = i / a.items;
    const int h = static_cast<int>(th % a.heads);
    const int64_t t = th / a.heads;
    const T *x = static_cast<const T *>(a.x) + t * a.xs_t + h * a.xs_h;
    T *out = static_cast<T *>(a.out) + th * a.dim;
    if (c >= a.half) {
      out[a.half + c] = x[a.half + c];
      continue;
    }
    const float2 cs = __ldg(a.table + checked_pos(a, t, c == 0 && h == 0) * a.half + c);
    const int ea = kInterleaved ? 2 * c : c, eb = kInterleaved ? 2 * c + 1 : c + a.half;
    float ra, rb;
    turn_pair(to_float(x[ea]), to_float(x[eb]), cs.x, a.sign * cs.y, ra, rb);
    from_float(out[ea], ra);
    from_float(out[eb], rb);
  }
}

template <typename T, bool kInterleaved>
int launch_rotary(RotaryArgs a, cudaStream_t stream) {
  constexpr int kN = Vec<T>::kN;
  int dev = 0, sms = 0;
  int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  const bool vec = aligned_to(a.x, 16) && aligned_to(a.out, 16) && a.xs_t % kN == 0 && a.xs_h % kN == 0 &&
                   a.dim % kN == 0 && (kInterleaved || a.half % kN == 0);
  if (!vec) {
    a.items = a.dim - a.half;
    const int64_t want = (a.tokens * a.heads * a.items + 255) / 256;
    const int64_t cap = int64_t(sms) * 8;
    rotary_scalar_kernel<T, kInterleaved><<<static_cast<unsigned>(want < cap ? want : cap), 256, 0, stream>>>(a);
    B200KV_CUDA_TRY(cudaGetLastError());
    return B200KV_OK;
  }
  a.items = kInterleaved ? a.dim / kN : a.half / kN + ((a.dim - 2 * a.half) / kN + 1) / 2;
  // Four heads per thread once that still leaves every SM its 2048 threads;
  // below, one head per thread: with few rows the latency of one load counts.
  const bool deep = a.tokens * a.heads * a.items >= int64_t(sms) * 2048 * 4;
  const int hpt = deep ? 4 : 1;
  a.groups = (a.heads + hpt - 1) / hpt;
  const int64_t per = int64_t(a.groups) * a.items;
  const int64_t kBlock = 256;
  a.tpb = static_cast<int>(per >= kBlock ? 1 : kBlock / per);
  const int64_t used = a.tpb * per;
  const unsigned block = static_cast<unsigned>(used >= kBlock ? kBlock : (used + 31) / 32 * 32);
  const dim3 grid(static_cast<unsigned>((a.tokens + a.tpb - 1) / a.tpb),
                  static_cast<unsigned>(a.tpb > 1 ? 1 : (per + block - 1) / block));
  if (deep)
    rotary_kernel<T, kInterleaved, 4><<<grid, block, 0, stream>>>(a);
  else
    rotary_kernel<T, kInterleaved, 1><<<grid, block, 0, stream>>>(a);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_rotary(const void *x, int32_t dtype, int64_t x_stride_t, int64_t x_stride_h, void *out,
                             const float *table, int64_t max_pos, int64_t rotary_dim, const int32_t *positions,
                             int64_t num_tokens, int64_t num_heads, int64_t head_dim, int32_t interleaved,
                             int32_t transpose, int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(dtype == B200KV_F16 || dtype == B200KV_BF16 || dtype == B200KV_F32, "dtype %d is not fp16, bf16 or fp32",
                   dtype);
  B200KV_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t{1} << 31), "num_tokens %lld out of range",
                   (long long)num_tokens);
  B200KV_CHECK_ARG(num_heads >= 0 && num_heads <= 65536, "num_heads %lld out of range", (long long)num_heads);
  B200KV_CHECK_ARG(head_dim > 0 && head_dim <= 4096, "head_dim %lld out of range", (long long)head_dim);
  B200KV_CHECK_ARG(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
                   "rotary_dim (%lld) must be even and in (0, head_dim = %lld]", (long long)rotary_dim,
                   (long long)head_dim);
  B200KV_CHECK_ARG(max_pos > 0, "max_pos must be > 0");
  if (num_tokens == 0 || num_heads == 0) return B200KV_OK;
  B200KV_CHECK_ARG(x && out && table && positions, "null pointer argument");
  B200KV_CHECK_ARG(aligned_to(table, 8), "table must be 8-byte aligned");
  RotaryArgs a{};
  a.x = x;
  a.xs_t = x_stride_t;
  a.xs_h = x_stride_h;
  a.out = out;
  a.table = reinterpret_cast<const float2 *>(table);
  a.max_pos = max_pos;
  a.positions = positions;
  a.tokens = num_tokens;
  a.heads = static_cast<int>(num_heads);
  a.dim = static_cast<int>(head_dim);
  a.half = static_cast<int>(rotary_dim / 2);
  a.sign = transpose ? -1.f : 1.f;
  a.error_flag = error_flag;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200KV_F16: return interleaved ? launch_rotary<__half, true>(a, s) : launch_rotary<__half, false>(a, s);
    case B200KV_BF16:
      return interleaved ? launch_rotary<__nv_bfloat16, true>(a, s) : launch_rotary<__nv_bfloat16, false>(a, s);
    default: return interleaved ? launch_rotary<float, true>(a, s) : launch_rotary<float, false>(a, s);
  }
}
