// K/V rows into and out of the paged stick cache, with one scale per row for
// 8-bit pools:
//   store   k is turned by its rotary position (optional, q beside it), then
//           s = max |x| / qmax, q = round(x * (1 / s)) clamped to +-qmax and
//           written to the row's slot, s beside it (16-bit pools: rounded once);
//   load    rows gathered by slot, q * s rounded once;
//   commit  the accepted path of a drafted tree moved to the end of the
//           committed tokens, bytes and scales as they are.
// All three are bound by HBM (or, for a few rows, by a chain of 2-3 dependent
// loads): one pass over the rows, 16-byte vectors, K and V in one launch.
#include "rows.cuh"

namespace b200kv {
namespace {

constexpr float kQMaxInt8 = 127.f, kQMaxE4M3 = 448.f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ------------------------------------------------------------------ store --
struct StoreArgs {
  const void *q, *k, *v;
  int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh;
  void *q_out;  // contiguous [N, Hq, D]
  void *k_pool, *v_pool;
  float *k_scales, *v_scales;
  const int64_t *slots;
  const float2 *table;
  int64_t max_pos;
  const int32_t *positions;
  int64_t tokens, num_slots;
  int hq, hkv, half;
  int32_t *error_flag;
};

// Eight fp32 -> eight 8-bit steps of 1 / inv.  fp32 arithmetic, each operation
// rounded by itself, so the same steps as x * (1 / s) computed anywhere else.
// |x * inv| exceeds qmax by a few 2^-24 at most (inv and s are rounded), which
// rounds to qmax: no clamp is needed.
__device__ __forceinline__ uint2 steps8_int8(const float (&f)[8], float inv) {
  // 1.5 * 2^23 + x: the nearest integer (ties to even) is in the low byte
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[i], inv), 12582912.f));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __byte_perm(b[2 * i], b[2 * i + 1], 0x0040);
  return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}
__device__ __forceinline__ uint2 steps8_e4m3(const float (&f)[8], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(f[2 * i], inv), __fmul_rn(f[2 * i + 1], inv)), __NV_SATFINITE,
                                    __NV_E4M3);
  return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}

// A group of lanes takes one row, kRows rows of a token and kind (q, K or V
// heads) one after the other, the cos / sin of its elements in registers.  A
// lane has one 16-byte vector, or in the half layout two: a vector and the one
// that holds its pairs' other elements (rotary_dim / 2 is a multiple of 8), or
// two neighbours past rotary_dim.
// kCache: B200KV_F16 (= the row type), B200KV_I8 or B200KV_E4M3.
//
// Bound: bytes, and the instructions of the conversions right behind them.  16381
// tokens of 32 + 16 heads, 128 elements of which 96 are turned, bf16 into e4m3
// (369 MB): 73 us, 0.78 of the copy rate, and 101 with two readings back; into
// bf16 100, in the half layout 102 (into int8 105).  Rows and blocks per SM, us
// with the readings: interleaved four and five 101, eight and five 121; half
// layout two and four 105, two and three 114, four and three 100, four and two
// 112.  A lane of the half layout with one vector, its partner's by shuffle: 127.
template <typename T, int D, int kCache, int kTurn, int kRows>  // kTurn 0 none, 1 half, 2 interleaved
__global__ void __launch_bounds__(256, kRows > 1 ? (kTurn == 1 ? 3 : 5) : 1) kv_store_kernel(const StoreArgs a) {
  constexpr int kVecs = kTurn == 1 ? 2 : 1, kLanes = D / 8 / kVecs;
  constexpr int kStick = kCache == B200KV_F16 ? 64 : 128;
  const int lane = threadIdx.x % kLanes;
  const bool paired = kTurn == 1 && lane < a.half / 8;
  const int e = kTurn == 1 && !paired ? 16 * lane : 8 * lane;  // the first vector's elements
  const int beside = paired ? a.half : 8;                      // from the first vector to the second
  const uint32_t of_q = (a.hq + kRows - 1) / kRows, of_kv = (a.hkv + kRows - 1) / kRows;  // units of a kind
  const uint32_t unit = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const uint32_t t32 = unit / (of_q + 2 * of_kv);
  uint32_t u = unit - t32 * (of_q + 2 * of_kv);
  const int kind = u < of_q ? 0 : (u < of_q + of_kv ? 1 : 2);  // q, K, V
  u -= kind == 0 ? 0 : (kind == 1 ? of_q : of_q + of_kv);
  const int h0 = static_cast<int>(u) * kRows;
  const int64_t t = t32;
  const bool live_t = t < a.tokens;  // dead lanes stay for the shuffles
  const int rows = live_t ? min(kRows, (kind == 0 ? a.hq : a.hkv) - h0) : 0;

  uint4 raw[kRows][kVecs];
  {
    const int64_t sn = kind == 0 ? a.q_sn : (kind == 1 ? a.k_sn : a.v_sn);
    const int64_t sh = kind == 0 ? a.q_sh : (kind == 1 ? a.k_sh : a.v_sh);
    const T *src = static_cast<const T *>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v)) + t * sn + h0 * sh + e;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int x = 0; x < kVecs; ++x)
        if (i < rows) raw[i][x] = __ldg(reinterpret_cast<const uint4 *>(src + i * sh + x * beside));
  }
  int64_t slot = -1;
  if (rows > 0 && kind > 0) {
    slot = __ldg(a.slots + t);
    if (slot >= a.num_slots) {
      if (a.error_flag && lane == 0) atomicOr(a.error_flag, B200KV_DEVERR_BAD_SLOT);
      slot = -1;
    }
  }
  // cos / sin of this lane's pairs: 8 in the half layout, 4 interleaved
  constexpr int kPairs = kTurn == 2 ? 4 : 8;
  float cosv[kPairs], sinv[kPairs];
  const bool turned = rows > 0 && kind < 2 && (kTurn == 1 ? paired : kTurn == 2 && e < 2 * a.half);
  const bool whole = kTurn == 1 || e / 2 + 4 <= a.half;  // no pair past rotary_dim
  if (turned) {
    int64_t pos = __ldg(a.positions + t);
    if (pos < 0 || pos >= a.max_pos) {
      if (a.error_flag && lane == 0) atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
      pos = pos < 0 ? 0 : a.max_pos - 1;
    }
    const float2 *row = a.table + pos * a.half + (kTurn == 2 ? e / 2 : e);
    if (kTurn == 1 || (a.half % 2 == 0 && whole)) {  // 16-byte aligned, all inside
#pragma unroll
      for (int i = 0; i < kPairs; i += 2) {
        const float4 cs = __ldg(reinterpret_cast<const float4 *>(row + i));
        cosv[i] = cs.x, sinv[i] = cs.y, cosv[i + 1] = cs.z, sinv[i + 1] = cs.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        // an interleaved vector cut by rotary_dim: nothing past it is used
        const float2 cs = e / 2 + i < a.half ? __ldg(row + i) : make_float2(1.f, 0.f);
        cosv[i] = cs.x;
        sinv[i] = cs.y;
      }
    }
  }
  // of the first row; the next head's is D elements (q) or a page on
  T *q_out = static_cast<T *>(a.q_out) + (t * a.hq + h0) * D + e;
  const int64_t page = (slot >> 6) * a.hkv + h0;
  const int in_page = static_cast<int>(slot & 63);
  const int64_t at = page * (64 * D) + in_page * kStick;
  int in_row[kVecs];  // a vector's place in the pool, from its row's
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    const int ex = e + x * beside;
    in_row[x] = ex / kStick * (64 * kStick) + ex % kStick;
  }
  void *pool = kind == 1 ? a.k_pool : a.v_pool;
  float *scale = (kind == 1 ? a.k_scales : a.v_scales) + page * 64 + in_page;
  // (units of two kinds can meet in a warp: it skips what none of them needs)
  const bool any_stored = __any_sync(0xffffffffu, rows > 0 && kind > 0);

#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const bool live = i < rows;
    float f[kVecs][8];
    if (live) {
#pragma unroll
      for (int x = 0; x < kVecs; ++x) unpack8(raw[i][x], f[x], T());
      if (kTurn == 1 && turned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) turn_pair(f[0][j], f[kVecs - 1][j], cosv[j], sinv[j], f[0][j], f[kVecs - 1][j]);
      } else if (kTurn == 2 && turned) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (whole || e / 2 + j < a.half)
            turn_pair(f[0][2 * j], f[0][2 * j + 1], cosv[j], sinv[j], f[0][2 * j], f[0][2 * j + 1]);
      }
    }
    if (live && kind == 0) {
#pragma unroll
      for (int x = 0; x < kVecs; ++x) *reinterpret_cast<uint4 *>(q_out + i * D + x * beside) = pack8(f[x], T());
    }
    if (!any_stored) continue;
    const bool write = live && kind > 0 && slot >= 0;
    if (kCache == B200KV_F16) {
#pragma unroll
      for (int x = 0; x < kVecs; ++x)
        if (write) *reinterpret_cast<uint4 *>(static_cast<T *>(pool) + at + in_row[x] + i * (64 * D)) = pack8(f[x], T());
    } else {
      float amax = 0.f;
      if (live) {
#pragma unroll
        for (int x = 0; x < kVecs; ++x)
#pragma unroll
          for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(f[x][j]));
      }
#pragma unroll
      for (int m = kLanes / 2; m >= 1; m >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, m, kLanes));
      if (write) {
        // a row without a normal scale (all zeros, or subnormal steps) is stored
        // as zeros; a row that holds NaN or inf reads back as NaN throughout
        float s = __fdiv_rn(amax, kCache == B200KV_I8 ? kQMaxInt8 : kQMaxE4M3);
        if (s < 1.17549435e-38f) s = 0.f;
        const bool finite = s < CUDART_INF_F;
        const float inv = s > 0.f && finite ? __fdiv_rn(1.f, s) : 0.f;
#pragma unroll
        for (int x = 0; x < kVecs; ++x) {
          const uint2 w = !finite ? make_uint2(0, 0)
                          : kCache == B200KV_I8 ? steps8_int8(f[x], inv) : steps8_e4m3(f[x], inv);
          *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(pool) + at + in_row[x] + i * (64 * D)) = w;
        }
        if (lane == 0) scale[i * 64] = finite ? s : CUDART_NAN_F;
      }
    }
  }
}

template <typename T, int D, int kCache, int kTurn>
int launch_store(const StoreArgs &a, cudaStream_t stream) {
  int dev = 0, sms = 0;
  int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  constexpr int kVecs = kTurn == 1 ? 2 : 1, kLanes = D / 8 / kVecs;
  // Four rows per lane group once every SM still gets its 2048 threads; with
  // fewer rows one each, as the latency of the loads counts.
  constexpr int kDeep = 4;
  const int heads = a.hq + 2 * a.hkv;
  const bool deep = a.tokens * heads * (D / 8) >= int64_t(sms) * 2048 * 4;
  const int64_t units = a.tokens * (deep ? (a.hq + kDeep - 1) / kDeep + 2 * ((a.hkv + kDeep - 1) / kDeep) : heads);
  const int64_t blocks = (units * kLanes + 255) / 256;
  if (units >= (int64_t{1} << 31))  // the kernel counts them in 32 bits
    return set_error(B200KV_ERR_UNSUPPORTED, "%lld tokens of %d heads: 2^31 rows or more", (long long)a.tokens, heads);
  if (deep)
    kv_store_kernel<T, D, kCache, kTurn, kDeep><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  else
    kv_store_kernel<T, D, kCache, kTurn, 1><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}
template <typename T, int D, int kCache>
int store_turn(const StoreArgs &a, int turn, cudaStream_t s) {
  return turn == 0 ? launch_store<T, D, kCache, 0>(a, s)
                   : turn == 1 ? launch_store<T, D, kCache, 1>(a, s) : launch_store<T, D, kCache, 2>(a, s);
}
template <typename T>
int store_cache(const StoreArgs &a, int64_t dim, int cache, int turn, cudaStream_t s) {
  if (cache == B200KV_I8) return store_turn<T, 128, B200KV_I8>(a, turn, s);
  if (cache == B200KV_E4M3) return store_turn<T, 128, B200KV_E4M3>(a, turn, s);
  return dim == 64 ? store_turn<T, 64, B200KV_F16>(a, turn, s) : store_turn<T, 128, B200KV_F16>(a, turn, s);
}

// ------------------------------------------------------------------- load --
struct LoadArgs {
  const void *pool;
  const float *scales;
  const int64_t *slots;
  void *out;  // contiguous [N, Hkv, D]
  int64_t num_slots;
  uint32_t rows, hkv;
  int32_t *error_flag;
};

// A thread makes 16 bytes of output (kElems elements) of kUnroll rows; the
// kChunks threads of a row are neighbours, so reads and writes are whole lines.
// All kUnroll slots, then all rows and scales, are in flight together.  Row
// numbers are 32-bit (the host checks): a 64-bit division per row cost as much
// as the row's memory traffic.  131072 tokens of 8 heads, e4m3 to bf16 (408 MB):
// 70 us, 0.91 of the copy rate; int8 67.
template <int kCache, typename TIn, typename TOut, int D, int kUnroll>
__global__ void __launch_bounds__(256) kv_load_kernel(const LoadArgs a) {
  constexpr bool k8 = kCache != B200KV_F16;
  constexpr int kElems = 16 / sizeof(TOut);
  constexpr int kStick = k8 ? 128 : 64;
  constexpr int kChunks = D / kElems;
  constexpr int kRows = 256 / kChunks;
  const int e = static_cast<int>(threadIdx.x % kChunks) * kElems;
  const uint32_t row0 = blockIdx.x * (kRows * kUnroll) + threadIdx.x / kChunks;
  int64_t slot[kUnroll];
  uint32_t head[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t row = row0 + u * kRows;
    slot[u] = -1;
    if (row < a.rows) {
      const uint32_t n = row / a.hkv;
      head[u] = row - n * a.hkv;
      slot[u] = __ldg(a.slots + n);
    }
  }
  uint32_t w[kUnroll][4];
  float sc[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0;  // padding, and past the pool: a row of zeros
    sc[u] = 0.f;
    if (slot[u] < 0) continue;
    if (slot[u] >= a.num_slots) {
      if (a.error_flag && e == 0 && head[u] == 0) atomicOr(a.error_flag, B200KV_DEVERR_BAD_SLOT);
      continue;
    }
    const int64_t page = (slot[u] >> 6) * a.hkv + head[u];
    const int in_page = static_cast<int>(slot[u] & 63);
    const TIn *src = static_cast<const TIn *>(a.pool) +
                     (page * (D / kStick) + e / kStick) * (64 * kStick) + int64_t(in_page) * kStick + e % kStick;
    if constexpr (kElems * sizeof(TIn) == 16) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(src));
      w[u][0] = v.x, w[u][1] = v.y, w[u][2] = v.z, w[u][3] = v.w;
    } else if constexpr (kElems * sizeof(TIn) == 8) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(src));
      w[u][0] = v.x, w[u][1] = v.y;
    } else {
      w[u][0] = __ldcs(reinterpret_cast<const uint32_t *>(src));
    }
    if (k8) sc[u] = __ldg(a.scales + page * 64 + in_page);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t row = row0 + u * kRows;
    if (row >= a.rows) continue;
    TOut o[kElems];
#pragma unroll
    for (int j = 0; j < kElems; ++j) {
      if constexpr (kCache == B200KV_I8) {
        from_float(o[j], __fmul_rn(static_cast<float>(static_cast<int8_t>(w[u][j >> 2] >> (8 * (j & 3)))), sc[u]));
      } else if constexpr (kCache == B200KV_E4M3) {
        const __nv_fp8_storage_t b = static_cast<__nv_fp8_storage_t>(w[u][j >> 2] >> (8 * (j & 3)));
        from_float(o[j], __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3))), sc[u]));
      } else {
        const uint16_t b = static_cast<uint16_t>(w[u][j >> 1] >> (16 * (j & 1)));
        from_float(o[j], to_float(*reinterpret_cast<const TIn *>(&b)));
      }
    }
    __stcs(reinterpret_cast<uint4 *>(static_cast<TOut *>(a.out) + int64_t(row) * D + e), *reinterpret_cast<uint4 *>(o));
  }
}

template <int kCache, typename TIn, typename TOut, int D>
int launch_load(const LoadArgs &a, cudaStream_t stream) {
  int dev = 0, sms = 0;
  int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  constexpr int kRows = 256 / (D / (16 / static_cast<int>(sizeof(TOut))));
  // Eight rows per thread once every SM still gets its 2048 threads, else one.
  const bool deep = a.rows >= static_cast<uint32_t>(sms) * 8 * kRows * 8;
  const unsigned per = kRows * (deep ? 8 : 1);
  const unsigned grid = (a.rows + per - 1) / per;
  if (deep)
    kv_load_kernel<kCache, TIn, TOut, D, 8><<<grid, 256, 0, stream>>>(a);
  else
    kv_load_kernel<kCache, TIn, TOut, D, 1><<<grid, 256, 0, stream>>>(a);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}
template <int kCache, typename TIn, int D>
int load_out(const LoadArgs &a, int dtype, cudaStream_t s) {
  switch (dtype) {
    case B200KV_F16: return launch_load<kCache, TIn, __half, D>(a, s);
    case B200KV_BF16: return launch_load<kCache, TIn, __nv_bfloat16, D>(a, s);
    default: return launch_load<kCache, TIn, float, D>(a, s);
  }
}

// ----------------------------------------------------------------- commit --
struct CommitArgs {
  void *pool[2];
  float *scales[2];
  const int32_t *block_table;
  int64_t bt_stride;
  const int32_t *ctx, *path, *path_lens;
  int64_t path_stride;
  int32_t *new_lens;
  int hkv, max_blocks, max_path;
  int64_t num_blocks;
  int32_t *error_flag;
};

constexpr int kCommitThreads = 128, kCommitRows = 64;

// One CTA per sequence and KV head, K and V one after the other.  The path is
// taken 64 rows at a time: thread i finds where row i comes from and goes to, and
// moves its scale; then the rows move, 16 bytes per thread.  A batch is read
// whole before any of it is written; path[i] >= i (checked), so a later batch
// never reads what an earlier one wrote.
//
// Bound: bytes, each moved row read and written once; few rows: the chain length
// -> path -> block table -> row.  128 sequences, 8 KV heads, 32 rows each on
// average (33.6 MB): 7.5 us from HBM, 0.69 of the copy rate, and 6.2 where part of
// the rows is in L2.  There a CTA for K and one for V (every one walks that chain)
// took 9.7 us; four heads' CTAs in one 6.1, but 6.0 in place of 4.2 us for 4
// sequences.
template <int kRow, int kStickRow, bool kScaled>  // bytes of a row, of a row inside one stick (128)
__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(const CommitArgs a) {
  constexpr int kLanes = kRow / 16, kGroups = kCommitThreads / kLanes, kEach = kCommitRows / kGroups;
  constexpr int64_t kPage = 64 * kRow;
  __shared__ int64_t from[kCommitRows], to[kCommitRows];  // byte offsets of KV head 0's rows, to: -1 = stays
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
  const int cap = a.max_blocks * kPageTokens;
  const int ctx = __ldg(a.ctx + b);
  const int n_in = __ldg(a.path_lens + b);
  const bool bad = ctx < 0 || ctx > cap || n_in < 0 || n_in > a.max_path || ctx + n_in > cap;
  const int n = bad ? 0 : n_in;
  if (h == 0 && tid == 0) {
    if (bad && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
    a.new_lens[b] = bad ? ctx : ctx + n;
  }
  const int32_t *path = a.path + b * a.path_stride;
  const int32_t *table = a.block_table + b * a.bt_stride;
  auto offset = [&](int tok, bool inside) -> int64_t {  // -1 (flagged) outside
    if (!inside) {
      if (a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_SLOT);
      return -1;
    }
    const int blk = __ldg(table + (tok >> 6));
    if (blk < 0 || blk >= a.num_blocks) {
      if (a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_BLOCK);
      return -1;
    }
    return int64_t(blk) * a.hkv * kPage + (tok & 63) * kStickRow;
  };
  const int byte = (tid % kLanes) * 16, group = tid / kLanes;
  const int64_t part = h * kPage + byte / kStickRow * (64 * kStickRow) + byte % kStickRow;
  auto scale_at = [&](int64_t off) { return off / kPage * 64 + off % kPage / kStickRow + h * 64; };
  for (int base = 0; base < n; base += kCommitRows) {
    int64_t src = -1, dst = -1;
    if (tid < kCommitRows) {
      const int i = base + tid;
      if (i < n) {
        const int p = __ldg(path + i), before = i > 0 ? __ldg(path + i - 1) : -1;
        // (p < i: not ascending from 0 on, and so neither is any negative entry;
        // its row may have been overwritten already)
        if (p <= before || p < i) {  // the row stays where it is
          if (a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_SLOT);
        } else if (p != i) {
          src = offset(ctx + p, p < cap - ctx);
          dst = offset(ctx + i, true);
          if (src < 0) dst = -1;
        }
      }
      from[tid] = src;
      to[tid] = dst;
    }
    __syncthreads();
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint8_t *pool = static_cast<uint8_t *>(a.pool[kv]) + part;
      uint4 v[kEach];
      int64_t at[kEach];
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int r = u * kGroups + group;
        at[u] = to[r];
        if (at[u] >= 0) v[u] = *reinterpret_cast<const uint4 *>(pool + from[r]);
      }
      float s = 0.f;
      const bool scaled = kScaled && dst >= 0;
      if (scaled) s = a.scales[kv][scale_at(src)];
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kEach; ++u)
        if (at[u] >= 0) *reinterpret_cast<uint4 *>(pool + at[u]) = v[u];
      if (scaled) a.scales[kv][scale_at(dst)] = s;
    }
    __syncthreads();
  }
}

int check_cache(int32_t dtype, int64_t head_dim, const char *what) {
  const bool k8 = dtype == B200KV_I8 || dtype == B200KV_E4M3;
  if (!k8 && dtype != B200KV_F16 && dtype != B200KV_BF16)
    return set_error(B200KV_ERR_INVALID_ARG, "%s dtype %d is not fp16, bf16, int8 or e4m3", what, dtype);
  if (head_dim != 128 && !(head_dim == 64 && !k8))
    return set_error(B200KV_ERR_UNSUPPORTED, "head_dim %lld unsupported (128, or 64 in 16-bit pools)",
                     (long long)head_dim);
  return B200KV_OK;
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_kv_store(const void *q, int64_t q_stride_n, int64_t q_stride_h, void *q_out, const void *k,
                               int64_t k_stride_n, int64_t k_stride_h, const void *v, int64_t v_stride_n,
                               int64_t v_stride_h, int32_t row_dtype, void *k_pool, void *v_pool, int32_t pool_dtype,
                               float *k_scales, float *v_scales, const int64_t *slots, const float *table,
                               int64_t max_pos, int64_t rotary_dim, const int32_t *positions, int32_t interleaved,
                               int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                               int64_t num_blocks, int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(row_dtype == B200KV_F16 || row_dtype == B200KV_BF16, "row dtype %d is not fp16 or bf16", row_dtype);
  int st = check_cache(pool_dtype, head_dim, "pool");
  if (st != B200KV_OK) return st;
  const bool k8 = pool_dtype == B200KV_I8 || pool_dtype == B200KV_E4M3;
  B200KV_CHECK_ARG(k8 || pool_dtype == row_dtype, "a 16-bit pool must have the rows' dtype");
  B200KV_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t{1} << 31), "num_tokens %lld out of range", (long long)num_tokens);
  B200KV_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 65536 && num_q_heads >= 0 && num_q_heads <= 65536 &&
                       num_blocks > 0 && num_blocks < (int64_t{1} << 40),
                   "head counts or num_blocks out of range");
  if (table) {
    B200KV_CHECK_ARG(max_pos > 0, "max_pos must be > 0");
    B200KV_CHECK_ARG(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
                     "rotary_dim (%lld) must be even and in (0, head_dim]", (long long)rotary_dim);
    if (!interleaved && rotary_dim % 16 != 0)
      return set_error(B200KV_ERR_UNSUPPORTED, "rotary_dim %lld unsupported in the half layout (multiples of 16)",
                       (long long)rotary_dim);
  } else {
    B200KV_CHECK_ARG(num_q_heads == 0, "q is only taken to be turned: a table is needed");
  }
  if (num_tokens == 0) return B200KV_OK;
  B200KV_CHECK_ARG(k && v && k_pool && v_pool && slots, "null pointer argument");
  B200KV_CHECK_ARG(num_q_heads == 0 || (q && q_out), "null q or q_out");
  B200KV_CHECK_ARG(!k8 || (k_scales && v_scales), "8-bit pools need k_scales and v_scales");
  B200KV_CHECK_ARG(!table || positions, "a table needs positions");
  B200KV_CHECK_ARG(aligned_to(k, 16) && aligned_to(v, 16) && aligned_to(k_pool, 16) && aligned_to(v_pool, 16) &&
                       (num_q_heads == 0 || (aligned_to(q, 16) && aligned_to(q_out, 16))) && aligned_to(table, 16),
                   "buffers must be 16-byte aligned");
  // (a dimension of one element may have any stride)
  const bool many = num_tokens > 1;
  B200KV_CHECK_ARG((!many || (k_stride_n % 8 == 0 && v_stride_n % 8 == 0)) &&
                       (num_kv_heads == 1 || (k_stride_h % 8 == 0 && v_stride_h % 8 == 0)) &&
                       (num_q_heads == 0 || ((!many || q_stride_n % 8 == 0) && (num_q_heads == 1 || q_stride_h % 8 == 0))),
                   "row strides must be multiples of 8 elements");
  StoreArgs a{};
  a.q = q, a.q_sn = q_stride_n, a.q_sh = q_stride_h, a.q_out = q_out;
  a.k = k, a.k_sn = k_stride_n, a.k_sh = k_stride_h;
  a.v = v, a.v_sn = v_stride_n, a.v_sh = v_stride_h;
  a.k_pool = k_pool, a.v_pool = v_pool, a.k_scales = k_scales, a.v_scales = v_scales;
  a.slots = slots;
  a.table = reinterpret_cast<const float2 *>(table);
  a.max_pos = max_pos;
  a.positions = positions;
  a.tokens = num_tokens;
  a.num_slots = num_blocks * kPageTokens;
  a.hq = static_cast<int>(num_q_heads);
  a.hkv = static_cast<int>(num_kv_heads);
  a.half = table ? static_cast<int>(rotary_dim / 2) : 0;
  a.error_flag = error_flag;
  const int turn = !table ? 0 : (interleaved ? 2 : 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return row_dtype == B200KV_F16 ? store_cache<__half>(a, head_dim, pool_dtype, turn, s)
                                 : store_cache<__nv_bfloat16>(a, head_dim, pool_dtype, turn, s);
}

extern "C" int b200kv_kv_load(const void *pool, int32_t pool_dtype, const float *scales, const int64_t *slots,
                              void *out, int32_t out_dtype, int64_t num_tokens, int64_t num_kv_heads,
                              int64_t head_dim, int64_t num_blocks, int32_t *error_flag, void *stream) {
  clear_error();
  int st = check_cache(pool_dtype, head_dim, "pool");
  if (st != B200KV_OK) return st;
  const bool k8 = pool_dtype == B200KV_I8 || pool_dtype == B200KV_E4M3;
  B200KV_CHECK_ARG(out_dtype == B200KV_F16 || out_dtype == B200KV_BF16 || out_dtype == B200KV_F32,
                   "out dtype %d is not fp16, bf16 or fp32", out_dtype);
  B200KV_CHECK_ARG(num_tokens >= 0, "num_tokens must be >= 0 (got %lld)", (long long)num_tokens);
  B200KV_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 65536 && num_blocks > 0 && num_blocks < (int64_t{1} << 40) &&
                       num_tokens < (int64_t{1} << 31),
                   "num_kv_heads, num_blocks or num_tokens out of range");
  if (num_tokens * num_kv_heads >= (int64_t{1} << 31))
    return set_error(B200KV_ERR_UNSUPPORTED, "%lld tokens of %lld heads: 2^31 rows or more", (long long)num_tokens,
                     (long long)num_kv_heads);
  if (num_tokens == 0) return B200KV_OK;
  B200KV_CHECK_ARG(pool && slots && out, "null pointer argument");
  B200KV_CHECK_ARG(!k8 || scales, "8-bit pools need their scales");
  B200KV_CHECK_ARG(aligned_to(pool, 16) && aligned_to(out, 16), "buffers must be 16-byte aligned");
  LoadArgs a{};
  a.pool = pool, a.scales = scales, a.slots = slots, a.out = out;
  a.num_slots = num_blocks * kPageTokens;
  a.rows = static_cast<uint32_t>(num_tokens * num_kv_heads);
  a.hkv = static_cast<uint32_t>(num_kv_heads);
  a.error_flag = error_flag;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (pool_dtype) {
    case B200KV_I8: return load_out<B200KV_I8, int8_t, 128>(a, out_dtype, s);
    case B200KV_E4M3: return load_out<B200KV_E4M3, uint8_t, 128>(a, out_dtype, s);
    case B200KV_F16:
      return head_dim == 64 ? load_out<B200KV_F16, __half, 64>(a, out_dtype, s)
                            : load_out<B200KV_F16, __half, 128>(a, out_dtype, s);
    default:
      return head_dim == 64 ? load_out<B200KV_F16, __nv_bfloat16, 64>(a, out_dtype, s)
                            : load_out<B200KV_F16, __nv_bfloat16, 128>(a, out_dtype, s);
  }
}

extern "C" int b200kv_tree_commit(void *k_pool, void *v_pool, int32_t pool_dtype, float *k_scales, float *v_scales,
                                  const int32_t *block_table, int64_t block_table_stride, const int32_t *context_lens,
                                  const int32_t *path, int64_t path_stride, const int32_t *path_lens,
                                  int32_t *new_lens, int64_t batch, int64_t num_kv_heads, int64_t head_dim,
                                  int64_t num_blocks, int64_t max_blocks_per_seq, int64_t max_path,
                                  int32_t *error_flag, void *stream) {
  clear_error();
  int st = check_cache(pool_dtype, head_dim, "pool");
  if (st != B200KV_OK) return st;
  const bool k8 = pool_dtype == B200KV_I8 || pool_dtype == B200KV_E4M3;
  B200KV_CHECK_ARG(batch >= 0 && batch <= 65535, "batch %lld out of range", (long long)batch);
  B200KV_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 65536 && num_blocks > 0 && num_blocks < (int64_t{1} << 40) &&
                       max_blocks_per_seq > 0 && max_blocks_per_seq * kPageTokens < (int64_t{1} << 30),
                   "num_kv_heads, num_blocks or max_blocks_per_seq out of range");
  B200KV_CHECK_ARG(block_table_stride >= max_blocks_per_seq, "block_table_stride < max_blocks_per_seq");
  B200KV_CHECK_ARG(max_path >= 0 && max_path < (int64_t{1} << 30) && (path_stride >= max_path || path_stride == 0),
                   "max_path out of range or path_stride < max_path");
  if (batch == 0) return B200KV_OK;
  B200KV_CHECK_ARG(k_pool && v_pool && block_table && context_lens && path_lens && new_lens && (path || max_path == 0),
                   "null pointer argument");
  B200KV_CHECK_ARG(!k8 || (k_scales && v_scales), "8-bit pools need k_scales and v_scales");
  B200KV_CHECK_ARG(aligned_to(k_pool, 16) && aligned_to(v_pool, 16), "pools must be 16-byte aligned");
  CommitArgs a{};
  a.pool[0] = k_pool, a.pool[1] = v_pool, a.scales[0] = k_scales, a.scales[1] = v_scales;
  a.block_table = block_table, a.bt_stride = block_table_stride;
  a.ctx = context_lens, a.path = path, a.path_stride = path_stride, a.path_lens = path_lens, a.new_lens = new_lens;
  a.hkv = static_cast<int>(num_kv_heads);
  a.max_blocks = static_cast<int>(max_blocks_per_seq);
  a.max_path = static_cast<int>(max_path);
  a.num_blocks = num_blocks;
  a.error_flag = error_flag;
  const dim3 grid(static_cast<unsigned>(num_kv_heads), static_cast<unsigned>(batch));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (k8)
    tree_commit_kernel<128, 128, true><<<grid, kCommitThreads, 0, s>>>(a);
  else if (head_dim == 64)
    tree_commit_kernel<128, 128, false><<<grid, kCommitThreads, 0, s>>>(a);
  else
    tree_commit_kernel<256, 128, false><<<grid, kCommitThreads, 0, s>>>(a);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}
