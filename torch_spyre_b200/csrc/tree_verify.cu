// Verification of drafted tokens against the target's probabilities.
//
// Node 0 of a sequence is its last token, the others are drafted; p = target row
// of a node, q = the drafter's, from which the node's children were drawn.  From
// node 0 on the children x_1, x_2, .. of the node reached are tried in order:
//   accept x_r  iff  w_r(x_r) > u_r S_r q(x_r),
//   w_1 = p, S_1 = 1;  after a rejection  w_{r+1} = max(p - c_r q, 0),
//   c_r = c_{r-1} + S_r (c_0 = 0),  S_{r+1} = sum w_{r+1},
// which is rejection sampling with the residual max(p_r - q, 0) / Z of
// p_r = w_r / S_r written without its normalisations: max(w_r - S_r q, 0) =
// max(p - (c_{r-1} + S_r) q, 0).  Without a drafter's row a rejected token is
// taken out of p: w = p without the rejected ones, S = 1 - sum of theirs, accept
// iff w(x) > u S.  Where nothing is accepted any more the next token is drawn
// from w: the first x with w(0) + .. + w(x) > u sum w.  Weights and sums are in
// 64 bits, since a whole token hangs on each comparison.
//
// The numbers that the comparisons take (a child's p and q) are fetched for all
// nodes at once, so the walk itself runs in shared memory; only a rejection and
// the final draw read a row, spread over a cluster of CTAs whose sums meet in
// distributed shared memory in rank order (the same bits every time).
//
// Bound: the bytes of a row of p and q per sequence (more where a tree's node
// rejects several children), or, for few sequences, latency.  128 chains of 4 over 131072
// elements, fp32: 43 us, 134 MB of rows in 23 of them (5.8 TB/s), the walk before and the
// exchange and the search behind take 7 and 8; 16 trees of up to 32 nodes over 32000: 20 us.
// Chains over bf16 rows: 33 us, without the drafter's rows 34 (fp32 37); trees over bf16 rows 25, without the
// drafter's 14.  (Four CTAs to an SM leave a thread 64 registers: with a drafter's rows 128 to 196
// bytes of its state are spilled around the sums.)
#include <cooperative_groups.h>

#include "rows.cuh"

namespace b200kv {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxCluster = 8, kMaxNodes = 1024;

struct VerifyArgs {
  const int32_t *parents;
  const int64_t *tokens;
  const int32_t *indptr;
  const void *target, *draft;
  int64_t target_stride, draft_stride;
  const float *accept_u, *sample_u;
  int32_t *path, *path_lens;
  int64_t *next;
  int total, batch, vocab, max_path;
  int vectors;  // rows may be read 16 bytes at a time
  int32_t *error_flag;
};

struct Shared {
  int parent[kMaxNodes], token[kMaxNodes], gone[kMaxNodes];  // gone: rejected tokens of the node reached
  float u[kMaxNodes], p[kMaxNodes], q[kMaxNodes];
  double warp_sum[kWarps], cta_sum[2][kMaxCluster];
  // what the CTA's warps do next: the sum over row `row` with c and the `gone` ones, the last one or not
  double c;
  int row, num_gone, last;
  int found;  // the thread that has the next token
  uint64_t landed[2];  // all CTAs' sums of a pass
};

// Weight of an element; what is not a positive number counts as 0.
template <bool kDraft>
__device__ __forceinline__ double weight(float p, float q, double c) {
  const double w = kDraft && c > 0.0 ? fma(-c, static_cast<double>(q), static_cast<double>(p)) : static_cast<double>(p);
  return w > 0.0 && w < CUDART_INF ? w : 0.0;
}

template <int kVec, typename T>
__device__ __forceinline__ void load_whole(const T *at, float (&f)[kVec]) {
  if constexpr (kVec == 1) {
    f[0] = to_float(*at);
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(at));
    if constexpr (kVec == 4) {
      f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
      f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    } else {
      unpack8(v, f, T());
    }
  }
}
// The same of a row's elements x .. x + kVec - 1, zeros past its end.
template <int kVec, typename T>
__device__ __forceinline__ void load_elements(const T *row, int x, int vocab, float (&f)[kVec]) {
  if (x + kVec <= vocab) {
    load_whole<kVec>(row + x, f);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = x + i < vocab ? to_float(row[x + i]) : 0.f;
  }
}

// The weights of elements x .. x + kVec - 1.
template <typename T, bool kDraft, int kVec>
__device__ __forceinline__ void weights(const VerifyArgs &a, const Shared &s, int row, double c, int gone, const float (&p)[kVec],
                                        const float (&q)[kVec], int x, double (&w)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) w[i] = weight<kDraft>(p[i], q[i], c);
  for (int g = 0; g < gone; ++g) {
    const int at = s.gone[g] - x;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (at == i) w[i] = 0.0;
  }
}

// A warp's part [x0, x1) of a row: contiguous, ascending with rank and warp.
template <int kVec>
__device__ __forceinline__ void part_of(int vocab, int ranks, int rank, int warp, int &x0, int &x1) {
  const int step = 32 * kVec, steps = (vocab + step - 1) / step;
  const int each = (steps + ranks * kWarps - 1) / (ranks * kWarps);
  const int64_t first = int64_t(rank * kWarps + warp) * each * step;
  x0 = static_cast<int>(min(first, int64_t(vocab)));
  x1 = static_cast<int>(min(first + int64_t(each) * step, int64_t(vocab)));
}

// This lane's share of the sum over [x0, x1).  kKind: 0 nothing rejected (c = 0), 1 one
// token rejected (c = 1), 2 anything.  The first two decide in fp32, where p > q is exact,
// which elements have a weight: 9 instructions an element where the third takes 30.
template <typename T, bool kDraft, int kVec, int kKind>
__device__ __forceinline__ double sum_lane(const VerifyArgs &a, const Shared &s, int row, double c, int gone, int x0, int x1) {
  const T *p = static_cast<const T *>(a.target) + row * a.target_stride;
  const T *q = kDraft ? static_cast<const T *>(a.draft) + row * a.draft_stride : p;
  constexpr int kAhead = kVec == 1 ? 8 : 16 / kVec, kStep = 32 * kVec;
  constexpr bool kQ = kDraft && kKind > 0;
  double sum = 0.0;
  auto add = [&](const float (&fp)[kVec], const float (&fq)[kVec], int x) {
    if constexpr (kKind == 2) {
      double w[kVec];
      weights<T, kDraft, kVec>(a, s, row, c, gone, fp, fq, x, w);
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum += w[i];
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const bool has = fp[i] < CUDART_INF_F && fp[i] > (kKind == 1 ? fq[i] : 0.f) && (kKind == 0 || fq[i] > -CUDART_INF_F);
        const double w = static_cast<double>(has ? fp[i] : 0.f);
        sum += kKind == 1 ? w - static_cast<double>(has ? fq[i] : 0.f) : w;
      }
    }
  };
  const int full = min(x1, a.vocab / kVec * kVec);  // vectors before this are whole
  int x = x0 + static_cast<int>(threadIdx.x & 31) * kVec, base = x0;
  for (; base + kAhead * kStep <= full; base += kAhead * kStep, x += kAhead * kStep) {
    float fp[kAhead][kVec], fq[kAhead][kVec];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      load_whole<kVec>(p + x + k * kStep, fp[k]);
      if (kQ) load_whole<kVec>(q + x + k * kStep, fq[k]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) add(fp[k], kQ ? fq[k] : fp[k], x + k * kStep);
  }
  for (; x < x1; x += kStep) {
    float fp[kVec], fq[kVec];
    load_elements<kVec>(p, x, a.vocab, fp);
    if (kQ) load_elements<kVec>(q, x, a.vocab, fq);
    add(fp, kQ ? fq : fp, x);
  }
  return sum;
}
template <typename T, bool kDraft, int kVec>
__device__ __noinline__ double sum_part(const VerifyArgs &a, const Shared &s, int row, double c, int gone, int x0, int x1) {
  double sum;
  if (gone == 0 && c == 0.0)
    sum = sum_lane<T, kDraft, kVec, 0>(a, s, row, c, gone, x0, x1);
  else if (kDraft && c == 1.0)
    sum = sum_lane<T, kDraft, kVec, 1>(a, s, row, c, gone, x0, x1);
  else
    sum = sum_lane<T, kDraft, kVec, 2>(a, s, row, c, gone, x0, x1);
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  return sum;
}

// The first element of [x0, x1), a warp's part, whose running sum is above t, or the last
// with a weight.  The whole CTA looks, a run of elements to a thread.  (One warp, 32
// vectors at a time behind one another: 32 steps of a load and a scan, half of the
// kernel's time at 131072 elements on 4 CTAs.)
template <typename T, bool kDraft, int kVec>
__device__ __noinline__ int find_in_part(const VerifyArgs &a, Shared &s, int row, double c, int gone, int x0, int x1, double t) {
  const T *p = static_cast<const T *>(a.target) + row * a.target_stride;
  const T *q = kDraft ? static_cast<const T *>(a.draft) + row * a.draft_stride : p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = ((x1 - x0 + kThreads - 1) / kThreads + kVec - 1) / kVec * kVec;
  const int first = min(x0 + tid * run, x1), end = min(first + run, x1);
  auto each = [&](auto use) {
    for (int x = first; x < end; x += kVec) {
      float fp[kVec], fq[kVec];
      load_elements<kVec>(p, x, a.vocab, fp);
      if (kDraft && c > 0.0) load_elements<kVec>(q, x, a.vocab, fq);
      double w[kVec];
      weights<T, kDraft, kVec>(a, s, row, c, gone, fp, kDraft ? fq : fp, x, w);
      if (!use(x, w)) return;
    }
  };
  double mine = 0.0;
  each([&](int, const double (&w)[kVec]) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) mine += w[i];
    return true;
  });
  double upto = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, m);
    if (lane >= m) upto += y;
  }
  if (tid == 0) s.found = kThreads, s.last = -1;
  __syncthreads();  // (warp_sum is read by all before this)
  if (lane == 31) s.warp_sum[warp] = upto;
  __syncthreads();
  double before = 0.0;
  for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
  if (mine > 0.0) {
    atomicMax(&s.last, tid);
    if (before + upto > t) atomicMin(&s.found, tid);
  }
  __syncthreads();
  if (tid != (s.found < kThreads ? s.found : s.last)) return -1;
  // (its sum may pass t without one of its elements doing so, by rounding: its last)
  int found = -1;
  double sum = before + (upto - mine);
  each([&](int x, const double (&w)[kVec]) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (!(w[i] > 0.0)) continue;
      sum += w[i];
      found = x + i;
      if (sum > t) return false;
    }
    return true;
  });
  return found;
}

// A sum to the same place of CTA `rank` of the cluster, whose barrier counts its bytes.  (A barrier
// of the whole cluster orders all memory, and takes 1500 clocks and more.)
__device__ __forceinline__ void send(const double *to, const uint64_t *bar, int rank, double x) {
  asm volatile(
      "{\n\t.reg .b32 d, b;\n\tmapa.shared::cluster.u32 d, %0, %2;\n\tmapa.shared::cluster.u32 b, %1, %2;\n\t"
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [d], %3, [b];\n\t}" ::"r"(smem_u32(to)),
      "r"(smem_u32(bar)), "r"(rank), "l"(__double_as_longlong(x))
      : "memory");
}

// Waits for a pass's sums, with a limit.
__device__ __forceinline__ bool landed(uint64_t *bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0 && global_timer_ns() - t0 > kWaitLimitNs) return false;
  }
}

// The next child of `node` after node i (n: none); the whole warp calls it.
__device__ __forceinline__ int next_child(const Shared &s, int node, int i, int n) {
  const int lane = threadIdx.x & 31;
  for (int base = (i + 1) & ~31; base < n; base += 32) {
    const int k = base + lane;
    const unsigned hit = __ballot_sync(0xffffffffu, k > i && k < n && s.parent[k] == node);
    if (hit) return base + __ffs(hit) - 1;
  }
  return n;
}

template <typename T, bool kDraft>
__global__ void __launch_bounds__(kThreads, 4) tree_verify_kernel(const VerifyArgs a) {
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y;
  const bool tells = rank == 0 && tid == 0;
  // (waited for before another CTA's shared memory is written: it has to have begun)
  if (ranks > 1) {
    if (tid == 0) {
      mbar_init(&s.landed[0], 1);
      mbar_init(&s.landed[1], 1);
      fence_mbar_init();
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  auto report = [&](int bit) {
    if (a.error_flag) atomicOr(a.error_flag, bit);
  };
  const int first = __ldg(a.indptr + b), end = __ldg(a.indptr + b + 1);
  const bool bad = first < 0 || end < first || end > a.total || end - first > kMaxNodes;
  if (bad && tells) report(B200KV_DEVERR_BAD_LEN);
  const int n = first < 0 || end < first || end > a.total ? 0 : min(end - first, kMaxNodes);
  int32_t *path = a.path + int64_t(b) * a.max_path;
  if (n == 0) {  // (all CTAs of the cluster alike)
    if (rank == 0)
      for (int i = tid; i < a.max_path; i += kThreads) path[i] = -1;
    if (tells) a.path_lens[b] = 0, a.next[b] = -1;
    return;
  }
  for (int i = tid; i < n; i += kThreads) {
    int parent = __ldg(a.parents + first + i);
    const int64_t token = __ldg(a.tokens + first + i);
    if (parent < -2 || parent >= i) {
      if (rank == 0) report(B200KV_DEVERR_BAD_LEN);
      parent = -1;
    }
    s.u[i] = __ldg(a.accept_u + first + i);
    float p = 0.f, q = 0.f;
    if (i > 0 && parent >= 0) {
      if (token >= 0 && token < a.vocab) {
        p = to_float(static_cast<const T *>(a.target)[(first + parent) * a.target_stride + token]);
        if (kDraft) q = to_float(static_cast<const T *>(a.draft)[(first + parent) * a.draft_stride + token]);
      } else {
        if (rank == 0) report(B200KV_DEVERR_BAD_TOKEN);
        parent = -1;  // never tried
      }
    }
    s.parent[i] = i == 0 ? -1 : parent;
    s.token[i] = static_cast<int>(token);
    s.p[i] = p;
    s.q[i] = q;
  }
  __syncthreads();

  int x0, x1;
  if (a.vectors)
    part_of<16 / sizeof(T)>(a.vocab, ranks, rank, warp, x0, x1);
  else
    part_of<1>(a.vocab, ranks, rank, warp, x0, x1);

  // warp 0's state: the node reached, the last child tried, path length, c, S, rejected ones
  int cur = 0, at = 0, len = 1, gone = 0;
  double c = 0.0, mass = 1.0;
  bool whole = false;  // nothing was left: drawn from all of p
  if (tells) path[0] = 0;
  for (int pass = 0;; ++pass) {
    if (warp == 0) {
      bool last = whole;
      while (!last) {
        const int i = len < a.max_path ? next_child(s, cur, at, n) : n;
        if (i >= n) {
          last = true;
          break;
        }
        at = i;
        const int x = s.token[i];
        double w;
        bool yes;
        if (kDraft) {
          w = weight<true>(s.p[i], s.q[i], c);
          yes = w > static_cast<double>(s.u[i]) * mass * static_cast<double>(s.q[i]);
        } else {
          w = weight<false>(s.p[i], 0.f, 0.0);
          for (int g = 0; g < gone; ++g)
            if (s.gone[g] == x) w = 0.0;
          yes = w > static_cast<double>(s.u[i]) * fmax(mass, 0.0);
        }
        if (yes) {
          if (rank == 0 && lane == 0) path[len] = i;
          ++len;
          cur = i, gone = 0, c = 0.0, mass = 1.0;
        } else if (kDraft) {
          c += mass;
          last = next_child(s, cur, at, n) >= n;
          break;  // S over the row
        } else {
          mass -= w;
          if (lane == 0) s.gone[gone] = x;
          ++gone;
          __syncwarp();
        }
      }
      if (lane == 0) s.row = first + cur, s.c = c, s.num_gone = gone, s.last = last;
    }
    __syncthreads();
    const int row = s.row, num_gone = s.num_gone;
    const double coef = s.c;
    const bool last = s.last;
    constexpr int kVec = 16 / sizeof(T);
    const double part = a.vectors ? sum_part<T, kDraft, kVec>(a, s, row, coef, num_gone, x0, x1)
                                  : sum_part<T, kDraft, 1>(a, s, row, coef, num_gone, x0, x1);
    if (lane == 0) s.warp_sum[warp] = part;
    __syncthreads();
    double total = 0.0;
    if (ranks == 1) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) total += s.warp_sum[w];
      if (tid == 0) s.cta_sum[pass & 1][0] = total;
      __syncthreads();
    } else {
      if (pass == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
      if (tid == 0) mbar_arrive_expect_tx(&s.landed[pass & 1], static_cast<uint32_t>(ranks) * 8u);
      if (tid < ranks) {
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += s.warp_sum[w];
        send(&s.cta_sum[pass & 1][rank], &s.landed[pass & 1], tid, sum);
      }
      if (__syncthreads_or(!landed(&s.landed[pass & 1], (pass >> 1) & 1u))) {
        if (tells) report(B200KV_DEVERR_TIMEOUT), a.next[b] = -1;
        cluster.sync();  // (what the others send finds this CTA still there)
        break;
      }
      for (int r = 0; r < ranks; ++r) total += s.cta_sum[pass & 1][r];
    }
    if (!last) {
      mass = total;
      continue;
    }
    if (!(total > 0.0)) {
      if (whole) {  // a row without weight
        if (tells) {
          report(B200KV_DEVERR_BAD_TOKEN);
          a.next[b] = -1;
        }
        break;
      }
      whole = true, c = 0.0, gone = 0;
      continue;
    }
    // whose part passes t: the same in every CTA
    const double t = static_cast<double>(__ldg(a.sample_u + b)) * total;
    double before = 0.0, run = 0.0;
    int who = -1;
    for (int r = 0; r < ranks; ++r) {
      const double x = s.cta_sum[pass & 1][r];
      if (x > 0.0 && (who < 0 || !(run > t))) who = r, before = run;
      run += x;
      if (who >= 0 && run > t) break;
    }
    if (who == rank) {
      run = before;
      int mine = -1;
      for (int w = 0; w < kWarps; ++w) {
        const double x = s.warp_sum[w];
        if (x > 0.0 && (mine < 0 || !(run > t))) mine = w, before = run;
        run += x;
        if (mine >= 0 && run > t) break;
      }
      int y0, y1;  // that warp's part
      if (a.vectors)
        part_of<kVec>(a.vocab, ranks, rank, mine, y0, y1);
      else
        part_of<1>(a.vocab, ranks, rank, mine, y0, y1);
      const int x = a.vectors ? find_in_part<T, kDraft, kVec>(a, s, row, coef, num_gone, y0, y1, t - before)
                              : find_in_part<T, kDraft, 1>(a, s, row, coef, num_gone, y0, y1, t - before);
      if (x >= 0) a.next[b] = x;
    }
    break;
  }
  if (rank == 0 && warp == 0) {
    for (int i = len + lane; i < a.max_path; i += 32) path[i] = -1;
    if (lane == 0) a.path_lens[b] = len;
  }
}

template <typename T, bool kDraft>
int launch(const VerifyArgs &a, int ranks, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ranks), static_cast<unsigned>(a.batch));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, tree_verify_kernel<T, kDraft>, a));
  return B200KV_OK;
}
template <typename T>
int launch(const VerifyArgs &a, int ranks, cudaStream_t stream) {
  return a.draft ? launch<T, true>(a, ranks, stream) : launch<T, false>(a, ranks, stream);
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_tree_verify(const int32_t *parents, const int64_t *tokens, const int32_t *q_indptr,
                                  const void *target_probs, int64_t target_stride, const void *draft_probs,
                                  int64_t draft_stride, int32_t dtype, const float *accept_u, const float *sample_u,
                                  int32_t *path, int32_t *path_lens, int64_t *next_tokens, int64_t total_q,
                                  int64_t batch, int64_t vocab, int64_t max_path, int32_t *error_flag, void *stream) {
  clear_error();
  B200KV_CHECK_ARG(dtype == B200KV_F16 || dtype == B200KV_BF16 || dtype == B200KV_F32,
                   "dtype %d is not fp16, bf16 or fp32", dtype);
  B200KV_CHECK_ARG(batch >= 0 && batch <= 65535, "batch %lld out of range", (long long)batch);
  B200KV_CHECK_ARG(total_q >= 0 && total_q < (int64_t{1} << 31), "total_q %lld out of range", (long long)total_q);
  B200KV_CHECK_ARG(vocab > 0 && vocab < (1 << 30), "vocab %lld out of range", (long long)vocab);
  B200KV_CHECK_ARG(max_path > 0 && max_path < (1 << 30), "max_path %lld out of range", (long long)max_path);
  if (batch == 0) return B200KV_OK;
  B200KV_CHECK_ARG(q_indptr && sample_u && path && path_lens && next_tokens, "null pointer argument");
  B200KV_CHECK_ARG(total_q == 0 || (parents && tokens && target_probs && accept_u), "null pointer argument");
  const int64_t size = dtype == B200KV_F32 ? 4 : 2;
  B200KV_CHECK_ARG(aligned_to(target_probs, size) && aligned_to(draft_probs, size), "rows must be aligned to their elements");
  int dev = 0, sms = 0;
  const int st = current_device_sm_count(&dev, &sms);
  if (st != B200KV_OK) return st;
  VerifyArgs a{};
  a.parents = parents, a.tokens = tokens, a.indptr = q_indptr;
  a.target = target_probs, a.target_stride = target_stride, a.draft = draft_probs, a.draft_stride = draft_stride;
  a.accept_u = accept_u, a.sample_u = sample_u, a.path = path, a.path_lens = path_lens, a.next = next_tokens;
  a.total = static_cast<int>(total_q), a.batch = static_cast<int>(batch), a.vocab = static_cast<int>(vocab);
  a.max_path = static_cast<int>(max_path);
  const int64_t vec = 16 / size;
  auto vectors = [&](const void *p, int64_t stride) { return aligned_to(p, 16) && (total_q <= 1 || stride % vec == 0); };
  a.vectors = vectors(target_probs, target_stride) && (!draft_probs || vectors(draft_probs, draft_stride));
  a.error_flag = error_flag;
  // As many CTAs to a sequence as give every warp a step of the row, four to an SM at most in all.
  const int64_t steps = (vocab + 32 * vec - 1) / (32 * vec);
  int ranks = kMaxCluster;
  while (ranks > 1 && (batch * ranks > 4 * sms || steps < ranks * kWarps)) ranks /= 2;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200KV_F16: return launch<__half>(a, ranks, s);
    case B200KV_BF16: return launch<__nv_bfloat16>(a, ranks, s);
    default: return launch<float>(a, ranks, s);
  }
}
