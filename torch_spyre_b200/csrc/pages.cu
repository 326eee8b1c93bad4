// A step's block tables, slots and positions from the requests' lengths, without
// the host.  Free pages are a stack (free_pages[0 .. free_count - 1]).  With
//   want_b = ceil((ctx_b + n_b) / 64),  need_b = max(0, want_b - owned_b),
//   off_b  = need_0 + .. + need_{b-1},
// sequence b's j-th new page is free_pages[free_count - 1 - off_b - j] (extend),
// and release puts pages back in the opposite order, so that an extend that is
// released whole leaves the stack as it was.  Token i of sequence b has
//   slot = table[b][p / 64] * 64 + p % 64,  p = ctx_b + i.
//
// Bound: latency, a chain of lengths -> prefix sum -> page ids -> table -> slot in
// one CTA; a prompt's many slots, 12 bytes each, are a second launch over all SMs, which
// starts while the first runs.  64 sequences with up to 8 nodes: 5.2 us, release 3.8; 256 prompts of up to
// 1024 tokens: 6.3 + 5.6, release 6.4 (16 pages a sequence).
#include "common.cuh"

namespace b200kv {
namespace {

constexpr int kThreads = 1024, kMaxBatch = 1024;

struct PageArgs {
  int32_t *table;
  int64_t stride;
  int32_t *counts, *free_pages, *free_count;
  const int32_t *lens;    // extend: committed tokens; release: tokens that are kept
  const int32_t *indptr;  // extend
  const uint64_t *mask;
  int64_t words;
  int batch, max_blocks, capacity, total;
  int64_t *slots;
  int32_t *positions;
  int32_t *error_flag;
};

__device__ __forceinline__ void report(const PageArgs &a, int bit) {
  if (a.error_flag) atomicOr(a.error_flag, bit);
}

// The pages that a sequence of ctx committed tokens and new ones (first .. end - 1) fills,
// as far as its row of the table has room.  One whose length or offsets cannot be adds
// nothing, and fills none: taken as the nearest that can be, a length past the table
// would take all of its row from the stack.
__device__ __forceinline__ int pages_of(const PageArgs &a, int first, int end, int ctx, bool &bad) {
  const int cap = a.max_blocks * kPageTokens;
  bad = ctx < 0 || ctx > cap || first < 0 || end < first || end > a.total;
  if (bad) return 0;
  bad = end - first > cap - ctx;
  return (ctx + min(end - first, cap - ctx) + kPageTokens - 1) / kPageTokens;
}

// Depth of token t in its tree, less than 0 without a bit in its mask.
__device__ __forceinline__ int depth_of(const PageArgs &a, int t) {
  int depth = -1;
  for (int64_t w = 0; w < a.words; ++w) depth += __popcll(__ldg(a.mask + t * a.words + w));
  return depth;
}

// The slots of a token, from a table and counts that are complete.  `indptr`,
// `counts` and `lens` may be copies in shared memory; `depth`: depth_of(t).
__device__ __forceinline__ void place(const PageArgs &a, const int32_t *indptr, const int32_t *counts, const int32_t *lens,
                                      int t, int depth) {
  int lo = 0, hi = a.batch - 1;  // the last sequence that begins at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (indptr[mid] <= t) lo = mid; else hi = mid - 1;
  }
  int64_t slot = -1;
  int pos = 0;
  const int first = indptr[lo];
  if (first >= 0 && first <= t && t < indptr[lo + 1] && indptr[lo + 1] <= a.total) {
    const int cap = a.max_blocks * kPageTokens, ctx = min(max(lens[lo], 0), cap), i = t - first;
    depth = a.mask ? max(depth, 0) : i;
    pos = ctx + min(depth, INT_MAX - ctx);
    // (with a length that cannot be it has no slots: they would be those of committed tokens)
    if (ctx == lens[lo] && i < cap - ctx) {
      const int at = ctx + i, page = at / kPageTokens;
      const int id = page < counts[lo] ? a.table[lo * a.stride + page] : -1;
      if (id >= 0) slot = int64_t(id) * kPageTokens + at % kPageTokens;
      else if (page < counts[lo]) report(a, B200KV_DEVERR_BAD_BLOCK);
    }
  } else {
    report(a, B200KV_DEVERR_BAD_LEN);
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

__device__ __forceinline__ int scan_block(int x, int *warps) {  // inclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, m);
    if (lane >= m) x += y;
  }
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  int sum = warps[lane];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, m);
    if (lane >= m) sum += y;
  }
  const int before = __shfl_sync(0xffffffffu, sum, max(warp - 1, 0));
  return warp > 0 ? x + before : x;
}

// One CTA: thread b has sequence b.  kSlots: places the tokens too.
template <bool kRelease, bool kSlots>
__global__ void __launch_bounds__(kThreads) pages_kernel(const PageArgs a) {
  __shared__ int32_t indptr[kMaxBatch + 1], counts[kMaxBatch], lens[kMaxBatch];
  __shared__ int warps[32], moved, sums[kMaxBatch], firsts[kMaxBatch];
  const int b = threadIdx.x;
  if (!kRelease && !kSlots) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // slots_kernel
  // all that is read without waiting for something else, first
  const int stack_in = a.free_count[0];
  int owned_in = 0, len = 0, begin = 0, end = 0;
  if (b < a.batch) {
    owned_in = a.counts[b];
    len = a.lens[b];
    if (!kRelease) begin = a.indptr[b], end = a.indptr[b + 1];
  }
  const int depth = kSlots && a.mask && b < a.total ? depth_of(a, b) : 0;
  if (b == 0) moved = 0;
  const int stack = min(max(stack_in, 0), a.capacity);
  if (b == 0 && stack != stack_in) report(a, B200KV_DEVERR_BAD_LEN);
  int first = 0, need = 0, owned = 0;
  if (b < a.batch) {
    owned = min(max(owned_in, 0), a.max_blocks);
    bool bad;
    if (kRelease) {
      bad = len < 0;
      first = bad ? owned : min(owned, len / kPageTokens + (len % kPageTokens != 0));
      need = owned - first;
    } else {
      if (kSlots) {
        indptr[b] = begin, lens[b] = len;
        if (b == a.batch - 1) indptr[a.batch] = end;
      }
      first = owned;
      need = max(pages_of(a, begin, end, len, bad) - owned, 0);
    }
    if (bad || owned != owned_in) report(a, B200KV_DEVERR_BAD_LEN);
  }
  const int upto = scan_block(need, warps);  // (the sums fit: batch * max_blocks < 2^31)
  const int room = kRelease ? a.capacity - stack : stack;
  const bool served = upto <= room;
  if (need > 0 && !served) report(a, B200KV_DEVERR_NO_PAGES);
  const int n = served ? need : 0, off = upto - need;
  if (n > 0) atomicMax(&moved, upto);  // who is served: all before the first who is not
  if (b < a.batch) {
    const int now = kRelease ? owned - n : owned + n;
    if (kSlots) counts[b] = now;
    a.counts[b] = now;
  }
  __syncthreads();  // (release counts down from its end)
  // Page `at` of all that move is entry `from` of sequence `seq`.
  auto move = [&](int seq, int from, int at, int j) {
    int32_t *entry = a.table + seq * a.stride + from + j;
    if (kRelease) {
      a.free_pages[stack + moved - 1 - (at + j)] = *entry;
      *entry = -1;
    } else {
      *entry = __ldg(a.free_pages + stack - 1 - (at + j));
    }
  };
  // few pages each: a thread for a sequence; many: a thread for a page, whose sequence is
  // the first that the sum passes it at (256 prompts of up to 16 pages: a warp for a
  // sequence after the other took 16 us, this 6)
  sums[b] = served ? upto : INT_MAX;
  firsts[b] = first - off;
  if (!__syncthreads_or(n > 4)) {
    for (int j = 0; j < n; ++j) move(b, first, off, j);
  } else {
    for (int k = b; k < moved; k += kThreads) {
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > k) hi = mid; else lo = mid + 1;
      }
      move(lo, firsts[lo] + k, k, 0);
    }
  }
  __syncthreads();
  if (b == 0) a.free_count[0] = kRelease ? stack + moved : stack - moved;
  if (kSlots)
    for (int t = b; t < a.total; t += kThreads) place(a, indptr, counts, lens, t, t == b || !a.mask ? depth : depth_of(a, t));
}

__global__ void __launch_bounds__(256) slots_kernel(const PageArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  const int depth = a.mask && t < a.total ? depth_of(a, t) : 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the table and the counts are pages_kernel's
  if (t < a.total) place(a, a.indptr, a.counts, a.lens, t, depth);
}

int check(const int32_t *table, int64_t stride, const int32_t *counts, const int32_t *free_pages, int64_t capacity,
          const int32_t *free_count, const int32_t *lens, int64_t batch, int64_t max_blocks) {
  B200KV_CHECK_ARG(batch >= 0, "batch %lld out of range", (long long)batch);
  if (batch > kMaxBatch)
    return set_error(B200KV_ERR_UNSUPPORTED, "batch %lld > %d unsupported", (long long)batch, kMaxBatch);
  B200KV_CHECK_ARG(max_blocks > 0 && max_blocks < (1 << 21), "max_blocks_per_seq %lld out of range (1 .. 2^21 - 1)",
                   (long long)max_blocks);
  B200KV_CHECK_ARG(stride >= max_blocks, "block_table_stride < max_blocks_per_seq");
  B200KV_CHECK_ARG(capacity >= 0 && capacity < (int64_t{1} << 31), "capacity %lld out of range", (long long)capacity);
  if (batch == 0) return B200KV_OK;
  B200KV_CHECK_ARG(table && counts && free_count && lens && (free_pages || capacity == 0), "null pointer argument");
  return B200KV_OK;
}

PageArgs args_of(int32_t *table, int64_t stride, int32_t *counts, int32_t *free_pages, int64_t capacity,
                 int32_t *free_count, const int32_t *lens, int64_t batch, int64_t max_blocks, int32_t *error_flag) {
  PageArgs a{};
  a.table = table, a.stride = stride, a.counts = counts, a.free_pages = free_pages, a.free_count = free_count;
  a.lens = lens;
  a.batch = static_cast<int>(batch), a.max_blocks = static_cast<int>(max_blocks);
  a.capacity = static_cast<int>(capacity);
  a.error_flag = error_flag;
  return a;
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_extend_pages(int32_t *block_table, int64_t block_table_stride, int32_t *page_counts,
                                   int32_t *free_pages, int64_t capacity, int32_t *free_count,
                                   const int32_t *context_lens, const int32_t *q_indptr, const int64_t *tree_mask,
                                   int64_t mask_words, int64_t *slots, int32_t *positions, int64_t num_tokens,
                                   int64_t batch, int64_t max_blocks_per_seq, int32_t *error_flag, void *stream) {
  clear_error();
  const int st = check(block_table, block_table_stride, page_counts, free_pages, capacity, free_count, context_lens,
                       batch, max_blocks_per_seq);
  if (st != B200KV_OK) return st;
  B200KV_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t{1} << 31) - 1024, "num_tokens %lld out of range",
                   (long long)num_tokens);
  B200KV_CHECK_ARG(!tree_mask || (mask_words > 0 && mask_words <= (1 << 20)), "mask_words %lld out of range",
                   (long long)mask_words);
  B200KV_CHECK_ARG(batch > 0 || num_tokens == 0, "tokens without a sequence");
  if (batch == 0) return B200KV_OK;
  B200KV_CHECK_ARG(q_indptr && (num_tokens == 0 || (slots && positions)), "null pointer argument");
  PageArgs a = args_of(block_table, block_table_stride, page_counts, free_pages, capacity, free_count, context_lens,
                       batch, max_blocks_per_seq, error_flag);
  a.indptr = q_indptr, a.mask = reinterpret_cast<const uint64_t *>(tree_mask), a.words = mask_words;
  a.slots = slots, a.positions = positions, a.total = static_cast<int>(num_tokens);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // One CTA places up to 4 tokens a thread itself.
  if (num_tokens <= 4 * kThreads) {
    pages_kernel<false, true><<<1, kThreads, 0, s>>>(a);
  } else {
    pages_kernel<false, false><<<1, kThreads, 0, s>>>(a);
    B200KV_CUDA_TRY(cudaGetLastError());
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((num_tokens + 255) / 256));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, slots_kernel, static_cast<const PageArgs>(a)));
  }
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}

extern "C" int b200kv_release_pages(int32_t *block_table, int64_t block_table_stride, int32_t *page_counts,
                                    int32_t *free_pages, int64_t capacity, int32_t *free_count,
                                    const int32_t *keep_lens, int64_t batch, int64_t max_blocks_per_seq,
                                    int32_t *error_flag, void *stream) {
  clear_error();
  const int st = check(block_table, block_table_stride, page_counts, free_pages, capacity, free_count, keep_lens, batch,
                       max_blocks_per_seq);
  if (st != B200KV_OK || batch == 0) return st;
  const PageArgs a = args_of(block_table, block_table_stride, page_counts, free_pages, capacity, free_count, keep_lens,
                             batch, max_blocks_per_seq, error_flag);
  pages_kernel<true, false><<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  B200KV_CUDA_TRY(cudaGetLastError());
  return B200KV_OK;
}
