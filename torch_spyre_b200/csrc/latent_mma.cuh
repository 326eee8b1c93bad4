// Tensor-core kernel of latent attention in the absorbed form (latent_attention.cu
// has the operator): cached rows c = (512 latent, 64 rotary) are key and value of
// all heads, so the rows of one product are a sequence's nodes times its heads,
// and a token's 1152 bytes serve all of them.
//
// A CTA holds a tile of up to 64 rows (node-major, of 64 heads at most; latent_pair.cuh
// has the kernel for more) and goes over pages of 64 tokens:
//   S [64 rows, 64 tokens]  = Q K^T        9 sticks of 64 elements
//   O^T [512, rows]        += V^T P^T      4 products of 128 latent elements
// O is kept transposed: as M = 128 latent elements by N = rows it takes 256 TMEM
// columns and the products run at the full rate whatever the number of rows; with
// rows on M it would take all 512.  V^T is the page as it lies (tokens are the
// reduction, their 64-element sticks M-major), P goes through shared memory.
//
// The cache's page is loaded once, in two halves (the rotary stick with the first),
// and its slots are free again once O has taken it.  Two pages are held: one warp
// issues the next page's scores as its halves arrive, another this page's values as
// soon as its weights are there.
//
// The blocks' pages, all sequences one after the other, form one line that is cut
// into equal shares; blocks cut by a share's end are joined by latent_join_kernel.
//
// Bound, up to 64 rows: memory; the products take 1920 of the 3080 clocks that a page's
// 74 KB take at the copy rate on every SM.  What costs beside that are the hand-overs:
// a wait for a barrier that is already complete takes some 200 clocks of a warp's time
// between products, so there are few of them, and roles that would wait for one another
// are warps of their own.  64 sequences of up to 8192 tokens (321 MB), 16 heads: 68 us,
// 70 among other work, 4.7 TB/s with the plan (2 to 3 us), pieces' ends and the join (6.5 us by itself).
//
// Warps: 0-7 softmax and output (warp w: lanes 0-15 of quadrant w % 4 have rows
// 16 (w % 4) .., where an M = 64 accumulator lies, and half w / 4 of a page's tokens),
// 8 TMA producer, 9 issues the scores' MMAs, 10 the values'.
#pragma once

#include "latent_attention.h"
#include "umma.cuh"

namespace b200kv {
namespace latent {

using namespace umma;

constexpr int kThreads = 384;  // (one warp without a role here, the pairs' relay there)
constexpr int kSoftmaxWarps = 8;
constexpr int kTile = kPageTokens;
constexpr int kStickTile = kTile * 128, kPair = 2 * kStickTile, kPairs = 4, kSlots = 8;
constexpr float kLazyLog2 = 8.f;
constexpr int kOffQ = 2048;
constexpr int kOffP = kOffQ + kSticks * kStickTile;
constexpr int kOffRope = kOffP + 2 * kStickTile;
constexpr int kOffSlots = kOffRope + kStickTile;
constexpr int kSmem = kOffSlots + kSlots * kPair;
static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
static_assert(kSlots == 2 * kPairs, "page n has pairs (n & 1) * kPairs ..");

// TMEM columns: O^T, 64 for each 128 latent elements, and two score buffers
constexpr uint32_t kTmemCols = 512;
__device__ __forceinline__ uint32_t col_o(int m) { return uint32_t(m) * 64u; }
__device__ __forceinline__ uint32_t col_s(int b) { return 256u + uint32_t(b) * 64u; }

struct Seq {
  int ctx, nodes, q0, blocks;
  int end;  // the first row of q that is a later sequence's
};
struct Start {  // where a share of the line begins: in block `block`, whose units begin at u0
  Seq s;
  int b, block, u0;
};

struct Plan {
  int per, total;  // units of a share, of the line
  Start start;
  int scan[kThreads / 32];
};

struct Ctrl {
  uint64_t full[4], empty[4], rope_empty;  // halves of the two pages held (the rotary stick comes with the first)
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_ready[2], p_free[2], o_full, o_empty;
  uint32_t tmem;
  Plan plan;
  float top[2][kTileRows];  // maxima, then sums, of the halves of a row's tokens
  float factor[kTileRows];  // of O's columns
  int row_at[kTileRows];    // row of out, -1: none
};
static_assert(sizeof(Ctrl) <= kOffQ, "control block");

__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool any_softmax(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"(uint32_t(x))
               : "memory");
  return r != 0;
}

// -------------------------------------------------------------------- plan --
__device__ __forceinline__ Seq load_seq(const Args &a, int b, bool report) {
  const int cap = a.max_blocks * kPageTokens;
  Seq s;
  s.ctx = __ldg(a.ctx + b);
  s.q0 = __ldg(a.indptr + b);
  const int end = __ldg(a.indptr + b + 1);
  bool bad = s.ctx < 0 || s.ctx > cap || s.q0 < 0 || end < s.q0 || end > a.total_q || (b == 0 && s.q0 != 0) ||
             (b == a.batch - 1 && end != a.total_q);
  s.ctx = min(max(s.ctx, 0), cap);
  s.q0 = min(max(s.q0, 0), a.total_q);
  s.nodes = min(max(end, s.q0), a.total_q) - s.q0;
  s.end = b == a.batch - 1 ? a.total_q : min(max(end, 0), a.total_q);
  const int most = min(a.max_nodes, cap - s.ctx);
  bad = bad || s.nodes > most;
  s.nodes = min(s.nodes, most);
  if (bad && report && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
  s.blocks = (s.nodes + a.block_nodes - 1) / a.block_nodes;
  return s;
}
// Token tiles (of kStep tokens) of block k: what its last node can see.
template <int kStep>
__device__ __forceinline__ int block_tiles(const Args &a, const Seq &s, int k) {
  const int nodes = a.mask ? s.nodes : min(s.nodes, (k + 1) * a.block_nodes);
  return (s.ctx + nodes + kStep - 1) / kStep;
}
// The line is cut by cost: a tile counts one, a block's beginning and end kBegin.
constexpr int kBegin = 3;
template <int kStep>
__device__ __forceinline__ int block_units(const Args &a, const Seq &s, int k) {
  return kBegin + block_tiles<kStep>(a, s, k);
}
template <int kStep>
__device__ __forceinline__ int seq_units(const Args &a, const Seq &s) {
  if (a.mask) return s.blocks > 0 ? s.blocks * block_units<kStep>(a, s, 0) : 0;
  int n = 0;
  for (int k = 0; k < s.blocks; ++k) n += block_units<kStep>(a, s, k);
  return n;
}

// The blocks of a share, one piece (a block, or the part of it in this share) at
// a time.  Every role walks the same sequence.
template <int kStep>
struct Walk {
  Seq s;
  int b, block, u0, tiles, t0, t1;  // piece: token tiles [t0, t1) of `tiles`
  int first, end;                   // of the share

  __device__ __forceinline__ void init(const Args &a, const Plan &c) {
    const Start &f = c.start;
    s = f.s, b = f.b, block = f.block, u0 = f.u0;
    t0 = t1 = 0;
    const int share = static_cast<int>(blockIdx.x) / a.stride;
    first = share * c.per;
    end = min(c.total, first + c.per);
  }
  // Tile t belongs to the share that holds its unit; the begin goes with the first.
  __device__ __forceinline__ int tile_from(int unit) const { return min(max(unit - u0 - kBegin, 0), tiles); }
  __device__ __forceinline__ bool next(const Args &a) {
    for (;;) {
      if (u0 >= end || first >= end) return false;
      tiles = block_tiles<kStep>(a, s, block);
      t0 = tile_from(first);
      t1 = tile_from(end);
      if (t0 < t1) return true;
      advance(a);
    }
  }
  __device__ __forceinline__ void advance(const Args &a) {
    u0 += block_units<kStep>(a, s, block);
    if (u0 >= end) return;
    if (++block >= s.blocks) {
      block = 0;
      do s = load_seq(a, ++b, false);
      while (s.nodes == 0);
    }
  }
  __device__ __forceinline__ int share_of(int t, int per) const { return (u0 + kBegin + t) / per; }
  __device__ __forceinline__ int rows(const Args &a) const {  // of the Q tile
    return min(a.tile_nodes, s.nodes - block * a.tile_nodes) * a.head_box;
  }
};

// Rows of q that no sequence has (all of them flagged): they see nothing.
template <typename T>
__device__ __noinline__ void clear_rows(const Args &a, bool all) {
  for (int b = 0; b < a.batch; ++b) {
    const Seq s = load_seq(a, b, false);
    const int first = b == 0 ? 0 : s.q0, end = all ? (b == 0 ? a.total_q : 0) : s.end;
    for (int t = first + blockIdx.x; t < end; t += gridDim.x) {
      if (!all && t >= s.q0 && t < s.q0 + s.nodes) continue;
      uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + static_cast<int64_t>(t) * a.heads * kRank);
      for (int i = threadIdx.x; i < a.heads * (kRank / 8); i += blockDim.x) out[i] = make_uint4(0, 0, 0, 0);
      if (!a.lse) continue;
      for (int h = threadIdx.x; h < a.heads; h += blockDim.x) a.lse[static_cast<int64_t>(t) * a.heads + h] = -CUDART_INF_F;
    }
  }
}

// The line's length, a share's, and where this CTA's begins; all threads call it,
// a barrier follows.  (With a q_indptr that descends nothing has a sequence: its
// sequences could have the same rows, and the counts pass 31 bits.)
template <typename T, int kStep>
__device__ __forceinline__ void make_plan(const Args &a, Plan &c) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.batch + kThreads - 1) / kThreads;
  const int b0 = tid * each, b1 = min(b0 + each, a.batch);
  Seq s{};
  int mine = 0;
  bool unclaimed = false, descends = false;
  for (int b = b0; b < b1; ++b) {
    s = load_seq(a, b, blockIdx.x == 0);
    mine += seq_units<kStep>(a, s);
    unclaimed = unclaimed || (b == 0 && s.q0 > 0) || s.q0 + s.nodes < s.end;
    descends = descends || s.end < s.q0;
  }
  int incl = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, m);
    if (lane >= m) incl += y;
  }
  if (lane == 31) c.scan[warp] = incl;
  bool none = false;
  if (__syncthreads_or(unclaimed || descends)) {
    none = __syncthreads_or(descends);
    clear_rows<T>(a, none);
  }
  int total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += c.scan[w];
    total += c.scan[w];
  }
  if (none) total = mine = 0;
  const int shares = static_cast<int>(gridDim.x) / a.stride;
  const int per = max(2, static_cast<int>((static_cast<unsigned>(total) + shares - 1) / shares));
  const int first = static_cast<int>(blockIdx.x) / a.stride * per;
  int at = before + incl - mine;
  if (first >= at && first < at + mine) {
    int b = b0;
    for (;; ++b) {
      if (each > 1) s = load_seq(a, b, false);
      const int n = seq_units<kStep>(a, s);
      if (first < at + n) break;
      at += n;
    }
    int block = 0;
    if (a.mask) {
      const int n = block_units<kStep>(a, s, 0);
      block = (first - at) / n;
      at += block * n;
    } else {
      for (int n; first >= at + (n = block_units<kStep>(a, s, block)); ++block) at += n;
    }
    c.start = Start{s, b, block, at};
  }
  if (tid == 0) {
    c.per = per;
    c.total = total;
  }
}

// ------------------------------------------------------------------- roles --
// Page ids of a sequence, 32 at a time in a warp's lanes.  Invalid ids are flagged and become -1.
__device__ __forceinline__ int load_ids(const Args &a, int b, int window, int pages) {
  const int p = window * 32 + (threadIdx.x & 31);
  if (p >= pages) return -1;
  const int id = __ldg(a.block_table + static_cast<int64_t>(b) * a.bt_stride + p);
  if (id < 0 || id >= a.num_blocks) {
    if (a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_BLOCK);
    return -1;
  }
  return id;
}

// Brings page `id` into L2.
__device__ __forceinline__ void page_ahead(const Args &a, int id) {
  prefetch_l2(static_cast<const uint8_t *>(a.pool) + static_cast<int64_t>(id) * (kSticks * kStickTile), kSticks * kStickTile);
}

__device__ __forceinline__ void producer(const Args &a, Ctrl &c, uint8_t *smem, const CUtensorMap *qm,
                                         const CUtensorMap *rm, const CUtensorMap *hm, const CUtensorMap *sm) {
  const int lane = threadIdx.x & 31;
  const uint32_t q_bytes = static_cast<uint32_t>(a.box_nodes * a.head_box * 128);
  // a page is read once (by one block of one CTA; only a sequence of more nodes than a tile holds has
  // several, which read it each) and leaves L2 first
  const uint64_t policy = l2_policy_evict_first();
  bool dead = false;
  uint32_t halves = 0, pieces = 0;  // issued
  Walk<kTile> w;
  w.init(a, c.plan);
  while (w.next(a)) {
    const int pages = (w.s.ctx + w.s.nodes + kPageTokens - 1) / kPageTokens;
    int window = w.t0 / 32, ids = load_ids(a, w.b, window, pages), ids_next = load_ids(a, w.b, window + 1, pages);
    wait(&c.q_empty, (pieces & 1u) ^ 1u, dead, a.error_flag);
    if ((dead = __any_sync(0xffffffffu, dead))) break;
    if (lane == 0) mbar_arrive_expect_tx(&c.q_full, kSticks * q_bytes);
    __syncwarp();
    if (lane < kSticks)
      tma_3d(smem + kOffQ + lane * kStickTile, lane < kSticks - 1 ? qm : rm, &c.q_full, lane < kSticks - 1 ? lane * 64 : 0,
             0, w.s.q0 + w.block * a.tile_nodes);
    ++pieces;
    for (int t = w.t0; t < w.t1 && !dead; ++t) {
      if (t / 32 > window) {
        ids = ids_next;
        ids_next = load_ids(a, w.b, ++window + 1, pages);
      }
      const int id = __shfl_sync(0xffffffffu, ids, t & 31);
      const int page = id < 0 ? a.num_blocks : id;  // an invalid id reads past the last page: zeros
#pragma unroll
      for (int h = 0; h < 2; ++h, ++halves) {
        // halves 2n and 2n + 1 are page n's
        const uint32_t n = halves >> 1, b = halves & 3u;
        wait_until(
            [&] {
              const bool r = h == 1 || mbar_test(&c.rope_empty, (n & 1u) ^ 1u);
              return r & mbar_test(&c.empty[b], ((n >> 1) & 1u) ^ 1u);
            },
            dead, a.error_flag);
        if ((dead = __any_sync(0xffffffffu, dead))) break;
        if (lane == 0) mbar_arrive_expect_tx(&c.full[b], 2 * kPair + (h == 0 ? kStickTile : 0));
        __syncwarp();
        if (lane == 0)
          tma_load_3d(smem + kOffSlots + b * 2 * kPair, hm, &c.full[b], 0, h * 4 * kTile, page, policy);
        else if (lane == 1 && h == 0)
          tma_load_3d(smem + kOffRope, sm, &c.full[b], 0, (kSticks - 1) * kTile, page, policy);
        __syncwarp();
      }
    }
    if (dead) break;
    w.advance(a);
  }
  if (dead) {  // the copies under way, with a limit
    bool late = false;
    if (pieces > 0) wait(&c.q_full, (pieces - 1) & 1u, late, a.error_flag);
    for (uint32_t n = halves - min(halves, 4u); n < halves; ++n) wait(&c.full[n & 3u], (n >> 2) & 1u, late, a.error_flag);
  }
  // the last arrival that the MMAs owe this CTA: not before it may the CTA end
  if (lane == 0 && pieces > 0) {
    bool late = false;
    wait(&c.q_empty, (pieces & 1u) ^ 1u, late, a.error_flag);
  }
  __syncwarp();
}

// The two MMA warps, converged, issue from an elected lane.  Operands are made uniform
// first: an MMA whose descriptors come from ordinary registers takes 60 to 80 clocks to
// issue, twice its own time.
template <typename T>
constexpr uint32_t kIdesc = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10));

template <typename T>
__device__ __forceinline__ void score_issuer(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem_any) {
  const uint32_t go = elect_one(), tmem = uniform(tmem_any);
  const uint32_t idesc = kIdesc<T> | (uint32_t(kTile >> 3) << 17) | (uint32_t(kTileRows >> 4) << 24) |
                         (a.scale < 0.f ? 1u << 13 : 0u);  // a negative scale turns Q's sign
  const uint32_t qd = desc_kmajor(smem_u32(smem + kOffQ)), rd = desc_kmajor(smem_u32(smem + kOffRope));
  const uint32_t kd = desc_kmajor(smem_u32(smem + kOffSlots));
  auto done = [&](uint64_t *bar) {
    if (go) commit(bar);
  };
  bool dead = false;
  uint32_t n = 0, pieces = 0;  // pages, pieces
  Walk<kTile> w;
  w.init(a, c.plan);
  while (w.next(a)) {
    for (int t = w.t0; t < w.t1; ++t, ++n) {
      const uint32_t odd = uniform(n & 1u);
      // this score buffer is free once the page before last has weights
      wait_until(
          [&] {
            const bool free = n < 2 || mbar_test(&c.p_ready[odd], ((n - 2) >> 1) & 1u);
            const bool q = t > w.t0 || mbar_test(&c.q_full, pieces & 1u);
            return free & q & mbar_test(&c.full[2 * odd], (n >> 1) & 1u);
          },
          dead, a.error_flag);
      fence_after();
      const uint32_t s = tmem + col_s(0) + odd * 64, k0 = kd + (odd * kPairs * kPair >> 4);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma_ss(s, qd + ((kSticks - 1) * kStickTile + k * 32 >> 4), rd + (k * 32 >> 4), idesc, k > 0, go);
      done(&c.rope_empty);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t off = ((k >> 2) * kStickTile + (k & 3) * 32) >> 4;
        mma_ss(s, qd + off, k0 + off, idesc, 1, go);
      }
      wait_until([&] { return mbar_test(&c.full[2 * odd + 1], (n >> 1) & 1u); }, dead, a.error_flag);
      fence_after();
#pragma unroll
      for (int k = 16; k < 32; ++k) {
        const uint32_t off = ((k >> 2) * kStickTile + (k & 3) * 32) >> 4;
        mma_ss(s, qd + off, k0 + off, idesc, 1, go);
      }
      done(&c.s_full[odd]);
    }
    done(&c.q_empty);
    ++pieces;
    w.advance(a);
  }
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ void value_issuer(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem_any) {
  const uint32_t go = elect_one(), tmem = uniform(tmem_any);
  const uint32_t pd = desc_kmajor(smem_u32(smem + kOffP));
  const uint32_t vd = (smem_u32(smem + kOffSlots) >> 4) | (uint32_t(kStickTile >> 4) << 16);
  auto done = [&](uint64_t *bar) {
    if (go) commit(bar);
  };
  bool dead = false;
  uint32_t n = 0, pieces = 0;  // pages, pieces
  Walk<kTile> w;
  w.init(a, c.plan);
  while (w.next(a)) {
    // A (V^T): M-major; N: the rows there are
    const uint32_t idesc = uniform(kIdesc<T> | (1u << 15) | (uint32_t(128 >> 4) << 24) | (uint32_t((w.rows(a) + 15) / 16 * 2) << 17));
    for (int t = w.t0; t < w.t1; ++t, ++n) {
      const uint32_t odd = uniform(n & 1u), later = uniform(t > w.t0);
      wait_until(
          [&] {
            const bool free = t > w.t0 || mbar_test(&c.o_empty, (pieces & 1u) ^ 1u);
            return free & mbar_test(&c.p_ready[odd], (n >> 1) & 1u);
          },
          dead, a.error_flag);
      fence_after();
      const uint32_t p = pd + (odd * kStickTile >> 4), v = vd + (odd * kPairs * kPair >> 4);
#pragma unroll
      for (int m = 0; m < kPairs; ++m) {
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          mma_ss(tmem + col_o(m), v + (m * kPair + k * 2048 >> 4), p + (k * 32 >> 4), idesc, k > 0 ? 1 : later, go);
        if (m & 1) done(&c.empty[odd * 2 + m / 2]);
      }
      done(&c.p_free[odd]);
    }
    done(&c.o_full);
    ++pieces;
    w.advance(a);
  }
  __syncwarp();
}

// Which of the tokens pos .. pos + 31 node `node` sees.
__device__ __forceinline__ uint32_t visible32(const Args &a, const Seq &s, int node, int pos) {
  if (!a.mask) return low_bits(s.ctx + node + 1 - pos);
  uint32_t bits = low_bits(s.ctx - pos);
  const int off = pos - s.ctx;
  if (off > -32) {
    const uint64_t *row = a.mask + static_cast<int64_t>(s.q0 + node) * a.words;
    const int w = max(off, 0) >> 6;
    uint64_t m = w < a.words ? __ldg(row + w) : 0;
    if (off < 0) {
      m <<= -off;
    } else {
      const int sh = off & 63;
      m >>= sh;
      if (sh > 32 && w + 1 < a.words) m |= __ldg(row + w + 1) << (64 - sh);
    }
    bits |= static_cast<uint32_t>(m) & low_bits(s.ctx + s.nodes - pos);
  }
  return bits;
}

template <bool kTail>
__device__ __forceinline__ float mask_max(uint32_t (&s)[32], uint32_t vis) {
  if (kTail) {
#pragma unroll
    for (int j = 0; j < 32; ++j) s[j] = vis >> j & 1u ? s[j] : 0xff800000u;  // -inf
  }
  float t = __uint_as_float(s[0]);
#pragma unroll
  for (int j = 1; j < 31; j += 2) t = fmaxf(fmaxf(t, __uint_as_float(s[j])), __uint_as_float(s[j + 1]));
  return fmaxf(t, __uint_as_float(s[31]));
}

// This warp's part of O, two of the four products, times its columns' factors.
static __device__ __noinline__ void rescale(const Ctrl &c, uint32_t quad, int half, int rows) {
#pragma unroll 1
  for (int m = 2 * half; m < 2 * half + 2; ++m)
#pragma unroll 1
    for (int j0 = 0; j0 < rows; j0 += 16) {
      uint32_t r[16];
      tmem_ld16(quad + col_o(m) + j0, r);
      wait_ld(r);
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * c.factor[j0 + j]);
      tmem_st16(quad + col_o(m) + j0, r);
    }
  wait_st();
}

// Scores of 32 tokens -> weights in 16 bits, as 64 bytes of a row of P (`at`, with the
// row's swizzle), and their sum.
template <typename T>
__device__ __forceinline__ float put_weights(const uint32_t (&s)[32], float cl, float m, uint8_t *at, int chunk, int swizzle,
                                             bool store) {
  const float minus = m == -CUDART_INF_F ? 0.f : -m;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = make_float2(__uint_as_float(s[8 * k + 2 * j]), __uint_as_float(s[8 * k + 2 * j + 1]));
      const float2 y = fma2(x, make_float2(cl, cl), make_float2(minus, minus));
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      sum[j & 1] = add2(sum[j & 1], e);
      p[j] = pack2(e.x, e.y, T());
    }
    if (store) *reinterpret_cast<uint4 *>(at + (((chunk + k) ^ swizzle) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
  }
  const float2 x = add2(sum[0], sum[1]);
  return x.x + x.y;
}

// Rows of some of a page's sticks in shared memory: those from `end` on, past
// the sequence's end, hold anything and become zeros, so that weights of zero meet
// finite values; so do non-finite elements from `from` on, of nodes that not every row
// sees (a row that sees such a node has its score, which is not finite either: NaN
// everywhere, or no weight for it).  128 threads, 16 bytes each: row 16 k + tid / 8.
template <typename T, int kOf>  // sticks
__device__ __noinline__ void clean(uint8_t *half, int tid, int from, int end) {
#pragma unroll 1
  for (int st = 0; st < kOf; ++st)
#pragma unroll 1
    for (int k = min(from, max(end, 0)) / 16; k < 4; ++k) {
      uint4 *cell = reinterpret_cast<uint4 *>(half + st * kStickTile + k * 2048 + tid * 16);
      const int row = 16 * k + (tid >> 3);
      if (row >= end) {
        *cell = make_uint4(0, 0, 0, 0);
      } else if (row >= from) {
        uint4 x = *cell;
        if (!any_non_finite<T>(x)) continue;
        drop_non_finite<T>(x);
        *cell = x;
      }
    }
}

// Softmax of the CTA's rows, and their output.
template <typename T>
__device__ __forceinline__ void softmax(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int half = warp >> 2, row = 16 * (warp & 3) + (lane & 15);
  const bool has_row = lane < 16;
  const uint32_t quad = tmem + (uint32_t((warp & 3) * 32) << 16);
  // (a scale of zero: too small to move a score, and -inf stays -inf)
  const float cl = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1e-37f);
  bool dead = false;
  uint32_t n = 0;  // pages
  unsigned piece = 0;
  Walk<kTile> wk;
  wk.init(a, c.plan);
  while (wk.next(a)) {
    ++piece;
    const int len = wk.s.ctx + wk.s.nodes, rows = wk.rows(a);
    const int node = wk.block * a.tile_nodes + row / a.head_box;
    const int head = row % a.head_box;
    const bool live = has_row && row < rows;
    const bool warp_live = __any_sync(0xffffffffu, live);
    // tokens before this one are seen by every row of the tile
    const int common = wk.s.ctx + (a.mask ? 0 : wk.block * a.tile_nodes + 1);
    float m = -CUDART_INF_F, l = 0.f;
    for (int t = wk.t0; t < wk.t1; ++t, ++n) {
      const int pos = t * kTile;
      const bool first = t == wk.t0, tail = pos + kTile > common;
      const uint32_t vis = tail && live ? visible32(a, wk.s, node, pos + 32 * half) : ~0u;
      wait(&c.s_full[n & 1], (n >> 1) & 1u, dead, a.error_flag);
      fence_after();
      uint32_t s[32];
      float mt = -CUDART_INF_F;
      if (warp_live) {
        tmem_ld32(quad + col_s(n & 1) + 32 * half, s);
        wait_ld(s);
        mt = fmaf(tail ? mask_max<true>(s, vis) : mask_max<false>(s, ~0u), cl, -kWeightLog2<T>);
      }
      // the maximum is that of both halves of the row; it moves when either has risen far enough
      if (first || any_softmax(live && mt > m + kLazyLog2)) {
        if (has_row) c.top[half][row] = mt;
        bar_softmax();
        mt = fmaxf(mt, c.top[half ^ 1][row]);
        const bool rise = live && mt > m + (first ? 0.f : kLazyLog2);
        if (!first) {
          // O moves to the new maxima once the values before are in it
          const float keep = rise ? ex2(m - mt) : 1.f;
          l *= keep;
          if (has_row && half == 0) c.factor[row] = keep;
          wait(&c.p_free[(n - 1) & 1], ((n - 1) >> 1) & 1u, dead, a.error_flag);
          fence_after();
          bar_softmax();
          rescale(c, quad, half, rows);
        }
        if (rise) m = mt;
        bar_softmax();  // (maxima and factors are read)
      }
      // P's buffer is free once the values of two pages before are in O
      if (n >= 2) wait(&c.p_free[n & 1], ((n - 2) >> 1) & 1u, dead, a.error_flag);
      if (warp_live)
        l += put_weights<T>(s, cl, m, smem + kOffP + (n & 1) * kStickTile + row * 128, 4 * half, row & 7, has_row);
      if (pos + kTile > min(common, len)) {
        wait(&c.full[(n & 1) * 2 + half], (n >> 1) & 1u, dead, a.error_flag);
        clean<T, 4>(smem + kOffSlots + ((n & 1) * 2 + half) * 2 * kPair, tid & 127, max(common - pos, 0), len - pos);
      }
      fence_async_smem();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(&c.p_ready[n & 1]);
    }

    // -------------------------------------------------------- end of piece --
    const bool split = wk.t0 > 0 || wk.t1 < wk.tiles;
    const int64_t pslot = 2 * blockIdx.x + (wk.t0 > 0 ? 0 : 1);  // one of each kind per share
    const int64_t orow = static_cast<int64_t>(wk.s.q0 + node) * a.heads + head;
    if (has_row) c.top[half][row] = l;
    bar_softmax();
    if (has_row && half == 0) {
      l = c.top[0][row] + c.top[1][row];
      c.factor[row] = split ? 1.f : (l == 0.f ? 0.f : 1.f / l);
      c.row_at[row] = live ? static_cast<int>(orow) : -1;
      if (live && split)
        a.part_ml[pslot * kTileRows + row] = make_float2(m, l);
      else if (live && a.lse)
        a.lse[orow] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * 0.69314718055994530942f;
    }
    bar_softmax();
    wait(&c.o_full, (piece - 1) & 1u, dead, a.error_flag);
    fence_after();
#pragma unroll 1
    for (int x = 0; x < 4; ++x) {
      const int mblock = 2 * half + (x >> 1), j0 = (x & 1) * 32;
      if (j0 >= rows) continue;
      const int d = 128 * mblock + 32 * (warp & 3) + lane;  // this lane's latent element
      uint32_t r[32];
      tmem_ld32(quad + col_o(mblock) + j0, r);
      wait_ld(r);
      if (split) {
        float *to = a.part_o + (pslot * kTileRows + j0) * kRank + d;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c.row_at[j0 + j] >= 0) to[j * kRank] = __uint_as_float(r[j]);
      } else {
        // lanes in pairs: two neighbouring elements of every other row each
        T *out = static_cast<T *>(a.out) + (d & ~1);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float y[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = c.factor[j0 + j + i];
            y[i] = f == 0.f ? 0.f : __uint_as_float(r[j + i]) * f;
          }
          const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? y[0] : y[1], 1);
          const int to = c.row_at[j0 + j + (lane & 1)];
          const uint32_t two = lane & 1 ? pack2(other, y[1], T()) : pack2(y[0], other, T());
          if (to >= 0) *reinterpret_cast<uint32_t *>(out + static_cast<int64_t>(to) * kRank) = two;
        }
      }
    }
    fence_before();
    bar_softmax();  // (the factors and rows are read)
    if (lane == 0) arrive(&c.o_empty);
    // the second share of a split block describes it to the join
    if (wk.t0 > 0 && tid == 0) {
      const int first = wk.share_of(0, c.plan.per);
      if (static_cast<int>(blockIdx.x) == first + 1) {
        Join j;
        j.rows0 = wk.s.q0;
        j.node0 = wk.block * a.tile_nodes;
        j.nodes = min(wk.s.nodes - j.node0, a.tile_nodes);
        j.head0 = 0;
        j.first = first;
        j.last = wk.share_of(wk.tiles - 1, c.plan.per);
        a.joins[blockIdx.x] = j;
      }
    }
    wk.advance(a);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    latent_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap rm,
                  const __grid_constant__ CUtensorMap hm, const __grid_constant__ CUtensorMap,
                  const __grid_constant__ CUtensorMap sm, const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Ctrl &c = *reinterpret_cast<Ctrl *>(smem);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    prefetch_tensormap(&qm);
    prefetch_tensormap(&rm);
    prefetch_tensormap(&hm);
    prefetch_tensormap(&sm);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 1);
    }
    mbar_init(&c.rope_empty, 1);
    mbar_init(&c.q_full, 1);
    mbar_init(&c.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.s_full[i], 1);
      mbar_init(&c.p_ready[i], kSoftmaxWarps);
      mbar_init(&c.p_free[i], 1);
    }
    mbar_init(&c.o_full, 1);
    mbar_init(&c.o_empty, kSoftmaxWarps);
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) a.joins[blockIdx.x].nodes = 0;  // no block begins to be split here, unless the epilogue says so
  make_plan<T, kTile>(a, c.plan);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = c.tmem;
  if (warp < kSoftmaxWarps)
    softmax<T>(a, c, smem, tmem);
  else if (warp == 8)
    producer(a, c, smem, &qm, &rm, &hm, &sm);
  else if (warp == 9)
    score_issuer<T>(a, c, smem, tmem);
  else if (warp == 10)
    value_issuer<T>(a, c, smem, tmem);
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------- join --
// Blocks cut by shares: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the
// pieces in order (the same bits every time).  4 rows a CTA, 2 x 4 elements a thread.
// The pieces' maxima and sums come first, one to a lane, so that the sums over their
// elements are loads that wait for nothing, eight under way.
template <typename T, bool kPairs>
__global__ void __launch_bounds__(256) latent_join_kernel(const __grid_constant__ Args a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float weight[4][kMaxCtas];
  __shared__ float2 whole[4];  // rows' maxima and sums
  const Join j = a.joins[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = static_cast<int>(blockIdx.x) % a.stride;
  if (blockIdx.y * 4 / a.head_box >= j.nodes) return;  // (the whole CTA)
  auto live = [&](int r) {
    const int row = blockIdx.y * 4 + r;
    return row / a.head_box < j.nodes && j.head0 + row % a.head_box < a.heads;
  };
  const int pieces = j.last - j.first + 1;
  // the partials of piece i are in slot first_slot + i * step, the first piece's in the odd one
  const int64_t slot0 = 2 * (int64_t{j.first} * a.stride + part), step = 2 * a.stride;
  if (warp < 4 && live(warp)) {
    const int row = blockIdx.y * 4 + warp;
    float M = -CUDART_INF_F, l = 0.f;
    for (int i0 = 0; i0 < pieces; i0 += 32) {
      const int i = i0 + lane;
      if (i < pieces) M = fmaxf(M, a.part_ml[(slot0 + i * step + (i == 0)) * kTileRows + row].x);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float mm = M == -CUDART_INF_F ? 0.f : M;
    for (int i0 = 0; i0 < pieces; i0 += 32) {
      const int i = i0 + lane;
      float y = 0.f;
      if (i < pieces) {
        const float2 ml = a.part_ml[(slot0 + i * step + (i == 0)) * kTileRows + row];
        const float w = exp2f(ml.x - mm);
        y = ml.y * w;
        weight[warp][i] = w;
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) y += __shfl_xor_sync(0xffffffffu, y, x);
      l += y;
    }
    if (lane == 0) whole[warp] = make_float2(M, l);
  }
  __syncthreads();
  // rows' elements as the kernel before laid them: neighbours in a warp, or for pairs
  // (there a lane has a row) the 4 rows of 4 elements side by side
  const int r = kPairs ? threadIdx.x & 3 : warp >> 1;
  const int e = kPairs ? threadIdx.x >> 2 : (warp & 1) * 64 + lane, e_step = kPairs ? 64 : 32;  // in fours
  if (!live(r)) return;
  const int row = blockIdx.y * 4 + r;
  const float4 *from = reinterpret_cast<const float4 *>(a.part_o) + (kPairs ? e * kTileRows + row : row * (kRank / 4) + e);
  constexpr int kNext = kPairs ? 64 * kTileRows : 32;
  float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i0 = 0; i0 < pieces; i0 += 4) {
    float4 v[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(i0 + k, pieces - 1);
      const float4 *p = from + (slot0 + i * step + (i == 0)) * (kTileRows * kRank / 4);
      v[k][0] = p[0];
      v[k][1] = p[kNext];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i0 + k >= pieces) continue;
      const float w = weight[r][i0 + k];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        o[x].x = fmaf(v[k][x].x, w, o[x].x), o[x].y = fmaf(v[k][x].y, w, o[x].y);
        o[x].z = fmaf(v[k][x].z, w, o[x].z), o[x].w = fmaf(v[k][x].w, w, o[x].w);
      }
    }
  }
  const float M = whole[r].x, l = whole[r].y;
  const int64_t orow = (j.rows0 + j.node0 + row / a.head_box) * a.heads + j.head0 + row % a.head_box;
  const bool none = l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
  T *out = static_cast<T *>(a.out) + orow * kRank + 4 * e;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t lo = pack2(none ? 0.f : o[x].x * inv, none ? 0.f : o[x].y * inv, T());
    const uint32_t hi = pack2(none ? 0.f : o[x].z * inv, none ? 0.f : o[x].w * inv, T());
    *reinterpret_cast<uint2 *>(out + 4 * e_step * x) = make_uint2(lo, hi);
  }
  if (e == 0 && a.lse) a.lse[orow] = none ? -CUDART_INF_F : (M + log2f(l)) * 0.69314718055994530942f;
}

}  // namespace latent
}  // namespace b200kv
