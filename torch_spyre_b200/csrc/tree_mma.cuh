// Tensor-core kernel of tree attention (tree_attention.cu has the operator).
//
// Rows: the nodes of a sequence and the G = Hq / Hkv query heads of a KV head
// are the rows of one matrix (node-major, so row = node * G + head), cut into Q
// tiles of floor(128 / G) nodes.  Two consecutive Q tiles of the same sequence
// and KV head form a block; a block's cached tokens are cut into tiles of 128
// (two pages).  The blocks' tiles, all sequences and KV heads one after the
// other, form one line that is cut into equal shares, one per CTA; a block cut
// by a share's end is joined by tree_join_kernel.
//
// Inside a CTA two streams run side by side, each with its own warpgroup, score
// buffer S and accumulator O in TMEM.  A block of two Q tiles gives each stream
// one of them, both over every token tile; a block of one Q tile (the usual
// draft) gives the streams alternate token tiles, and their two states are
// merged when the block ends.  Per tile: S = Q K^T (tcgen05.mma, fp32), the
// warpgroup (thread = row) masks and exponentiates, P goes back into S's TMEM
// columns in 16 bits, O += P V with P as the TMEM operand.  While one stream's
// warpgroup works on its scores the tensor pipe works for the other.  O is only
// rescaled when a row's maximum has risen by more than 2^8 (weights then stay
// below 2^8, far from fp16's range), so most tiles touch it in the MMA alone.
//
// Bound, 16-bit caches: with up to 128 rows a 128-token tile costs the tensor pipe
// 0.55 us (2 x 128^3 products at 8192 FLOP per clock) and HBM 1.5 us per SM, so
// drafts run at the cache's bandwidth (4 sequences of 118k tokens, 16 nodes, 32/8
// heads, fp16, 1.93 GB: 288 to 303 us, the copy rate would be 300); short ones by
// what a piece costs besides its steps (16 sequences of 4.3k tokens and up to 64
// nodes, bf16, 295 MB: 75 us, the copy rate would be 46).  Blocks of two Q tiles are bound by the tensor pipe and
// the exponentials (16 per clock and SM, as long as the products), which follow
// one another within a stream: two prompts' chunks of 1024 tokens over 8.1k, 64/8
// heads, 578 GFLOP: 528 us, 0.64 of the matrix rate.
//
// 8-bit caches: widening (2 x 16 KB a tile), softmax and products take 0.6 to 0.7
// us a tile and SM each and are a chain with handshakes, which 3 raw and 4
// operand tiles let overlap in part only: 1.7 us a tile, 4 sequences of 118k
// tokens, 1.0 GB: 325 us over int8, 324 over e4m3.  Without widening 0.88 of that, without softmax 0.77,
// without products 0.92.  More than 128 rows: every Q tile widens the tile
// again.  (Tried: two Q tiles a block with three operand tiles, 0.93 of the time
// with all blocks full but 1.08 with ragged drafts; widening by 16 warps in two
// groups, 1.2; by two groups of four, one for K and one for V, 1.1; scores in
// matrix fragments, a quarter of the factors' reads, 1.0.)
//
// Warps: 0-3 and 4-7 the two softmax warpgroups, 8 the TMA producer, 9 the MMA
// issuer (owns the TMEM), 8-bit caches: 12-19 converters, which turn 8-bit
// pages into 16-bit operand tiles of exact steps (the scales: see Factors).
#pragma once

#include <type_traits>

#include "tree_attention.h"
#include "umma.cuh"

namespace b200kv {
namespace tree {

using namespace umma;

constexpr int kTileRows = 128, kTileTokens = 128;
constexpr float kLazyLog2 = 8.f;

template <typename T, int D, int kCache>
struct Cfg {
  static constexpr bool k8 = kCache != B200KV_F16;
  static constexpr int kThreads = k8 ? 640 : 384;
  // Registers a thread, softmax / issue / converter warpgroups, after
  // setmaxnreg (a 16-bit cache's softmax thread holds its row's 128 scores).
  // Sums within the launch's own: 384 threads of 168, or 640 of 96.
  static constexpr int kRegsSoftmax = k8 ? 144 : 208, kRegsIssue = k8 ? 64 : 80, kRegsConvert = 64;
  static constexpr int kConverters = 8;  // warps
  static constexpr int kSticks = D / 64;
  static constexpr int kStickTile = kTileTokens * 128;      // one 64-element column of 128 rows
  static constexpr int kTile = kSticks * kStickTile;        // a Q, K or V tile
  static constexpr int kQ = k8 ? 1 : 2;                      // most Q tiles of a block
  static constexpr int kSlots = k8 ? 4 : (D == 64 ? 8 : 5);  // operand tiles in flight
  static constexpr int kRaw = k8 ? 3 : 0;                    // 8-bit tiles in flight
  static constexpr int kRawTile = kTileTokens * 128;
  static constexpr int kCtrl = k8 ? 19456 : 3072;
  static constexpr int kOffQ = kCtrl;
  static constexpr int kOffSlots = kOffQ + kQ * kTile;
  static constexpr int kOffRaw = kOffSlots + kSlots * kTile;
  static constexpr int kSmem = kOffRaw + kRaw * kRawTile;
  // The type of P and V: an 8-bit cache's steps are exact in fp16, whatever q's
  // type, and fp16 keeps three bits more of each weight than bf16.
  using P = typename std::conditional<k8, __half, T>::type;
  // kind::f16: fp32 accumulator, A and B both fp16 or both bf16, M = 128
  static constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(kTileRows >> 4) << 24);
  static constexpr uint32_t kBf16 = (1u << 7) | (1u << 10);
  static constexpr uint32_t kIdescQK =
      kIdesc | (std::is_same<T, __half>::value ? 0u : kBf16) | (uint32_t(kTileTokens >> 3) << 17);
  static constexpr uint32_t kIdescPV =  // V: N-major
      kIdesc | (std::is_same<P, __half>::value ? 0u : kBf16) | (1u << 16) | (uint32_t(D >> 3) << 17);
  static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

// TMEM columns
constexpr uint32_t kTmemCols = 512;
__device__ __forceinline__ uint32_t col_s(int w) { return uint32_t(w) * 128u; }
__device__ __forceinline__ uint32_t col_o(int w) { return 256u + uint32_t(w) * 128u; }

struct Seq {
  int ctx, nodes, q0, blocks, qtiles;
  int end;  // the first row of q that is a later sequence's
};
// Where a CTA's share of the line begins: in block `block`, whose units begin at
// unit u0 of the line.
struct Start {
  Seq s;
  int b, kvh, block, u0;
};

struct Ctrl {
  uint64_t full[8], empty[8];          // operand tiles
  uint64_t raw_full[8], raw_empty[8];  // 8-bit tiles
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_ready[2], o_full[2];
  uint32_t tmem;
  int per, total;  // units of a share, of the line
  Start start;
  int scan[32];
  unsigned bad_piece;       // last piece (counted from 1) that met a non-finite value in a node's V row
  float2 ml[2][kTileRows];  // (maximum, sum) of the streams' rows
  float unit[2][4];         // 8-bit caches: what O counts in (see Factors), by stream and warp
  unsigned spoilt_piece;    // last piece (counted from 1) that met a V scale that is not finite
};
// 8-bit caches: [8 warps][3][128] factors of a tile's tokens (see Factors), or,
// when a block ends, [2 warpgroups][4][128] float4 of its rows' copies
constexpr int kOffFactors = 3072;
static_assert(sizeof(Ctrl) <= kOffFactors, "control block");

__device__ __forceinline__ void bar_group(int w) {  // one warpgroup
  if (w == 0)
    asm volatile("bar.sync 2, 128;" ::: "memory");
  else
    asm volatile("bar.sync 3, 128;" ::: "memory");
}
__device__ __forceinline__ void bar_pair() { asm volatile("bar.sync 1, 256;" ::: "memory"); }  // both warpgroups

// ---------------------------------------------------------------- operands --
// 128-byte swizzle, descriptor version 1.  K-major (Q, K): rows of 128 bytes,
// groups of 8 rows 1024 bytes apart.  N-major (V): 64 head elements of a token
// are 128 contiguous bytes; groups of 8 tokens 1024 bytes apart, the next 64
// elements one stick column (128 tokens) on.
__device__ __forceinline__ uint32_t desc_nmajor(uint32_t addr) {
  return (addr >> 4) | (uint32_t((kTileTokens * 128) >> 4) << 16);
}
// -------------------------------------------------------------------- plan --
template <int kQ>
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
  s.qtiles = (s.nodes + a.tile_nodes - 1) / a.tile_nodes;
  s.blocks = (s.qtiles + kQ - 1) / kQ;
  return s;
}
// Token tiles of block k: what its last node can see.
template <int kQ>
__device__ __forceinline__ int block_tiles(const Args &a, const Seq &s, int k) {
  const int nodes = a.mask ? s.nodes : min(s.nodes, (k + 1) * kQ * a.tile_nodes);
  return (s.ctx + nodes + kTileTokens - 1) / kTileTokens;
}
// The line is cut by cost, in units of half a microsecond: a step over a token
// tile takes 1.1 us with one Q tile and 2.05 with two, and a block begins with
// what every piece costs besides its steps (Q, the first products, the epilogue),
// 5 and 7 us (least squares over the CTAs' times of eight batches of 1 to 16
// sequences over 16-bit caches; they are within 1 to 2 us of it).  8-bit caches are
// cut by the same weights, although their steps take 1.75 to 2.4 us and their pieces
// 10 to 14.
template <int kQ>
__device__ __forceinline__ bool two_tiles(const Seq &s, int k) {
  return kQ == 2 && 2 * k + 1 < s.qtiles;
}
template <int kQ>
__device__ __forceinline__ int step_units(const Seq &s, int k) {
  return two_tiles<kQ>(s, k) ? 4 : 2;
}
template <int kQ>
__device__ __forceinline__ int begin_units(const Seq &s, int k) {
  return two_tiles<kQ>(s, k) ? 13 : 9;
}
template <int kQ>
__device__ __forceinline__ int block_units(const Args &a, const Seq &s, int k) {
  return begin_units<kQ>(s, k) + step_units<kQ>(s, k) * block_tiles<kQ>(a, s, k);
}
template <int kQ>
__device__ __forceinline__ int head_units(const Args &a, const Seq &s) {
  if (s.blocks == 0) return 0;
  // with a mask all blocks have as many tiles, and only the last may be of one Q tile
  if (a.mask) return (s.blocks - 1) * block_units<kQ>(a, s, 0) + block_units<kQ>(a, s, s.blocks - 1);
  int n = 0;
  for (int k = 0; k < s.blocks; ++k) n += block_units<kQ>(a, s, k);
  return n;
}

// An 8-bit cache's Q tile holds its rows several times where they are few: 4
// times up to 32 rows, twice up to 64.  Every copy meets all tokens in the
// products, but weighs only its share of them (the rest get zeros), so that all
// four warps of a warpgroup work on a tile and a thread takes 32 or 64 scores
// of it.  The copies are separate states of the softmax until the block ends.
struct Copies {
  int copies, rows, boxes;  // rows: of the tile, per copy; boxes: TMA boxes of a copy
};
__device__ __forceinline__ Copies copies_of(const Args &a, const Seq &s, int block) {
  const int live = min(a.tile_nodes, s.nodes - block * a.tile_nodes) * a.group;
  Copies c;
  c.boxes = a.small_boxes ? (live + 31) / 32 : 1;
  const int held = a.small_boxes ? c.boxes * 32 : a.box_nodes * a.group;
  c.copies = held <= 32 ? 4 : (held <= 64 ? 2 : 1);
  c.rows = kTileRows / c.copies;
  return c;
}

// The blocks of a CTA's share, one piece (a block, or the part of it in this
// share) at a time.  Every role walks the same sequence.
template <int kQ>
struct Walk {
  Seq s;
  int b, kvh, block, u0, tiles, t0, t1;  // piece: token tiles [t0, t1) of `tiles`
  int end;                               // of the share

  __device__ __forceinline__ void init(const Ctrl &c) {
    const Start &f = c.start;
    s = f.s, b = f.b, kvh = f.kvh, block = f.block, u0 = f.u0;
    t1 = 0;
    end = min(c.total, (static_cast<int>(blockIdx.x) + 1) * c.per);
  }
  // Tile t belongs to the share that holds its first unit.
  __device__ __forceinline__ int tile_from(int unit) const {
    const int w = step_units<kQ>(s, block), x = unit - u0 - begin_units<kQ>(s, block);
    return x <= 0 ? 0 : min(tiles, (x + w - 1) / w);
  }
  // The next piece, false when the share is done.
  __device__ __forceinline__ bool next(const Args &a, const Ctrl &c) {
    const int first = static_cast<int>(blockIdx.x) * c.per;
    for (;;) {
      if (u0 >= end || first >= c.total) return false;
      tiles = block_tiles<kQ>(a, s, block);
      t0 = tile_from(first);
      t1 = tile_from(end);
      if (t0 < t1) return true;
      advance(a);
    }
  }
  __device__ __forceinline__ void advance(const Args &a) {
    u0 += block_units<kQ>(a, s, block);
    if (u0 >= end) return;
    if (++block >= s.blocks) {
      block = 0;
      if (++kvh >= a.hkv) {
        kvh = 0;
        do s = load_seq<kQ>(a, ++b, false);
        while (s.nodes == 0);
      }
    }
  }
  __device__ __forceinline__ bool two() const { return two_tiles<kQ>(s, block); }
  // The share that holds the first unit of tile t.
  __device__ __forceinline__ int share_of(int t, int per) const {
    return (u0 + begin_units<kQ>(s, block) + t * step_units<kQ>(s, block)) / per;
  }
};

// Rows of q that no sequence has (all of them flagged): before the first
// sequence's, past a sequence's nodes as they were clamped, after the last's.
// They see nothing.  Every CTA takes some.  `all`: no row has a sequence.
template <typename T, int D, int kQ>
__device__ __noinline__ void clear_rows(const Args &a, bool all) {
  for (int b = 0; b < a.batch; ++b) {
    const Seq s = load_seq<kQ>(a, b, false);
    const int first = b == 0 ? 0 : s.q0, end = all ? (b == 0 ? a.total_q : 0) : s.end;
    for (int t = first + blockIdx.x; t < end; t += gridDim.x) {
      if (!all && t >= s.q0 && t < s.q0 + s.nodes) continue;
      uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + static_cast<int64_t>(t) * a.hq * D);
      for (int i = threadIdx.x; i < a.hq * (D / 8); i += blockDim.x) out[i] = make_uint4(0, 0, 0, 0);
      if (!a.lse) continue;
      for (int h = threadIdx.x; h < a.hq; h += blockDim.x) a.lse[static_cast<int64_t>(t) * a.hq + h] = -CUDART_INF_F;
    }
  }
}

// The line's length, a share's, and where this CTA's begins; all threads of the
// CTA call it, a barrier follows.  The counts fit 31 bits (the host checks) where
// no two sequences have the same row: a q_indptr that descends could make them
// anything, so then nothing has a sequence.
template <typename T, int D, int kThreads, int kQ>
__device__ __forceinline__ void make_plan(const Args &a, Ctrl &c) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.batch + kThreads - 1) / kThreads;
  const int b0 = tid * each, b1 = min(b0 + each, a.batch);
  Seq s{};
  int mine = 0;
  bool unclaimed = false, descends = false;
  for (int b = b0; b < b1; ++b) {
    s = load_seq<kQ>(a, b, blockIdx.x == 0);
    mine += head_units<kQ>(a, s) * a.hkv;
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
    clear_rows<T, D, kQ>(a, none);
  }
  int total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += c.scan[w];
    total += c.scan[w];
  }
  if (none) total = mine = 0;
  // (at least a step, so that a share inside a block holds the start of a tile)
  const int per = max(4, static_cast<int>((static_cast<unsigned>(total) + gridDim.x - 1) / gridDim.x));
  const int first = static_cast<int>(blockIdx.x) * per;
  int at = before + incl - mine;
  if (first >= at && first < at + mine) {
    int b = b0, hu = 0;
    for (;; ++b) {
      if (each > 1) s = load_seq<kQ>(a, b, false);
      hu = head_units<kQ>(a, s);
      if (first < at + hu * a.hkv) break;
      at += hu * a.hkv;
    }
    const int kvh = (first - at) / hu;
    at += kvh * hu;
    int block = 0;
    if (a.mask) {
      const int n = block_units<kQ>(a, s, 0);
      block = min((first - at) / n, s.blocks - 1);
      at += block * n;
    } else {
      for (int n; first >= at + (n = block_units<kQ>(a, s, block)); ++block) at += n;
    }
    c.start = Start{s, b, kvh, block, at};
  }
  if (tid == 0) {
    c.per = per;
    c.total = total;
  }
}

// Page ids of a sequence, 32 at a time in a warp's lanes.  Invalid ids are
// flagged and become -1.
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

// The pages of a raw tile that are not among `valid`; the whole warp calls it.
static __device__ __noinline__ void zero_pages(uint8_t *tile, uint32_t valid) {
  uint4 *at = reinterpret_cast<uint4 *>(tile);
  for (int i = threadIdx.x & 31; i < 2 * kPageTokens * 8; i += 32)
    if (!(valid >> (i / (kPageTokens * 8)) & 1u)) at[i] = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

// ------------------------------------------------------------------ roles --
// Waits, with a limit, for the copies that are under way: the last of `issued` tiles and Q of the last piece.
template <typename C>
__device__ __noinline__ void drain(const Args &a, Ctrl &c, uint32_t issued, uint32_t pieces) {
  bool late = false;
  if (pieces > 0) wait(&c.q_full, (pieces - 1) & 1u, late, a.error_flag);
  constexpr uint32_t kDepth = C::k8 ? C::kRaw : C::kSlots;
  for (uint32_t n = issued - min(issued, kDepth); n < issued; ++n)
    wait(C::k8 ? &c.raw_full[n % kDepth] : &c.full[n % kDepth], (n / kDepth) & 1u, late, a.error_flag);
}

template <typename C>
__device__ __forceinline__ void producer(const Args &a, Ctrl &c, uint8_t *smem, const CUtensorMap *qm,
                                         const CUtensorMap *km, const CUtensorMap *vm) {
  const int lane = threadIdx.x & 31;
  // Pages are read once and leave L2 first, unless more than two blocks read them
  // (two prompts' chunks of 1024 tokens: 582 us, 528 with the plain policy; with
  // two blocks, drafts up to 64 nodes of 64/8 heads, 116 and 118).
  const uint64_t policy_once = l2_policy_evict_first();
  uint64_t policy_again;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy_again));
  bool dead = false;
  uint32_t slot = 0, ring = 0, pieces = 0;  // tiles issued (16-bit, 8-bit), pieces begun
  Walk<C::kQ> w;
  w.init(c);
  while (w.next(a, c)) {
    const bool two = w.two();
    const uint64_t policy = w.s.blocks > 2 ? policy_again : policy_once;
    const int pages = (w.s.ctx + w.s.nodes + kPageTokens - 1) / kPageTokens;
    int window = w.t0 / 16, ids = load_ids(a, w.b, window, pages), ids_next = load_ids(a, w.b, window + 1, pages);
    wait(&c.q_empty, (pieces & 1u) ^ 1u, dead, a.error_flag);
    dead = __any_sync(0xffffffffu, dead);
    if (dead) break;
    // lane: a box of Q (16-bit pools: of one or two Q tiles; 8-bit: of the
    // tile's copies) and stick column
    const int st = lane % C::kSticks, box = lane / C::kSticks;
    if constexpr (C::k8) {
      const Copies q = copies_of(a, w.s, w.block);
      const int n = q.copies * q.boxes, k = box / q.boxes, i = box - k * q.boxes;
      if (lane == 0) mbar_arrive_expect_tx(&c.q_full, uint32_t(n) * C::kSticks * a.q_box_bytes);
      __syncwarp();
      if (box < n)
        tma_3d(smem + C::kOffQ + st * C::kStickTile + (k * q.rows + i * 32) * 128, qm, &c.q_full, st * 64,
               w.kvh * a.group, w.s.q0 + w.block * a.tile_nodes + i * a.box_nodes);
    } else {
      const int n = two ? 2 : 1;
      if (lane == 0) mbar_arrive_expect_tx(&c.q_full, uint32_t(n) * C::kSticks * a.q_box_bytes);
      __syncwarp();
      if (box < n)
        tma_3d(smem + C::kOffQ + box * C::kTile + st * C::kStickTile, qm, &c.q_full, st * 64, w.kvh * a.group,
               w.s.q0 + (C::kQ * w.block + box) * a.tile_nodes);
    }
    ++pieces;
    int ids_before = ids;
    auto issue = [&](bool is_v, int t) {
      if (dead) return;
      if (t / 16 > window) {  // K leads, V follows by at most two tiles
        ids_before = ids;
        ids = ids_next;
        ids_next = load_ids(a, w.b, ++window + 1, pages);
      }
      // lane: a page of the tile and, in 16-bit pools, one of its stick columns
      constexpr int kParts = C::k8 ? 1 : C::kSticks;
      const int have = t / 16 == window ? ids : ids_before;
      const int part = lane % kParts, at = lane / kParts;
      const int id = __shfl_sync(0xffffffffu, have, (2 * t + (at & 1)) & 31);
      const int n = min(2, pages - 2 * t);
      if constexpr (!C::k8) {
        const uint32_t s = slot % C::kSlots;
        wait(&c.empty[s], ((slot / C::kSlots) & 1u) ^ 1u, dead, a.error_flag);
        if (lane == 0) mbar_arrive_expect_tx(&c.full[s], uint32_t(n) * C::kSticks * (kPageTokens * 128));
        if ((dead = __any_sync(0xffffffffu, dead))) return;
        // an invalid id reads past the last page: zeros
        const int page = id < 0 ? a.num_blocks * a.hkv : id * a.hkv + w.kvh;
        if (at < n)
          tma_load_3d(smem + C::kOffSlots + s * C::kTile + part * C::kStickTile + at * (kPageTokens * 128), is_v ? vm : km,
                      &c.full[s], 0, part * kPageTokens, page, policy);
        ++slot;
      } else {
        const uint32_t r = ring % C::kRaw;
        wait(&c.raw_empty[r], ((ring / C::kRaw) & 1u) ^ 1u, dead, a.error_flag);
        // a page is one contiguous run; one with an invalid id is written as zeros
        const uint32_t valid = __ballot_sync(0xffffffffu, at < n && id >= 0);
        if (valid != (1u << n) - 1u) zero_pages(smem + C::kOffRaw + r * C::kRawTile, valid);
        if (lane == 0) mbar_arrive_expect_tx(&c.raw_full[r], __popc(valid) * (kPageTokens * 128));
        if ((dead = __any_sync(0xffffffffu, dead))) return;
        const int64_t page = id * a.hkv + w.kvh;
        if (at < n && id >= 0)
          bulk_load(smem + C::kOffRaw + r * C::kRawTile + at * (kPageTokens * 128),
                    static_cast<const uint8_t *>(is_v ? a.v_pool : a.k_pool) + page * (kPageTokens * 128),
                    kPageTokens * 128, &c.raw_full[r]);
        ++ring;
      }
    };
    // K leads V by one tile per stream that needs it: the order the MMA warp
    // consumes them in
    const int lead = two ? 1 : 2;
    for (int t = w.t0; t < min(w.t0 + lead, w.t1); ++t) issue(false, t);
    for (int t = w.t0; t < w.t1; ++t) {
      issue(true, t);
      if (t + lead < w.t1) issue(false, t + lead);
    }
    w.advance(a);
  }
  if (dead) drain<C>(a, c, C::k8 ? ring : slot, pieces);
  // the last arrival that the MMAs owe this CTA: not before it may the CTA end
  if (lane == 0 && pieces > 0) {
    bool late = false;
    wait(&c.q_empty, (pieces & 1u) ^ 1u, late, a.error_flag);
  }
  __syncwarp();
}

// Non-finite values of drafted nodes.  A weight of zero does not keep an inf or
// NaN of V out of a matrix product, and a node may be hidden from some rows of
// a tile only.  So the nodes' V rows are looked through in shared memory:
// non-finite elements become zeros there, and when the block ends the rows that
// see such a node get its elements added from the cache (repair_row).
// Eight-bit pages -> operand tiles.  A lane takes 16 bytes of a row and writes
// the two 16-byte vectors they become.  Lanes 0-3 of eight take the first half
// of row r, lanes 4-7 the second half of row r ^ 1: the swizzle then puts the
// eight vectors of a store on eight different bank groups, as it does the reads.
//
// Every step is exact in the operand type.  int8 -> fp16: 0x64xx is 1024 + xx,
// taken as b + 128, less 1152.  int8 -> bf16: b = (b & 127) - (b & 128), both
// over 128 as 0x43xx.  e4m3 -> fp16 in hardware, two at a time into the register
// that holds them (put together from two 16-bit halves they cost 1.4 times the
// kernel), on to bf16 by way of fp32, of whose mantissa at most three bits are set.
template <typename T, int kCache>
__device__ __forceinline__ void widen16(uint4 v, uint4 &lo, uint4 &hi) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t &r = o[2 * i + k];
      if constexpr (kCache == B200KV_I8 && kHalf) {
        const uint32_t u = __byte_perm(w[i] ^ 0x80808080u, 0x64646464u, k ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));
        r = *reinterpret_cast<const uint32_t *>(&h);
      } else if constexpr (kCache == B200KV_I8) {
        const uint32_t u = __byte_perm(w[i], 0u, k ? 0x4342 : 0x4140);
        const uint32_t a = (u & 0x007f007fu) | 0x43004300u, b = (u & 0x00800080u) | 0x43004300u;
        const __nv_bfloat162 h =
            __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
        r = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        if (k == 0)
          asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w[i]));
        else
          asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w[i]));
        if constexpr (!kHalf) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
          r = __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
        }
      }
    }
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

template <typename C, typename T, int kCache>
__device__ __forceinline__ void converter(const Args &a, Ctrl &c, uint8_t *smem, int warp) {
  const int lane = threadIdx.x & 31, sub = lane & 7;
  // this lane's rows of a tile are row0, row0 + 32, + 64 and + 96
  const int row0 = warp * 4 + ((lane >> 3) ^ (sub >> 2));
  const int chunk = (sub & 3) * 2;
  const uint32_t from = row0 * 128 + sub * 16;
  const uint32_t even = (sub >> 2) * C::kStickTile + row0 * 128, at0 = (chunk ^ (row0 & 7)) << 4;
  bool dead = false;
  uint32_t slot = 0, ring = 0;
  unsigned piece = 0;
  // one tile of K (To the compute type) or V (to fp16)
  auto tile = [&](auto to, bool is_v, int t, int len, int ctx) {
    using To = decltype(to);
    const uint32_t s = slot % C::kSlots;
    wait(&c.empty[s], ((slot / C::kSlots) & 1u) ^ 1u, dead, a.error_flag);
    uint8_t *dst = smem + C::kOffSlots + s * C::kTile + even;
    const uint32_t r = ring % C::kRaw;
    wait(&c.raw_full[r], (ring / C::kRaw) & 1u, dead, a.error_flag);
    const uint8_t *src = smem + C::kOffRaw + r * C::kRawTile + from;
    const int rows = len - t * kTileTokens;  // those from the sequence's end on become zeros
    uint4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      x[k] = row0 + 32 * k < rows ? *reinterpret_cast<const uint4 *>(src + k * 4096) : make_uint4(0, 0, 0, 0);
    ++ring;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 lo, hi;
      widen16<To, kCache>(x[k], lo, hi);
      if (kCache == B200KV_E4M3 && is_v && t * kTileTokens + row0 + 32 * k >= ctx) {  // a node's row: e4m3 has NaN
        const bool hit = drop_non_finite<__half>(lo);
        if (drop_non_finite<__half>(hi) || hit) atomicMax(&c.bad_piece, piece);
      }
      *reinterpret_cast<uint4 *>(dst + k * 4096 + at0) = lo;
      *reinterpret_cast<uint4 *>(dst + k * 4096 + (at0 ^ 16)) = hi;
    }
    fence_async_smem();
    __syncwarp();
    // The raw tile is released here and not right after its loads: an arrival
    // can overtake shared-memory loads whose values nothing has used yet, and
    // the next bulk copy then overwrites what they were to read.
    if (lane == 0) arrive(&c.raw_empty[r]);
    if (lane == 0) arrive(&c.full[s]);
    ++slot;
  };
  Walk<C::kQ> w;
  w.init(c);
  while (w.next(a, c)) {
    ++piece;
    const int len = w.s.ctx + w.s.nodes;
    const int lead = w.two() ? 1 : 2;
    for (int t = w.t0; t < min(w.t0 + lead, w.t1); ++t) tile(T(), false, t, len, w.s.ctx);
    for (int t = w.t0; t < w.t1; ++t) {
      tile(__half(), true, t, len, w.s.ctx);
      if (t + lead < w.t1) tile(T(), false, t + lead, len, w.s.ctx);
    }
    w.advance(a);
  }
}

// One warp, converged, issues every MMA from an elected lane.
template <typename C, int D>
__device__ __forceinline__ void mma_issuer(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem_any) {
  bool dead = false;
  uint32_t slot = 0, pieces = 0, p_uses[2] = {0, 0};
  const uint32_t go = elect_one(), tmem = uniform(tmem_any);
  const uint32_t qbase = smem_u32(smem + C::kOffQ), sbase = smem_u32(smem + C::kOffSlots);
  const uint32_t negate = a.scale < 0.f ? 1u << 13 : 0u;  // a negative scale turns Q's sign
  auto done = [&](uint64_t *bar) {
    if (go) commit(bar);
  };
  auto ready = [&](uint32_t n) {
    wait(&c.full[n % C::kSlots], (n / C::kSlots) & 1u, dead, a.error_flag);
    fence_after();
    return uniform(sbase + (n % C::kSlots) * C::kTile);
  };
  auto qk = [&](int w, int qtile, uint32_t k) {
    const uint32_t qd = desc_kmajor(qbase + qtile * C::kTile), kd = desc_kmajor(k);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint32_t off = ((i >> 2) * C::kStickTile + (i & 3) * 32) >> 4;
      mma_ss(tmem + col_s(w), qd + off, kd + off, C::kIdescQK | negate, i > 0, go);
    }
    done(&c.s_full[w]);
  };
  auto pv = [&](int w, uint32_t v, bool first) {
    wait(&c.p_ready[w], p_uses[w]++ & 1u, dead, a.error_flag);
    fence_after();
    const uint32_t vd = desc_nmajor(v);
#pragma unroll
    for (int i = 0; i < kTileTokens / 16; ++i)
      mma_ts(tmem + col_o(w), tmem + col_s(w) + i * 8, vd + (i * 2048 >> 4), C::kIdescPV, !first || i > 0, go);
  };
  Walk<C::kQ> w;
  w.init(c);
  while (w.next(a, c)) {
    wait(&c.q_full, pieces++ & 1u, dead, a.error_flag);
    fence_after();
    const int n = w.t1 - w.t0;
    if (w.two()) {
      // both streams over every tile; a slot is free when the second has used it
      uint32_t k = ready(slot);
      qk(0, 0, k);
      qk(1, 1, k);
      done(&c.empty[slot++ % C::kSlots]);
      for (int t = 0; t < n; ++t) {
        const uint32_t vs = slot++, v = ready(vs);
        const bool more = t + 1 < n;
        pv(0, v, t == 0);
        if (more)
          qk(0, 0, k = ready(slot));
        else
          done(&c.o_full[0]);
        pv(1, v, t == 0);
        done(&c.empty[vs % C::kSlots]);
        if (more) {
          qk(1, 1, k);
          done(&c.empty[slot++ % C::kSlots]);
        } else {
          done(&c.o_full[1]);
        }
      }
    } else {
      // stream t & 1 takes tile t
      auto pair = [&](int w0, int t) {
        pv(w0, ready(slot), t < 2);
        done(&c.empty[slot++ % C::kSlots]);
        if (t + 2 < n) {
          qk(w0, 0, ready(slot));
          done(&c.empty[slot++ % C::kSlots]);
        } else {
          done(&c.o_full[w0]);
        }
      };
      qk(0, 0, ready(slot));
      done(&c.empty[slot++ % C::kSlots]);
      if (n > 1) {
        qk(1, 0, ready(slot));
        done(&c.empty[slot++ % C::kSlots]);
      }
      for (int t = 0; t < n; t += 2) {
        pair(0, t);
        if (t + 1 < n) pair(1, t + 1);
      }
    }
    done(&c.q_empty);
    w.advance(a);
  }
  __syncwarp();
}

// Which of the tokens pos .. pos + 31 row `node` sees.
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

// Per-token factors of an 8-bit cache.  The scales leave the products: K and V
// enter them as exact steps, and the weight that V's steps get is
//   p v = 2^(k_factor s + log2 v) = 2^y,   y = s * (scale * log2(e) * k) + log2 v,
// so the running maximum is that of y, and the softmax's own sum takes 2^y / v.
// Scales may be any normal number, and 2^y / v has to stay one: v is taken in
// units of a power of two, so O counts in it too, and m and l do not depend on it.
// The unit is 1 if the scales of a warp's first tile are within 2^-20 .. 2^30 (no
// tile of such a cache needs more than a look at its scales), else the power of the
// largest of them, and follows when scales 2^30 times as large come up (O with it).
// In that unit
//   a row of zeros (v = 0) weighs in the sum alone: v = 2^-60, small enough not
//     to move the maximum and large enough for 2^(y - m) to stay normal for
//     whatever matters in the sum;
//   others below 2^-90 count as that, next to rows more than 2^70 times their size.
struct Factors {
  float4 k[kTileTokens / 4], log2v[kTileTokens / 4], inv_v[kTileTokens / 4];
};
constexpr uint32_t kExp = 1u << 23;  // of a float's exponent
constexpr uint32_t kMostUnits = 157u * kExp, kLeastUnits = 37u * kExp, kLeastFirst = 107u * kExp;  // 2^30, 2^-90, 2^-20
__device__ __forceinline__ float inverse_of_power(float x) { return __uint_as_float(254u * kExp - __float_as_uint(x)); }
// Whether a lane's four scales, in units, are positive numbers within the bounds
// (compared as integers: NaN, inf and negative numbers are above all others).
__device__ __forceinline__ bool ordinary(float4 u, uint32_t least) {
  const uint32_t x = __float_as_uint(u.x), y = __float_as_uint(u.y), z = __float_as_uint(u.z), w = __float_as_uint(u.w);
  return max(max(x, y), max(z, w)) <= kMostUnits && min(min(x, y), min(z, w)) >= least;
}
__device__ __forceinline__ void put_v(Factors *fac, float4 u) {
  const int lane = threadIdx.x & 31;
  fac->log2v[lane] = make_float4(__log2f(u.x), __log2f(u.y), __log2f(u.z), __log2f(u.w));
  fac->inv_v[lane] = make_float4(__fdividef(1.f, u.x), __fdividef(1.f, u.y), __fdividef(1.f, u.z), __fdividef(1.f, u.w));
}
// V's factors of a tile whose scales are not all ordinary in units of 1 / per, four
// to a lane (`have`: so many of them are of the sequence's rows).  Returns 1 / unit
// from this tile on, 0 as long as all rows were zero.
// A scale that is not finite makes NaN of whoever sees its row (see sees_spoilt), but
// not of the sums, which go by K alone: the row weighs as one of zeros.
static __device__ __noinline__ float odd_scales(Factors *fac, float4 v, int have, float per, unsigned piece,
                                                unsigned *spoilt_piece) {
  const int lane = threadIdx.x & 31;
  auto of = [&](float x, int i) { return i < have && x > 0.f && x < CUDART_INF_F ? x : 0.f; };
  const float mine = fmaxf(fmaxf(of(v.x, 0), of(v.y, 1)), fmaxf(of(v.z, 2), of(v.w, 3)));
  const uint32_t largest = __reduce_max_sync(0xffffffffu, __float_as_uint(mine));
  if (largest != 0 && (per == 0.f || __uint_as_float(largest) * per > __uint_as_float(kMostUnits)))
    // (bounds that keep a row's sum and its inverse, times the unit, normal)
    per = inverse_of_power(__uint_as_float(min(max(largest & (255u * kExp), 27u * kExp), 217u * kExp)));  // 2^-100, 2^90
  auto in_units = [&](float x) {
    const float u = x * (per == 0.f ? 1.f : per);
    return x == 0.f || !(x < CUDART_INF_F) ? 8.67361738e-19f : u < __uint_as_float(kLeastUnits) ? __uint_as_float(kLeastUnits) : u;
  };
  put_v(fac, make_float4(in_units(v.x), in_units(v.y), in_units(v.z), in_units(v.w)));
  auto spoilt = [&](float x, int i) { return i < have && !(x < CUDART_INF_F); };
  if (spoilt(v.x, 0) || spoilt(v.y, 1) || spoilt(v.z, 2) || spoilt(v.w, 3)) *spoilt_piece = piece;
  return per;
}

// Moves the running maximum when a row's has risen far enough, O and l with it.
template <int D>
__device__ __forceinline__ void follow(uint32_t to, float mt, bool first, bool live, float &m, float &l) {
  const bool rise = mt > m + (first ? 0.f : kLazyLog2);
  if (!first && __any_sync(0xffffffffu, rise && live)) {
    const float keep = rise ? ex2(m - mt) : 1.f;
    l *= keep;
#pragma unroll 1
    for (int i = 0; i < D; i += 16) {
      uint32_t r[16];
      tmem_ld16(to + i, r);
      wait_ld(r);
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
      tmem_st16(to + i, r);
    }
  }
  if (rise) m = mt;
}

template <int D>
__device__ __noinline__ void rescale(uint32_t to, float by) {
#pragma unroll 1
  for (int i = 0; i < D; i += 16) {
    uint32_t r[16];
    tmem_ld16(to + i, r);
    wait_ld(r);
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * by);
    tmem_st16(to + i, r);
  }
  wait_st();
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

// Scores of a row's 128 tokens -> weights, in place in TMEM.  kTail: vis tells
// which tokens the row sees.
template <typename P, int D, bool kTail>
__device__ __forceinline__ void weigh(uint32_t ts, uint32_t to, const uint32_t (&vis)[4], float cl, bool first, bool live,
                                      float &m, float &l) {
  uint32_t s[4][32];
#pragma unroll
  for (int i = 0; i < 4; ++i) tmem_ld32(ts + 32 * i, s[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) wait_ld(s[i]);
  float top[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = mask_max<kTail>(s[i], vis[i]);
  follow<D>(to, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * cl, first, live, m, l);
  const float minus = m == -CUDART_INF_F ? 0.f : -m;
  float2 sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[i] = make_float2(0.f, 0.f);
    uint32_t p[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 x = make_float2(__uint_as_float(s[i][2 * j]), __uint_as_float(s[i][2 * j + 1]));
      const float2 y = fma2(x, make_float2(cl, cl), make_float2(minus, minus));
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      sum[i] = add2(sum[i], e);
      p[j] = pack2(e.x, e.y, P());
    }
    tmem_st16(ts + 16 * i, p);
  }
  const float2 t = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
  l += t.x + t.y;
  wait_st();
}

// The same for an 8-bit cache: the 32 * kN tokens that this copy of the row
// weighs, from token 32 * kN * copy on.
template <int kN, int D, bool kTail, typename Arrived>
__device__ __forceinline__ void weigh8(uint32_t ts, uint32_t to, const uint32_t (&vis)[4], const Factors *fac, int copy,
                                       Arrived arrived, bool first, bool live, float &m, float &l) {
  constexpr bool kKeep = kN <= 2;  // scores stay in registers (else they go back to TMEM for the second pass)
  const int c0 = copy * kN;
  uint32_t y[kKeep ? kN : 1][32];
  float mt = -CUDART_INF_F;
  // factors of 16 tokens are fetched together, the first before the scores are there
  const float4 *kf = fac->k + 8 * c0, *vf = fac->log2v + 8 * c0, *inv = fac->inv_v + 8 * c0;
  float4 k[4], v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) k[j] = kf[j], v[j] = vf[j];
  arrived();
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    uint32_t(&s)[32] = y[kKeep ? i : 0];
    tmem_ld32(ts + 32 * (c0 + i), s);
    wait_ld(s);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t *r = &s[16 * h + 4 * j];
        const float2 lo = fma2(make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])), make_float2(k[j].x, k[j].y),
                               make_float2(v[j].x, v[j].y));
        const float2 hi = fma2(make_float2(__uint_as_float(r[2]), __uint_as_float(r[3])), make_float2(k[j].z, k[j].w),
                               make_float2(v[j].z, v[j].w));
        r[0] = __float_as_uint(lo.x), r[1] = __float_as_uint(lo.y);
        r[2] = __float_as_uint(hi.x), r[3] = __float_as_uint(hi.y);
      }
      if (i < kN - 1 || h == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = kf[8 * i + 4 * h + 4 + j], v[j] = vf[8 * i + 4 * h + 4 + j];
      }
    }
    mt = fmaxf(mt, mask_max<kTail>(s, vis[i]));
    if (!kKeep) tmem_st32(ts + 32 * i, s);
  }
  if (!kKeep) wait_st();
  follow<D>(to, mt, first, live, m, l);
  const float minus = m == -CUDART_INF_F ? 0.f : -m;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    uint32_t(&s)[32] = y[kKeep ? i : 0];
    if (!kKeep) tmem_ld32(ts + 32 * i, s);
    if (!kKeep) wait_ld(s);
    uint32_t p[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 x = add2(make_float2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), make_float2(minus, minus));
      const float2 e = make_float2(ex2(x.x), ex2(x.y));
      const float4 f = inv[8 * i + j / 2];
      sum[j & 1] = fma2(e, j & 1 ? make_float2(f.z, f.w) : make_float2(f.x, f.y), sum[j & 1]);
      p[j] = pack2(e.x, e.y, __half());
    }
    tmem_st16(ts + 16 * (c0 + i), p);
  }
  if (kN < 4) {
    // the tokens of the other copies
    uint32_t zero[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) zero[j] = 0;
#pragma unroll
    for (int i = 1; i < 4 / kN; ++i)
#pragma unroll
      for (int k = 0; k < kN; ++k) tmem_st16(ts + 16 * (((copy + i) % (4 / kN)) * kN + k), zero);
  }
  const float2 t = add2(sum[0], sum[1]);
  l += t.x + t.y;
  wait_st();
}
template <int D, bool kTail, typename Arrived>
__device__ __forceinline__ void weigh8(uint32_t ts, uint32_t to, const uint32_t (&vis)[4], const Factors *fac, int copies,
                                       int copy, Arrived arrived, bool first, bool live, float &m, float &l) {
  if (copies == 4)
    weigh8<1, D, kTail>(ts, to, vis, fac, copy, arrived, first, live, m, l);
  else if (copies == 2)
    weigh8<2, D, kTail>(ts, to, vis, fac, copy, arrived, first, live, m, l);
  else
    weigh8<4, D, kTail>(ts, to, vis, fac, copy, arrived, first, live, m, l);
}

// Element d of a cached V row (8-bit caches: its steps).
template <typename T, int D, int kCache>
__device__ float cached_v(const Args &a, const void *pool, int id, int kvh, int row, int d) {
  constexpr int kStick = kCache == B200KV_F16 ? 64 : 128;
  const int64_t page = static_cast<int64_t>(id) * a.hkv + kvh;
  const int64_t at = (page * (D / kStick) + d / kStick) * (kPageTokens * kStick) + row * kStick + d % kStick;
  if constexpr (kCache == B200KV_F16)
    return to_float(static_cast<const T *>(pool)[at]);
  else if constexpr (kCache == B200KV_I8)
    return static_cast<float>(static_cast<const int8_t *>(pool)[at]);
  else
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t *>(pool)[at], __NV_E4M3)));
}
// Whether row `node` (-1: none) sees a V row whose scale is not finite, in tiles [t0, t1); the whole warp calls it.
static __device__ __noinline__ bool sees_spoilt(const Args &a, const Seq s, int b, int kvh, int node, int t0, int t1) {
  const int lane = threadIdx.x & 31;
  bool sees = false;
  for (int t = t0; t < t1; ++t) {
    const int page = 2 * t + (lane >> 4), have = s.ctx + s.nodes - t * kTileTokens - 4 * lane;
    const int id = have > 0 ? __ldg(a.block_table + static_cast<int64_t>(b) * a.bt_stride + page) : -1;
    uint32_t bad = 0;
    if (id >= 0 && id < a.num_blocks) {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(
                                 a.v_scales + (static_cast<int64_t>(id) * a.hkv + kvh) * kPageTokens) + (lane & 15));
      auto bit = [&](float x, int i) { return i < have && !(x < CUDART_INF_F) ? 1u << i : 0u; };
      bad = bit(v.x, 0) | bit(v.y, 1) | bit(v.z, 2) | bit(v.w, 3);
    }
    if (!__any_sync(0xffffffffu, bad != 0)) continue;
    for (int g = 0; g < 4; ++g) {
      const uint32_t word = __reduce_or_sync(0xffffffffu, lane / 8 == g ? bad << (4 * (lane & 7)) : 0u);
      if (node >= 0 && (word & visible32(a, s, node, t * kTileTokens + 32 * g))) sees = true;
    }
  }
  return sees;
}
// Adds the non-finite elements of the piece's visible nodes to elements
// [d0, d1) of a row that has been written, to its partial sums or its output.
template <typename T, int D, int kCache>
__device__ __noinline__ void repair_row(const Args &a, const Seq &s, int b, int kvh, int node, int from, int to, int d0,
                                        int d1, float *part, T *out) {
  for (int p = max(from, s.ctx); p < min(to, s.ctx + s.nodes); ++p) {
    if (!(visible32(a, s, node, p) & 1u)) continue;
    const int id = __ldg(a.block_table + static_cast<int64_t>(b) * a.bt_stride + p / kPageTokens);
    if (id < 0 || id >= a.num_blocks) continue;
    for (int d = d0; d < d1; ++d) {
      const float v = cached_v<T, D, kCache>(a, a.v_pool, id, kvh, p % kPageTokens, d);
      if (fabsf(v) < CUDART_INF_F) continue;
      if (part)
        part[d / 4 * 1024 + d % 4] += v;
      else
        from_float(out[d], to_float(out[d]) + v);
    }
  }
}

// One softmax warpgroup (w = 0 or 1); thread = row of its Q tile.
template <typename C, typename T, int D, int kCache>
__device__ __forceinline__ void softmax(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem, int w) {
  const int tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5;
  const uint32_t quad = tmem + (uint32_t(warp * 32) << 16);
  const uint32_t ts = quad + col_s(w), to = quad + col_o(w);
  // (a scale of zero: too small to move a score, and -inf stays -inf)
  const float cl = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1e-37f);
  Factors *fac = reinterpret_cast<Factors *>(smem + kOffFactors) + (w * 4 + warp);
  bool dead = false;
  uint32_t s_uses = 0, o_uses[2] = {0, 0}, slot = 0;
  unsigned piece = 0;
  Walk<C::kQ> wk;
  wk.init(c);
  while (wk.next(a, c)) {
    ++piece;
    const bool two = wk.two();
    const int n = wk.t1 - wk.t0, lead = two ? 1 : 2;
    const int len = wk.s.ctx + wk.s.nodes;
    const int qt = C::kQ * wk.block + (two ? w : 0);
    Copies q{1, kTileRows, 1};
    if (C::k8) q = copies_of(a, wk.s, wk.block);
    const int row = tid & (q.rows - 1), copy = tid / q.rows;
    const int node = qt * a.tile_nodes + row / a.group;
    const bool live = row < a.tile_nodes * a.group && node < wk.s.nodes;
    const bool warp_live = __any_sync(0xffffffffu, live);
    // tokens before this one are seen by every row of the Q tile
    const int common = wk.s.ctx + (a.mask ? 0 : qt * a.tile_nodes + 1);
    float m = -CUDART_INF_F, l = 0.f;
    float per = 1.f;  // 8-bit caches: the inverse of what O counts in, 0 as long as all rows were zero
    // 8-bit caches: the scales of this stream's next tile, four tokens per lane
    auto scales_of = [&](int t, float4 &k, float4 &v) {
      const int page = 2 * t + (lane >> 4);
      k = make_float4(0.f, 0.f, 0.f, 0.f), v = make_float4(1.f, 1.f, 1.f, 1.f);
      if (page * kPageTokens >= len) return;  // (what is past the end weighs nothing, and 1 is an ordinary scale)
      v = k;
      const int id = __ldg(a.block_table + static_cast<int64_t>(wk.b) * a.bt_stride + page);
      if (id < 0 || id >= a.num_blocks) return;
      const int64_t at = (static_cast<int64_t>(id) * a.hkv + wk.kvh) * kPageTokens;
      k = __ldg(reinterpret_cast<const float4 *>(a.k_scales + at) + (lane & 15));
      v = __ldg(reinterpret_cast<const float4 *>(a.v_scales + at) + (lane & 15));
    };
    const int step = two ? 1 : 2;
    const int tfirst = wk.t0 + (two ? 0 : w);
    float4 ks, vs;
    if (C::k8 && warp_live && tfirst < wk.t1) scales_of(tfirst, ks, vs);
    for (int t = tfirst; t < wk.t1; t += step) {
      const int pos = t * kTileTokens;
      const bool tail = pos + kTileTokens > common;
      uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
      if (tail && live) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < 4 / q.copies) vis[i] = visible32(a, wk.s, node, pos + copy * q.rows + 32 * i);
      }
      float regain = 1.f;  // the factor that O takes when its unit moves
      if (C::k8 && warp_live) {
        const float4 u = make_float4(vs.x * per, vs.y * per, vs.z * per, vs.w * per);
        __syncwarp();
        fac->k[lane] = make_float4(ks.x * cl, ks.y * cl, ks.z * cl, ks.w * cl);
        if (__all_sync(0xffffffffu, ordinary(u, t == tfirst ? kLeastFirst : kLeastUnits))) {
          put_v(fac, u);
        } else {
          const float now = odd_scales(fac, vs, len - pos - 4 * lane, t == tfirst ? 0.f : per, piece, &c.spoilt_piece);
          if (now != per && t != tfirst) regain = per == 0.f ? 0.f : now * inverse_of_power(per);
          per = now;
        }
        if (t + step < wk.t1) scales_of(t + step, ks, vs);
        __syncwarp();
      }
      auto arrived = [&] {
        wait(&c.s_full[w], s_uses++ & 1u, dead, a.error_flag);
        fence_after();
        if (C::k8 && regain != 1.f) rescale<D>(to, regain);
      };
      if (!C::k8 || !warp_live) arrived();
      if (warp_live) {
        const bool first = t == tfirst;
        if constexpr (C::k8) {
          if (tail)
            weigh8<D, true>(ts, to, vis, fac, q.copies, copy, arrived, first, live, m, l);
          else
            weigh8<D, false>(ts, to, vis, fac, q.copies, copy, arrived, first, live, m, l);
        } else {
          if (tail)
            weigh<typename C::P, D, true>(ts, to, vis, cl, first, live, m, l);
          else
            weigh<typename C::P, D, false>(ts, to, vis, cl, first, live, m, l);
        }
      }
      if (!C::k8 && pos + kTileTokens > min(common, len)) {
        // the pool's rows past the sequence's end hold anything and become
        // zeros, so that weights of zero meet finite values; so do non-finite
        // elements of nodes that not every row sees
        const int i = t - wk.t0;
        const uint32_t vslot = slot + i + min(n, i + lead);
        wait(&c.full[vslot % C::kSlots], (vslot / C::kSlots) & 1u, dead, a.error_flag);
        uint8_t *v = smem + C::kOffSlots + (vslot % C::kSlots) * C::kTile + tid * 16;
        // 16 bytes per thread: row = 16 k + tid / 8
        const int from = max(common - pos, 0), end = len - pos;
        for (int st = 0; st < C::kSticks; ++st) {
#pragma unroll 1
          for (int k = from / 16; k < 8; ++k) {
            uint4 *at = reinterpret_cast<uint4 *>(v + st * C::kStickTile + k * 2048);
            const int vrow = 16 * k + (tid >> 3);
            if (vrow >= end) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (vrow >= from) {
              uint4 x = *at;
              if (!any_non_finite<T>(x)) continue;
              atomicMax(&c.bad_piece, piece);  // before the element goes: the other stream looks too
              __threadfence_block();
              drop_non_finite<T>(x);
              *at = x;
            }
          }
        }
        fence_async_smem();
      }
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(&c.p_ready[w]);
    }
    slot += 2 * n;

    // -------------------------------------------------------- end of piece --
    const bool split = wk.t0 > 0 || wk.t1 < wk.tiles;
    const int pslot = 2 * blockIdx.x + (wk.t0 > 0 ? 0 : 1);  // one of each kind per share
    auto o_wait = [&](int k) {
      wait(&c.o_full[k], o_uses[k]++ & 1u, dead, a.error_flag);
      fence_after();
    };
    float keep0 = 1.f, keep1 = 0.f, unit = 0.f;
    const bool both = !two && n > 1;
    int d0 = 0, d1 = D;
    if (two) {
      o_wait(w);
      ++o_uses[1 - w];
    } else {
      c.ml[w][tid] = make_float2(m, l);
      if (C::k8 && lane == 0) c.unit[w][warp] = per == 0.f || tfirst >= wk.t1 || !warp_live ? 0.f : inverse_of_power(per);
      o_wait(0);
      if (both) o_wait(1);
      bar_pair();
      const float2 x = c.ml[0][tid], y = c.ml[1][tid];
      m = fmaxf(x.x, y.x);
      for (int k = 1; k < q.copies; ++k) {
        const int at = tid ^ (k * q.rows);
        m = fmaxf(m, fmaxf(c.ml[0][at].x, c.ml[1][at].x));
      }
      const float mm = m == -CUDART_INF_F ? 0.f : m;
      keep0 = ex2(x.x - mm);
      keep1 = ex2(y.x - mm);
      if (C::k8) {  // O of both, and of the row's copies, in the largest of their units
#pragma unroll
        for (int k = 0; k < 4; ++k) unit = fmaxf(unit, fmaxf(c.unit[0][k], c.unit[1][k]));
        const float per_unit = unit > 0.f ? inverse_of_power(unit) : 0.f;
        keep0 *= c.unit[0][warp] * per_unit;
        keep1 *= c.unit[1][warp] * per_unit;
      }
      l = 0.f;
      for (int k = 0; k < q.copies; ++k) {
        const float2 xk = c.ml[0][row + k * q.rows], yk = c.ml[1][row + k * q.rows];
        l = fmaf(xk.y, ex2(xk.x - mm), l);
        if (both) l = fmaf(yk.y, ex2(yk.x - mm), l);
      }
      d0 = w * (D / 2);
      d1 = d0 + D / 2;
    }
    const int64_t orow = static_cast<int64_t>(wk.s.q0 + node) * a.hq + wk.kvh * a.group + row % a.group;
    float inv = l == 0.f ? 0.f : 1.f / l;
    if (C::k8) {
      inv *= unit;
      if (*reinterpret_cast<volatile unsigned *>(&c.spoilt_piece) == piece &&
          sees_spoilt(a, wk.s, wk.b, wk.kvh, live ? node : -1, wk.t0, wk.t1))
        inv = CUDART_NAN_F;
    }
    const int prow = (two ? w : 0) * kTileRows + row;
    if (C::k8 && q.copies > 1) {
      // add the copies up, 16 columns at a time through shared memory
      float4 *red = reinterpret_cast<float4 *>(smem + kOffFactors) + w * 4 * kTileRows;
#pragma unroll 1
      for (int d = d0; d < d1; d += 16) {
        uint32_t r[16], r1[16];
        tmem_ld16(quad + col_o(0) + d, r);
        wait_ld(r);
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep0);
        if (both) {
          tmem_ld16(quad + col_o(1) + d, r1);
          wait_ld(r1);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            r[j] = __float_as_uint(fmaf(__uint_as_float(r1[j]), keep1, __uint_as_float(r[j])));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          red[j * kTileRows + tid] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                                                 __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
        bar_group(w);
        for (int j = copy; live && j < 4; j += q.copies) {
          float4 o = red[j * kTileRows + row];
          for (int k = 1; k < q.copies; ++k) {
            const float4 x = red[j * kTileRows + row + k * q.rows];
            o = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
          }
          const int dj = d + 4 * j;
          const bool none = l == 0.f;
          o = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
          if (split)
            *reinterpret_cast<float4 *>(a.part_o + ((static_cast<int64_t>(pslot) * (D / 4) + dj / 4) * 256 + prow) * 4) = o;
          else
            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + orow * D + dj) =
                make_uint2(pack2(o.x, o.y, T()), pack2(o.z, o.w, T()));
        }
        bar_group(w);
      }
    } else if (warp_live) {
      // (short steps: this code runs once per piece, mostly out of a cold
      // instruction cache)
#pragma unroll 1
      for (int d = d0; d < d1; d += 16) {
        uint32_t r[16];
        tmem_ld16(two ? to + d : quad + col_o(0) + d, r);
        wait_ld(r);
        if (!two) {
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep0);
          if (both) {
            uint32_t r1[16];
            tmem_ld16(quad + col_o(1) + d, r1);
            wait_ld(r1);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              r[j] = __float_as_uint(fmaf(__uint_as_float(r1[j]), keep1, __uint_as_float(r[j])));
          }
        }
        const bool none = l == 0.f;
        if (C::k8 && split) {
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = none ? 0u : __float_as_uint(__uint_as_float(r[j]) * inv);
        }
        if (live && split) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4 *>(a.part_o + ((static_cast<int64_t>(pslot) * (D / 4) + d / 4 + j) * 256 + prow) * 4) =
                make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        } else if (live) {
          T *out = static_cast<T *>(a.out) + orow * D + d;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = none ? 0.f : __uint_as_float(r[8 * j + k]) * inv;
            *reinterpret_cast<uint4 *>(out + 8 * j) = pack8(f, T());
          }
        }
        __syncwarp();
      }
    }
    if (live && copy == 0 && *reinterpret_cast<volatile unsigned *>(&c.bad_piece) >= piece)
      repair_row<T, D, kCache>(a, wk.s, wk.b, wk.kvh, node, wk.t0 * kTileTokens, wk.t1 * kTileTokens, d0, d1,
                               split ? a.part_o + (static_cast<int64_t>(pslot) * (D / 4) * 256 + prow) * 4 : nullptr,
                               static_cast<T *>(a.out) + orow * D);
    if (live && copy == 0 && (two || w == 0)) {
      if (split)
        a.part_ml[static_cast<int64_t>(pslot) * 256 + prow] = make_float2(m, l);
      else if (a.lse)
        a.lse[orow] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * 0.69314718055994530942f;
    }
    // the second share of a split block describes it to the join
    if (wk.t0 > 0 && w == 0 && tid == 0) {
      const int first = wk.share_of(0, c.per);
      if (static_cast<int>(blockIdx.x) == first + 1) {
        Join j;
        j.rows0 = wk.s.q0;
        j.node0 = C::kQ * wk.block * a.tile_nodes;
        j.nodes = min(wk.s.nodes - j.node0, C::kQ * a.tile_nodes);
        j.kvh = wk.kvh;
        j.first_cta = first;
        j.last_cta = wk.share_of(wk.tiles - 1, c.per);
        a.joins[blockIdx.x] = j;
      }
    }
    fence_before();
    if (!two) bar_pair();  // both have read O and ml before either goes on
    fence_after();
    wk.advance(a);
  }
}

template <typename T, int D, int kCache>
__global__ void __launch_bounds__((Cfg<T, D, kCache>::kThreads), 1)
    tree_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                const __grid_constant__ CUtensorMap vm, const __grid_constant__ Args a) {
  using C = Cfg<T, D, kCache>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Ctrl &c = *reinterpret_cast<Ctrl *>(smem);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    prefetch_tensormap(&qm);
    if (!C::k8) {
      prefetch_tensormap(&km);
      prefetch_tensormap(&vm);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&c.full[i], C::k8 ? C::kConverters : 1);
      mbar_init(&c.empty[i], 1);
    }
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(&c.raw_full[i], 1);
      mbar_init(&c.raw_empty[i], C::kConverters);
    }
    mbar_init(&c.q_full, 1);
    mbar_init(&c.q_empty, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&c.s_full[w], 1);
      mbar_init(&c.p_ready[w], 4);
      mbar_init(&c.o_full[w], 1);
    }
    fence_mbar_init();
    c.bad_piece = c.spoilt_piece = 0;
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
  make_plan<T, D, C::kThreads, C::kQ>(a, c);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = c.tmem;
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
    softmax<C, T, D, kCache>(a, c, smem, tmem, warp >> 2);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsIssue));
    if (warp == 8) {
      producer<C>(a, c, smem, &qm, &km, &vm);
    } else if (warp == 9) {
      mma_issuer<C, D>(a, c, smem, tmem);
    }
  } else {
    if constexpr (C::k8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsConvert));
      converter<C, T, kCache>(a, c, smem, warp - 12);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------- join --
// Blocks cut by CTA boundaries: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// over the pieces in order (the same bits every time).  The pieces of an 8-bit
// cache have units of their own and come divided by their l (kDivided).  One CTA
// per boundary and 32 rows; lane = row, warp = an eighth of the head.
template <typename T, int D, bool kDivided>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ Args a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Join j = a.joins[blockIdx.x];
  const int tile_rows = a.tile_nodes * a.group;
  const int prow = blockIdx.y * 32 + (threadIdx.x & 31);
  const int in_tile = prow & (kTileRows - 1), tile = prow / kTileRows;
  const int node = tile * a.tile_nodes + in_tile / a.group;
  if (in_tile >= tile_rows || node >= j.nodes) return;
  constexpr int kPer = D / 8 / 4, kAhead = 4;
  const int d4 = (threadIdx.x >> 5) * kPer;
  float M = -CUDART_INF_F, l = 0.f, o[4 * kPer];
#pragma unroll
  for (int i = 0; i < 4 * kPer; ++i) o[i] = 0.f;
  for (int x0 = j.first_cta; x0 <= j.last_cta; x0 += kAhead) {
    float2 ml[kAhead];
    float4 v[kAhead][kPer];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      ml[k] = make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (x0 + k > j.last_cta) continue;
      const int64_t s = 2 * (x0 + k) + (x0 + k == j.first_cta ? 1 : 0);
      ml[k] = a.part_ml[s * 256 + prow];
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        v[k][i] = *reinterpret_cast<const float4 *>(a.part_o + ((s * (D / 4) + d4 + i) * 256 + prow) * 4);
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) top = fmaxf(top, ml[k].x);
    const float mm = top == -CUDART_INF_F ? 0.f : top;
    const float old = exp2f(M - mm);
    M = top;
    l *= old;
#pragma unroll
    for (int i = 0; i < 4 * kPer; ++i) o[i] *= old;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float keep = exp2f(ml[k].x - mm);
      l = fmaf(ml[k].y, keep, l);
      const float weight = kDivided ? ml[k].y * keep : keep;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        o[4 * i] = fmaf(v[k][i].x, weight, o[4 * i]);
        o[4 * i + 1] = fmaf(v[k][i].y, weight, o[4 * i + 1]);
        o[4 * i + 2] = fmaf(v[k][i].z, weight, o[4 * i + 2]);
        o[4 * i + 3] = fmaf(v[k][i].w, weight, o[4 * i + 3]);
      }
    }
  }
  const int64_t orow = (j.rows0 + j.node0 + node) * a.hq + j.kvh * a.group + in_tile % a.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *out = static_cast<T *>(a.out) + orow * D + 4 * d4;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t lo = pack2(l == 0.f ? 0.f : o[4 * i] * inv, l == 0.f ? 0.f : o[4 * i + 1] * inv, T());
    const uint32_t hi = pack2(l == 0.f ? 0.f : o[4 * i + 2] * inv, l == 0.f ? 0.f : o[4 * i + 3] * inv, T());
    *reinterpret_cast<uint2 *>(out + 4 * i) = make_uint2(lo, hi);
  }
  if (threadIdx.x < 32 && a.lse) a.lse[orow] = l == 0.f ? -CUDART_INF_F : (M + log2f(l)) * 0.69314718055994530942f;
}

// ----------------------------------------------------------------- launch --
template <typename T, int D, int kCache>
int launch(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, const Args &a, int ctas,
           cudaStream_t stream) {
  using C = Cfg<T, D, kCache>;
  static int configured[64] = {0};
  int dev = 0;
  B200KV_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return set_error(B200KV_ERR_UNSUPPORTED, "device ordinal %d", dev);
  if (!__atomic_load_n(&configured[dev], __ATOMIC_ACQUIRE)) {
    B200KV_CUDA_TRY(cudaFuncSetAttribute(tree_kernel<T, D, kCache>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    __atomic_store_n(&configured[dev], 1, __ATOMIC_RELEASE);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, tree_kernel<T, D, kCache>, qm, km, vm, a));
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), C::kQ == 2 && a.max_nodes > a.tile_nodes ? 8 : 4);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, tree_join_kernel<T, D, C::k8>, a));
  return B200KV_OK;
}

}  // namespace tree
}  // namespace b200kv
