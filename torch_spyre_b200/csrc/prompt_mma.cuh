// Tensor-core kernel of prompt attention (prompt_attention.cu has the operator):
// heads with keys of 128 own and 64 shared elements, values of 128.
//
// The rows of a sequence and head are cut into Q tiles of 128, two of which form a
// block; a block's tokens are cut into tiles of 80.  The blocks' tiles, all
// sequences and heads one after the other, form one line that is cut into equal
// shares, one per CTA; a block cut by a share's end is joined by prompt_join_kernel.
//
// Inside a CTA two streams run side by side, each with its own eight warps, scores S,
// weights P and accumulator O in TMEM: the block's two Q tiles over every token
// tile, or, with one Q tile, alternate token tiles, whose states are merged when
// the block ends.  Per tile: S = Q K^T (12 products of 16 elements), the warps take S
// into registers (then the next tile's S may come), mask and exponentiate, P goes to
// TMEM in 16 bits, O += P V with P as the TMEM operand.  O is only rescaled when a
// row's maximum has risen by more than 2^8.
//
// 80 tokens, since a stream has 256 of TMEM's columns: 80 S, 40 P, 128 O.  (Tiles of 128 with P in
// S's place have 25 % fewer clocks of products, 2560 for 128 tokens and both streams, but a
// stream's products and softmax then follow one another: 233 us for four prompts where these took 225, 1440
// for two chunks and 1345.)
//
// What bounds it: the softmax warps, which are never idle: of 2700 clocks for a tile of both
// streams 200 to take S, 200 for the rows' maxima, 1300 to 1450 for exponentials (1280 of
// the special-function units', which both streams use at once; in turns they are no
// faster), 300 to write P, the rest waits and arrivals; the products take 1900.  Then the
// power limit: in long runs the clock falls from 1965 to some 1600 MHz.  Four prompts of up to 4096 rows, 16
// heads: 219 us, in long runs 252; two chunks of 777 to 1024 rows over 4001 to 8000 tokens, 128 heads: 1325 and 1537.
// Exponentials by a polynomial on the FMA units, for a quarter or a half of the
// elements, waits that sleep, and code laid out without loops were as fast or slower.
//
// Shared memory holds two Q tiles and twelve columns of 64 elements x 80 tokens: a
// K tile is three (two of the head's, one of the shared part), a V tile two, so
// that the next tiles' come in while this one's are in use.
//
// Warps: 0-7 and 8-15 the streams' softmax (a row is in two threads, each with half of a
// tile's tokens and of O's columns), 16 the TMA producer, 17 and 18 issue the streams' MMAs.
#pragma once

#include "prompt_attention.h"
#include "umma.cuh"

namespace b200kv {
namespace prompt {

using namespace umma;

constexpr int kThreads = 640;
constexpr int kRegsSoftmax = 104, kRegsIssue = 64;  // a thread, after setmaxnreg (640 threads of 96 at launch)
constexpr int kTile = 128;                          // rows of a Q tile
constexpr int kTok = 80, kHalf = kTok / 2;          // tokens of a K or V tile
constexpr int kColQ = kTile * 128, kCol = kTok * 128;  // bytes of a column of 64 elements
constexpr int kColsQ = 3, kColsV = 2, kSlots = 12;
constexpr int kLead = 2;                            // tiles that keys are ahead of values
constexpr int kOffQ = 3 * 1024;
constexpr int kOffSlots = kOffQ + 2 * kColsQ * kColQ;
constexpr int kSmem = kOffSlots + kSlots * kCol;
constexpr float kLazyLog2 = 8.f;
static_assert(kSmem <= 227 * 1024, "shared memory per CTA");

// TMEM columns
constexpr uint32_t kTmemCols = 512;
__device__ __forceinline__ uint32_t col_s(int w) { return uint32_t(w) * 128u; }
__device__ __forceinline__ uint32_t col_p(int w) { return uint32_t(w) * 128u + kTok; }
__device__ __forceinline__ uint32_t col_o(int w) { return 256u + uint32_t(w) * 128u; }

struct Seq {
  int q0, rows, kv0, len, blocks;
  int past;  // tokens before the first row's own (may be negative)
  int end;   // the first row of q that is a later sequence's
};
struct Start {  // where a share begins: in a block whose units begin at u0, counted from the share's first
  Seq s;
  int b, head, block, u0;
};

struct Ctrl {
  uint64_t full[kSlots], empty[kSlots];  // (a slot is empty when both streams say so)
  uint64_t q_full, q_empty;
  uint64_t s_full[2], s_free[2], p_ready[2], p_free[2], o_full[2];
  uint32_t tmem;
  int per, end;  // units of a share, of this CTA's (the last may have fewer, or none)
  Start start;
  int64_t scan[kThreads / 32];
  unsigned bad_piece;  // last piece (counted from 1) that met a non-finite value in a V row
  float top[2][2][kTile];  // streams' rows: the halves' maxima of a tile; sums, when a piece ends
};
static_assert(sizeof(Ctrl) <= kOffQ, "control block");

__device__ __forceinline__ void bar_all() { asm volatile("bar.sync 1, 512;" ::: "memory"); }  // both streams' softmax
// The two warps that have a stream's rows 32 q .. 32 q + 31.
__device__ __forceinline__ void bar_rows(int w, int q) { asm volatile("bar.sync %0, 64;" ::"r"(2 + 4 * w + q) : "memory"); }

__device__ __forceinline__ bool any_rows(int w, int q, bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"(uint32_t(x)), "r"(2 + 4 * w + q)
               : "memory");
  return r != 0;
}

// -------------------------------------------------------------------- plan --
__device__ __forceinline__ Seq load_seq(const Args &a, int b, bool report) {
  Seq s;
  s.q0 = __ldg(a.q_indptr + b);
  s.kv0 = __ldg(a.kv_indptr + b);
  const int end = __ldg(a.q_indptr + b + 1), kv_end = __ldg(a.kv_indptr + b + 1);
  const bool bad = s.q0 < 0 || end < s.q0 || end > a.total_q || s.kv0 < 0 || kv_end < s.kv0 || kv_end > a.total_kv ||
                   (b == 0 && s.q0 != 0) || (b == a.batch - 1 && end != a.total_q);
  s.q0 = min(max(s.q0, 0), a.total_q);
  s.rows = min(max(end, s.q0), a.total_q) - s.q0;
  s.end = b == a.batch - 1 ? a.total_q : min(max(end, 0), a.total_q);
  s.kv0 = min(max(s.kv0, 0), a.total_kv);
  s.len = min(max(kv_end, s.kv0), a.total_kv) - s.kv0;
  s.past = s.len - s.rows;
  if (bad && report && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_BAD_LEN);
  s.blocks = (s.rows + 2 * kTile - 1) / (2 * kTile);
  return s;
}
// Token tiles of block k: what its last row sees (one at least, which may be masked whole).
__device__ __forceinline__ int block_tiles(const Args &a, const Seq &s, int k) {
  const int seen = a.causal ? s.past + min(s.rows, (k + 1) * 2 * kTile) : s.len;
  return max((seen + kTok - 1) / kTok, 1);
}
// The line is cut by cost: a step over a token tile counts 2 with one Q tile and 4
// with two, a block's beginning and end kBegin[0] and [1].
constexpr int kBegin1 = 18, kBegin2 = 26;
__device__ __forceinline__ bool two_tiles(const Seq &s, int k) { return s.rows - k * 2 * kTile > kTile; }
__device__ __forceinline__ int step_units(const Seq &s, int k) { return two_tiles(s, k) ? 4 : 2; }
__device__ __forceinline__ int begin_units(const Seq &s, int k) { return two_tiles(s, k) ? kBegin2 : kBegin1; }
__device__ __forceinline__ int block_units(const Args &a, const Seq &s, int k) {
  return begin_units(s, k) + step_units(s, k) * block_tiles(a, s, k);
}
// (The line is counted in 64 bits, a share and a block in 31: the host has bounded a share.)
__device__ __forceinline__ int64_t head_units(const Args &a, const Seq &s) {
  if (s.blocks == 0) return 0;
  // without a mask all blocks have as many tiles, and only the last may be of one Q tile
  if (!a.causal) return static_cast<int64_t>(s.blocks - 1) * block_units(a, s, 0) + block_units(a, s, s.blocks - 1);
  int64_t n = 0;
  for (int k = 0; k < s.blocks; ++k) n += block_units(a, s, k);
  return n;
}

// The blocks of a CTA's share, one piece (a block, or the part of it in this
// share) at a time.  Every role walks the same sequence.
struct Walk {
  Seq s;
  int b, head, block, u0, tiles, t0, t1;  // piece: token tiles [t0, t1) of `tiles`
  int end;                                // of the share; units count from its first

  __device__ __forceinline__ void init(const Ctrl &c) {
    const Start &f = c.start;
    s = f.s, b = f.b, head = f.head, block = f.block, u0 = f.u0;
    t1 = 0;
    end = c.end;
  }
  // Tile t belongs to the share that holds its first unit.
  __device__ __forceinline__ int tile_from(int unit) const {
    const int w = step_units(s, block), x = unit - u0 - begin_units(s, block);
    return x <= 0 ? 0 : min(tiles, (x + w - 1) / w);
  }
  __device__ __forceinline__ bool next(const Args &a) {
    for (;;) {
      if (end <= 0 || u0 >= end) return false;
      tiles = block_tiles(a, s, block);
      t0 = tile_from(0);
      t1 = tile_from(end);
      if (t0 < t1) return true;
      advance(a);
    }
  }
  __device__ __forceinline__ void advance(const Args &a) {
    u0 += block_units(a, s, block);
    if (u0 >= end) return;
    if (++block >= s.blocks) {
      block = 0;
      if (++head >= a.heads) {
        head = 0;
        do s = load_seq(a, ++b, false);
        while (s.rows == 0);
      }
    }
  }
  __device__ __forceinline__ bool two() const { return two_tiles(s, block); }
  __device__ __forceinline__ int share_of(int t, int per) const {
    const int x = u0 + begin_units(s, block) + t * step_units(s, block);
    return static_cast<int>(blockIdx.x) + (x >= 0 ? x / per : -((per - 1 - x) / per));
  }
};

// Rows of q that no sequence has (all of them flagged): they see nothing.
template <typename T>
__device__ __noinline__ void clear_rows(const Args &a, bool all) {
  for (int b = 0; b < a.batch; ++b) {
    const Seq s = load_seq(a, b, false);
    const int first = b == 0 ? 0 : s.q0, end = all ? (b == 0 ? a.total_q : 0) : s.end;
    for (int t = first + blockIdx.x; t < end; t += gridDim.x) {
      if (!all && t >= s.q0 && t < s.q0 + s.rows) continue;
      uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + static_cast<int64_t>(t) * a.heads * kDim);
      for (int i = threadIdx.x; i < a.heads * (kDim / 8); i += blockDim.x) out[i] = make_uint4(0, 0, 0, 0);
      if (!a.lse) continue;
      for (int h = threadIdx.x; h < a.heads; h += blockDim.x) a.lse[static_cast<int64_t>(t) * a.heads + h] = -CUDART_INF_F;
    }
  }
}

// The line's length, a share's, and where this CTA's begins; all threads call it,
// a barrier follows.  A share fits 31 bits (the host checks) where no two sequences have
// the same row or token: with offsets that descend nothing has a sequence.
template <typename T>
__device__ __forceinline__ void make_plan(const Args &a, Ctrl &c) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.batch + kThreads - 1) / kThreads;
  const int b0 = tid * each, b1 = min(b0 + each, a.batch);
  Seq s{};
  int64_t mine = 0;
  bool unclaimed = false, descends = false;
  for (int b = b0; b < b1; ++b) {
    descends = descends || __ldg(a.q_indptr + b + 1) < __ldg(a.q_indptr + b) || __ldg(a.kv_indptr + b + 1) < __ldg(a.kv_indptr + b);
  }
  const bool none = __syncthreads_or(descends);
  for (int b = b0; b < b1; ++b) {
    s = load_seq(a, b, blockIdx.x == 0);
    if (!none) mine += head_units(a, s) * a.heads;
    unclaimed = unclaimed || (b == 0 && s.q0 > 0) || s.q0 + s.rows < s.end;
  }
  int64_t incl = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, m);
    if (lane >= m) incl += y;
  }
  if (lane == 31) c.scan[warp] = incl;
  if (__syncthreads_or(unclaimed || none)) clear_rows<T>(a, none);
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += c.scan[w];
    total += c.scan[w];
  }
  // (at least a step, so that a share inside a block holds the start of a tile)
  const int per = max(4, static_cast<int>((total + gridDim.x - 1) / gridDim.x));
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per;
  int64_t at = before + incl - mine;
  if (first >= at && first < at + mine) {
    int64_t hu = 0;
    int b = b0;
    for (;; ++b) {
      if (each > 1) s = load_seq(a, b, false);
      hu = head_units(a, s);
      if (first < at + hu * a.heads) break;
      at += hu * a.heads;
    }
    const int head = static_cast<int>((first - at) / hu);
    at += head * hu;
    int block = 0;
    if (!a.causal) {
      const int n = block_units(a, s, 0);
      block = static_cast<int>(min((first - at) / n, static_cast<int64_t>(s.blocks - 1)));
      at += static_cast<int64_t>(block) * n;
    } else {
      for (int n; first >= at + (n = block_units(a, s, block)); ++block) at += n;
    }
    c.start = Start{s, b, head, block, static_cast<int>(at - first)};
  }
  if (tid == 0) {
    c.per = per;
    c.end = static_cast<int>(max(min(total - first, static_cast<int64_t>(per)), int64_t{0}));
  }
}

// The columns' places, one tile after the other.  A V tile's two lie side by side (one
// product reads both), so one that would begin in the last slot begins in the first, and
// that slot is not used in its turn: every slot has a parity of its own.
struct Ring {
  uint32_t pos = 0, parities = 0;
  struct Tile {
    uint32_t at, parities;  // first slot, the slots' parities
    __device__ __forceinline__ uint32_t slot(uint32_t c) const { return (at + c) % kSlots; }
    __device__ __forceinline__ uint32_t parity(uint32_t c) const { return parities >> slot(c) & 1u; }
  };
  template <int kCols>
  __device__ __forceinline__ Tile take() {
    if (kCols == kColsV && pos == kSlots - 1) pos = 0;
    const Tile t{pos, parities};
    const uint32_t used = ((1u << kCols) - 1u) << pos;
    parities ^= (used | used >> kSlots) & ((1u << kSlots) - 1u);
    pos = (pos + kCols) % kSlots;
    return t;
  }
  __device__ __forceinline__ Tile k() { return take<kColsQ>(); }
  __device__ __forceinline__ Tile v() { return take<kColsV>(); }
};

// ------------------------------------------------------------------- roles --
__device__ __forceinline__ void producer(const Args &a, Ctrl &c, uint8_t *smem, const CUtensorMap *qm,
                                         const CUtensorMap *km, const CUtensorMap *rm, const CUtensorMap *vm) {
  const int lane = threadIdx.x & 31;
  bool dead = false;
  uint32_t pieces = 0;  // begun
  Ring ring;
  uint32_t loaded = 0, last = 0;  // slots with a copy that was issued, their parities
  Walk w;
  w.init(c);
  while (w.next(a)) {
    const bool two = w.two();
    // a column to a lane
    auto issue = [&](const Ring::Tile &tile, uint32_t cols, const CUtensorMap *map, int t) {
      wait_until(
          [&] {
            bool ok = mbar_test(&c.empty[tile.slot(0)], tile.parity(0) ^ 1u) & mbar_test(&c.empty[tile.slot(1)], tile.parity(1) ^ 1u);
            if (cols == 3) ok = ok & mbar_test(&c.empty[tile.slot(2)], tile.parity(2) ^ 1u);
            return ok;
          },
          dead, a.error_flag);
      if ((dead = __any_sync(0xffffffffu, dead))) return;
      if (lane < static_cast<int>(cols)) {
        const uint32_t s = tile.slot(lane);
        mbar_arrive_expect_tx(&c.full[s], kCol);
        tma_3d(smem + kOffSlots + s * kCol, lane == 2 ? rm : map, &c.full[s], lane == 1 ? 64 : 0, lane == 2 ? 0 : w.head,
               w.s.kv0 + t * kTok);
      }
      __syncwarp();
      for (uint32_t x = 0; x < cols; ++x) {
        const uint32_t bit = 1u << tile.slot(x);
        loaded |= bit;
        last = (last & ~bit) | (tile.parities & bit);
      }
    };
    for (int t = w.t0; t < min(w.t0 + kLead, w.t1) && !dead; ++t) issue(ring.k(), kColsQ, km, t);
    // (the first keys may come before the piece before is done with Q)
    if (dead) break;
    wait(&c.q_empty, (pieces & 1u) ^ 1u, dead, a.error_flag);
    if ((dead = __any_sync(0xffffffffu, dead))) break;
    const int n = (two ? 2 : 1) * kColsQ;
    if (lane == 0) mbar_arrive_expect_tx(&c.q_full, uint32_t(n) * kColQ);
    __syncwarp();
    if (lane < n)
      tma_3d(smem + kOffQ + lane * kColQ, qm, &c.q_full, lane % kColsQ * 64, w.head,
             w.s.q0 + (2 * w.block + lane / kColsQ) * kTile);
    ++pieces;
    for (int t = w.t0; t < w.t1 && !dead; ++t) {
      issue(ring.v(), kColsV, vm, t);
      if (t + kLead < w.t1 && !dead) issue(ring.k(), kColsQ, km, t + kLead);
    }
    if (dead) break;
    w.advance(a);
  }
  if (dead) {  // the copies under way, with a limit
    bool late = false;
    if (pieces > 0) wait(&c.q_full, (pieces - 1) & 1u, late, a.error_flag);
    for (uint32_t s = 0; s < kSlots; ++s)
      if (loaded >> s & 1u) wait(&c.full[s], last >> s & 1u, late, a.error_flag);
  }
  // the last arrival that the MMAs owe this CTA: not before it may the CTA end
  if (lane == 0 && pieces > 0) {
    bool late = false;
    wait(&c.q_empty, (pieces & 1u) ^ 1u, late, a.error_flag);
  }
  __syncwarp();
}

// The MMA warp of stream w, converged, issues from an elected lane: the next tile's
// scores, which the softmax makes room for when it has taken this one's, then this one's
// values, when its weights are there.
template <typename T>
__device__ __forceinline__ void mma_issuer(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem_any, int w) {
  constexpr uint32_t kBase =
      (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | (uint32_t(kTile >> 4) << 24);
  constexpr uint32_t kIdescQK = kBase | (uint32_t(kTok >> 3) << 17);
  constexpr uint32_t kIdescPV = kBase | (1u << 16) | (uint32_t(kDim >> 3) << 17);  // V: N-major
  bool dead = false;
  uint32_t pieces = 0, s_uses = 0, p_uses = 0;
  const uint32_t go = elect_one(), s_at = uniform(tmem_any + col_s(w)), p_at = uniform(tmem_any + col_p(w)), o_at = uniform(tmem_any + col_o(w));
  const uint32_t idesc_qk = kIdescQK | (a.scale < 0.f ? 1u << 13 : 0u);  // a negative scale turns Q's sign
  const uint32_t kd = desc_kmajor(smem_u32(smem + kOffSlots));
  const uint32_t vd = (smem_u32(smem + kOffSlots) >> 4) | (uint32_t(kCol >> 4) << 16);
  auto done = [&](uint64_t *bar) {
    if (go) commit(bar);
  };
  // a slot waits for both streams: the one that a tile is for alone says it twice
  auto free = [&](const Ring::Tile &tile, uint32_t cols, bool alone) {
    for (uint32_t x = 0; x < cols; ++x) {
      done(&c.empty[tile.slot(x)]);
      if (alone) done(&c.empty[tile.slot(x)]);
    }
  };
  auto filled = [&](const Ring::Tile &tile, uint32_t x) { return mbar_test(&c.full[tile.slot(x)], tile.parity(x)); };
  // scores, once the softmax has taken those before out of their columns
  auto qk = [&](const Ring::Tile &tile, int qtile, bool alone) {
    wait_until(
        [&] {
          const bool ok = filled(tile, 0) & filled(tile, 1) & filled(tile, 2);
          return ok & (s_uses == 0 || mbar_test(&c.s_free[w], (s_uses - 1) & 1u));
        },
        dead, a.error_flag);
    ++s_uses;
    fence_after();
    const uint32_t qd = uniform(desc_kmajor(smem_u32(smem + kOffQ)) + (qtile * kColsQ * kColQ >> 4)), at = uniform(tile.at);
#pragma unroll
    for (int col = 0; col < kColsQ; ++col) {
      const uint32_t k0 = kd + ((at + col) % kSlots * kCol >> 4);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mma_ss(s_at, qd + ((col * kColQ + i * 32) >> 4), k0 + (i * 32 >> 4), idesc_qk, col + i > 0, go);
    }
    free(tile, kColsQ, alone);
    done(&c.s_full[w]);
  };
  auto pv = [&](const Ring::Tile &tile, bool first, bool alone) {
    wait_until([&] { return mbar_test(&c.p_ready[w], p_uses & 1u) & filled(tile, 0) & filled(tile, 1); }, dead, a.error_flag);
    ++p_uses;
    fence_after();
    const uint32_t v = uniform(vd + (tile.at * kCol >> 4)), later = uniform(!first);
#pragma unroll
    for (int i = 0; i < kTok / 16; ++i) mma_ts(o_at, p_at + i * 8, v + (i * 2048 >> 4), kIdescPV, i > 0 ? 1 : later, go);
    free(tile, kColsV, alone);
    done(&c.p_free[w]);
  };
  Ring ring;
  Walk wk;
  wk.init(c);
  while (wk.next(a)) {
    wait(&c.q_full, pieces++ & 1u, dead, a.error_flag);
    const int n = wk.t1 - wk.t0;
    Ring::Tile k[2] = {ring.k(), Ring::Tile{0, 0}};
    if (n > 1) k[1] = ring.k();
    if (wk.two()) {
      qk(k[0], w, false);
      for (int t = 0; t < n; ++t) {
        const Ring::Tile v = ring.v();
        if (t + 1 < n) qk(k[1], w, false);
        if (t + 2 == n || n == 1) done(&c.q_empty);
        if (t + 2 < n) k[1] = ring.k();
        pv(v, t == 0, false);
      }
      done(&c.o_full[w]);
    } else {
      // stream t & 1 takes tile t
      if (w < n) qk(w == 0 ? k[0] : k[1], 0, true);
      for (int t = 0; t < n; ++t) {
        const Ring::Tile v = ring.v();
        const bool mine = (t & 1) == w;
        if (t + 2 < n) {
          const Ring::Tile next = ring.k();
          if (mine) qk(next, 0, true);
        }
        if (mine) pv(v, t < 2, true);
      }
      if (w < n) done(&c.o_full[w]);
      done(&c.q_empty);
    }
    wk.advance(a);
  }
  __syncwarp();
}

template <bool kTail, int kN>
__device__ __forceinline__ float mask_max(uint32_t (&s)[kN], uint32_t vis) {
  if (kTail) {
#pragma unroll
    for (int j = 0; j < kN; ++j) s[j] = vis >> j & 1u ? s[j] : 0xff800000u;  // -inf
  }
  float t = __uint_as_float(s[0]);
#pragma unroll
  for (int j = 1; j < kN - 1; j += 2) t = fmaxf(fmaxf(t, __uint_as_float(s[j])), __uint_as_float(s[j + 1]));
  return fmaxf(t, __uint_as_float(s[kN - 1]));
}
// exp2(x * cl + minus) of kN scores, two to a word, their sum added to `sum`.
template <typename T, int kN>
__device__ __forceinline__ void weigh(const uint32_t (&s)[2 * kN], float cl, float minus, float2 (&sum)[2], uint32_t (&p)[kN]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const float2 x = make_float2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1]));
    const float2 y = fma2(x, make_float2(cl, cl), make_float2(minus, minus));
    const float2 e = make_float2(ex2(y.x), ex2(y.y));
    sum[j & 1] = add2(sum[j & 1], e);
    p[j] = pack2(e.x, e.y, T());
  }
}

// What a thread of the softmax keeps: a row of its stream's Q tile, half of a tile's tokens.
struct Half {
  uint32_t ts, tp, to;  // this half of the row's scores, weights, O
  float *top;
  const float *other;   // the halves' maxima
  uint64_t *s_free, *p_free;
  int w, q;
  uint32_t tiles;       // of the stream, so far
  float m, l;
};
// O moves to a new maximum once the values before are in it.
__device__ __noinline__ void rescale(uint32_t to, float keep) {
#pragma unroll 1
  for (int i = 0; i < kDim / 2; i += 16) {
    uint32_t r[16];
    tmem_ld16(to + i, r);
    wait_ld(r);
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
    tmem_st16(to + i, r);
  }
  wait_st();
}
// Scores of a row's 40 tokens of this half -> weights.  kTail: the row sees the first
// `seen` of them.
template <typename T, bool kTail>
__device__ __forceinline__ void tile(Half &h, int seen, float cl, bool first, bool live, bool &dead, int32_t *flag) {
  uint32_t s0[32], s1[8];
  tmem_ld32(h.ts, s0);
  tmem_ld8(h.ts + 32, s1);
  wait_ld(s0);
  wait_ld(s1);
  fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) arrive(h.s_free);  // the next tile's may come
  float mt = fmaxf(mask_max<kTail>(s0, kTail ? low_bits(seen) : ~0u), mask_max<kTail>(s1, kTail ? low_bits(seen - 32) : ~0u));
  mt = fmaf(mt, cl, -kWeightLog2<T>);
  const uint32_t before = (h.tiles - 1) & 1u;  // parity of the tile before's products
  // the row's maximum is that of both halves; it moves when one has risen far enough
  if (any_rows(h.w, h.q, first || (live && mt > h.m + kLazyLog2))) {
    *h.top = mt;
    bar_rows(h.w, h.q);
    mt = fmaxf(mt, *h.other);
    const bool rise = mt > h.m + (first ? 0.f : kLazyLog2);
    if (!first) {
      const float keep = rise ? ex2(h.m - mt) : 1.f;
      h.l *= keep;
      wait(h.p_free, before, dead, flag);
      __syncwarp();
      fence_after();
      rescale(h.to, keep);
    }
    if (rise) h.m = mt;
  }
  const float minus = h.m == -CUDART_INF_F ? 0.f : -h.m;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t p0[16], p1[4];
  weigh<T>(s0, cl, minus, sum, p0);
  const bool is_free = h.tiles == 0 || mbar_test(h.p_free, before);  // (an answer that takes as long as the rest)
  weigh<T>(s1, cl, minus, sum, p1);
  const float2 t = add2(sum[0], sum[1]);
  h.l += t.x + t.y;
  if (!is_free) wait(h.p_free, before, dead, flag);
  __syncwarp();
  fence_after();
  tmem_st16(h.tp, p0);
  tmem_st4(h.tp + 16, p1);
  wait_st();
}

// Adds the non-finite V elements of tokens [from, to) to a row that has been
// written, to its partial sums or its output.
template <typename T>
__device__ __noinline__ void repair_row(const Args &a, const Seq &s, int head, int from, int to, int d0, int d1, float *part,
                                        T *out) {
  for (int p = from; p < to; ++p) {
    const T *row = static_cast<const T *>(a.v) + (s.kv0 + p) * a.v_st + head * a.v_sh;
    for (int d = d0; d < d1; ++d) {
      const float v = to_float(row[d]);
      if (fabsf(v) < CUDART_INF_F) continue;
      if (part)
        part[d / 4 * 1024 + d % 4] += v;
      else
        from_float(out[d], to_float(out[d]) + v);
    }
  }
}

// The softmax of stream w; a thread has a row of its Q tile and a half of a tile's tokens.
template <typename T>
__device__ __forceinline__ void softmax(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem, int w) {
  const int tid = threadIdx.x & 127, lane = tid & 31, q = tid >> 5, half = (threadIdx.x >> 7) & 1;
  const uint32_t quad = tmem + (uint32_t(q * 32) << 16);
  float *top = &c.top[w][half][tid], *other = &c.top[w][half ^ 1][tid];
  Half h{quad + col_s(w) + half * kHalf, quad + col_p(w) + half * (kHalf / 2), quad + col_o(w) + half * (kDim / 2),
         top, other, &c.s_free[w], &c.p_free[w], w, q, 0, 0.f, 0.f};
  // (a scale of zero: too small to move a score, and -inf stays -inf)
  const float cl = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1e-37f);
  bool dead = false;
  uint32_t o_uses[2] = {0, 0};
  Ring ring;
  unsigned piece = 0;
  Walk wk;
  wk.init(c);
  while (wk.next(a)) {
    ++piece;
    const bool two = wk.two();
    const int n = wk.t1 - wk.t0;
    const int len = wk.s.len, row0 = (2 * wk.block + (two ? w : 0)) * kTile;
    const int row = row0 + tid;
    const bool live = row < wk.s.rows;
    const bool warp_live = __any_sync(0xffffffffu, live);
    // what this row sees, and what all rows of the Q tile see
    const int seen = a.causal ? min(wk.s.past + row + 1, len) : len;
    const int common = a.causal ? min(max(wk.s.past + row0 + 1, 0), len) : len;
    h.m = -CUDART_INF_F, h.l = 0.f;
    const int tfirst = wk.t0 + (two ? 0 : w);
    for (int i = 0; i < min(kLead, n); ++i) ring.k();
    for (int t = wk.t0; t < wk.t1; ++t) {
      const Ring::Tile vt = ring.v();
      if (t + kLead < wk.t1) ring.k();
      if (!two && ((t - wk.t0) & 1) != w) continue;
      const int pos = t * kTok;
      const bool tail = pos + kTok > common;
      wait(&c.s_full[w], h.tiles & 1u, dead, a.error_flag);
      fence_after();
      if (warp_live) {
        if (tail)
          tile<T, true>(h, seen - pos - kHalf * half, cl, t == tfirst, live, dead, a.error_flag);
        else
          tile<T, false>(h, kHalf, cl, t == tfirst, live, dead, a.error_flag);
      } else {
        // (no faster than the others: an arrival for the next tile would count for this one)
        if (lane == 0) arrive(&c.s_free[w]);
        if (h.tiles > 0) wait(&c.p_free[w], (h.tiles - 1) & 1u, dead, a.error_flag);
      }
      ++h.tiles;
      if (tail) {
        // V rows past the sequence's end are another's and become zeros, so that weights of
        // zero meet finite values; so do non-finite elements that not every row sees
        const int from = max(common - pos, 0), end = len - pos;
        wait(&c.full[vt.slot(half)], vt.parity(half), dead, a.error_flag);
        uint8_t *base = smem + kOffSlots + vt.slot(half) * kCol + tid * 16;
#pragma unroll 1
        for (int k = min(from, max(end, 0)) / 16; k < kTok / 16; ++k) {  // 16 bytes per thread: row = 16 k + tid / 8
          uint4 *at = reinterpret_cast<uint4 *>(base + k * 2048);
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
        fence_async_smem();
      }
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(&c.p_ready[w]);
    }

    // -------------------------------------------------------- end of piece --
    const bool split = wk.t0 > 0 || wk.t1 < wk.tiles;
    const int pslot = 2 * blockIdx.x + (wk.t0 > 0 ? 0 : 1);  // one of each kind per share
    auto o_wait = [&](int k) {
      wait(&c.o_full[k], o_uses[k]++ & 1u, dead, a.error_flag);
      fence_after();
    };
    // (once O is full all of the stream's threads have read the last tile's maxima)
    float m = h.m, l = h.l;
    float keep0 = 1.f, keep1 = 0.f;
    const bool both = !two && n > 1;
    int d0 = half * (kDim / 2), d1 = d0 + kDim / 2;
    if (two) {
      o_wait(w);
      ++o_uses[1 - w];
      *top = l;
      bar_rows(w, q);
      l += *other;
      bar_rows(w, q);
    } else {
      o_wait(0);
      if (both) o_wait(1);
      bar_all();
      *top = l;
      bar_all();
      const float l0 = c.top[0][0][tid] + c.top[0][1][tid], l1 = c.top[1][0][tid] + c.top[1][1][tid];
      bar_all();
      *top = m;
      bar_all();
      const float m0 = c.top[0][0][tid], m1 = both ? c.top[1][0][tid] : -CUDART_INF_F;
      m = fmaxf(m0, m1);
      const float mm = m == -CUDART_INF_F ? 0.f : m;
      keep0 = ex2(m0 - mm);
      keep1 = ex2(m1 - mm);
      l = l0 * keep0;
      if (both) l = fmaf(l1, keep1, l);
      d0 = (2 * w + half) * (kDim / 4);
      d1 = d0 + kDim / 4;
    }
    const int64_t orow = static_cast<int64_t>(wk.s.q0 + row) * a.heads + wk.head;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int prow = (two ? w : 0) * kTile + tid;
    if (warp_live) {
#pragma unroll 1
      for (int d = d0; d < d1; d += 16) {
        uint32_t r[16];
        tmem_ld16(quad + col_o(two ? w : 0) + d, r);
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
        if (live && split) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4 *>(a.part_o + ((static_cast<int64_t>(pslot) * (kDim / 4) + d / 4 + j) * 256 + prow) * 4) =
                make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        } else if (live) {
          T *out = static_cast<T *>(a.out) + orow * kDim + d;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = l == 0.f ? 0.f : __uint_as_float(r[8 * j + k]) * inv;
            *reinterpret_cast<uint4 *>(out + 8 * j) = pack8(f, T());
          }
        }
        __syncwarp();
      }
    }
    // (from what the first row of the block does not see: the other stream may have taken
    // elements out that all rows of this one see; added twice they are what they are)
    const int hidden = a.causal ? min(max(wk.s.past + 2 * wk.block * kTile + 1, 0), len) : len;
    if (live && *reinterpret_cast<volatile unsigned *>(&c.bad_piece) >= piece)
      repair_row<T>(a, wk.s, wk.head, max(wk.t0 * kTok, hidden), min(wk.t1 * kTok, seen), d0, d1,
                    split ? a.part_o + (static_cast<int64_t>(pslot) * (kDim / 4) * 256 + prow) * 4 : nullptr,
                    static_cast<T *>(a.out) + orow * kDim);
    if (live && half == 0 && (two || w == 0)) {
      if (split)
        a.part_ml[static_cast<int64_t>(pslot) * 256 + prow] = make_float2(m, l);
      else if (a.lse)
        a.lse[orow] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * 0.69314718055994530942f;
    }
    // the second share of a split block describes it to the join
    if (wk.t0 > 0 && threadIdx.x == 0) {
      const int first = wk.share_of(0, c.per);
      if (static_cast<int>(blockIdx.x) == first + 1) {
        Join j;
        j.rows0 = wk.s.q0;
        j.row0 = 2 * wk.block * kTile;
        j.rows = min(wk.s.rows - j.row0, 2 * kTile);
        j.head = wk.head;
        j.first_cta = first;
        j.last_cta = wk.share_of(wk.tiles - 1, c.per);
        a.joins[blockIdx.x] = j;
      }
    }
    fence_before();
    if (!two)
      bar_all();  // all have read O before any goes on
    else
      bar_rows(w, q);
    fence_after();
    wk.advance(a);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                  const __grid_constant__ CUtensorMap rm, const __grid_constant__ CUtensorMap vm,
                  const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Ctrl &c = *reinterpret_cast<Ctrl *>(smem);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    prefetch_tensormap(&qm);
    prefetch_tensormap(&km);
    prefetch_tensormap(&rm);
    prefetch_tensormap(&vm);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 2);
    }
    mbar_init(&c.q_full, 1);
    mbar_init(&c.q_empty, 2);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&c.s_full[w], 1);
      mbar_init(&c.s_free[w], 8);
      mbar_init(&c.p_ready[w], 8);
      mbar_init(&c.p_free[w], 1);
      mbar_init(&c.o_full[w], 1);
    }
    fence_mbar_init();
    c.bad_piece = 0;
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) a.joins[blockIdx.x].rows = 0;  // no block begins to be split here, unless the epilogue says so
  make_plan<T>(a, c);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = c.tmem;
  if (warp < 16) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    softmax<T>(a, c, smem, tmem, warp >> 3);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == 16)
      producer(a, c, smem, &qm, &km, &rm, &vm);
    else if (warp < 19)
      mma_issuer<T>(a, c, smem, tmem, warp - 17);
  }
  fence_before();
  __syncthreads();
  if (warp == 17) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------- join --
// Blocks cut by CTA boundaries: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// over the pieces in order (the same bits every time).  One CTA per boundary and
// 32 rows; lane = row, warp = an eighth of the head.
template <typename T>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ Args a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Join j = a.joins[blockIdx.x];
  const int prow = blockIdx.y * 32 + (threadIdx.x & 31);
  if (prow >= j.rows) return;
  constexpr int kPer = kDim / 8 / 4;
  const int d4 = (threadIdx.x >> 5) * kPer;
  float M = -CUDART_INF_F, l = 0.f;
  float4 o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x = j.first_cta; x <= j.last_cta; ++x) {
    const int64_t s = 2 * x + (x == j.first_cta ? 1 : 0);
    const float2 ml = a.part_ml[s * 256 + prow];
    const float top = fmaxf(M, ml.x), mm = top == -CUDART_INF_F ? 0.f : top;
    const float old = exp2f(M - mm), keep = exp2f(ml.x - mm);
    M = top;
    l = fmaf(ml.y, keep, l * old);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float4 v = *reinterpret_cast<const float4 *>(a.part_o + ((s * (kDim / 4) + d4 + i) * 256 + prow) * 4);
      o[i].x = fmaf(v.x, keep, o[i].x * old), o[i].y = fmaf(v.y, keep, o[i].y * old);
      o[i].z = fmaf(v.z, keep, o[i].z * old), o[i].w = fmaf(v.w, keep, o[i].w * old);
    }
  }
  const int64_t orow = (j.rows0 + j.row0 + prow) * a.heads + j.head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *out = static_cast<T *>(a.out) + orow * kDim + 4 * d4;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool none = l == 0.f;
    const uint32_t lo = pack2(none ? 0.f : o[i].x * inv, none ? 0.f : o[i].y * inv, T());
    const uint32_t hi = pack2(none ? 0.f : o[i].z * inv, none ? 0.f : o[i].w * inv, T());
    *reinterpret_cast<uint2 *>(out + 4 * i) = make_uint2(lo, hi);
  }
  if (threadIdx.x < 32 && a.lse) a.lse[orow] = l == 0.f ? -CUDART_INF_F : (M + log2f(l)) * 0.69314718055994530942f;
}

// ----------------------------------------------------------------- launch --
template <typename T>
int launch(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &rm, const CUtensorMap &vm, const Args &a, int ctas,
           cudaStream_t stream) {
  static int configured[64] = {0};
  int dev = 0;
  B200KV_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return set_error(B200KV_ERR_UNSUPPORTED, "device ordinal %d", dev);
  if (!__atomic_load_n(&configured[dev], __ATOMIC_ACQUIRE)) {
    B200KV_CUDA_TRY(cudaFuncSetAttribute(prompt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    __atomic_store_n(&configured[dev], 1, __ATOMIC_RELEASE);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, prompt_kernel<T>, qm, km, rm, vm, a));
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 8);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  B200KV_CUDA_TRY(cudaLaunchKernelEx(&cfg, prompt_join_kernel<T>, a));
  return B200KV_OK;
}

}  // namespace prompt
}  // namespace b200kv
