// Latent attention for blocks of up to 128 rows, on pairs of SMs (latent_mma.cuh
// has what the two kernels share, and the one for up to 64 rows).
//
// With 64 rows on one SM the products are bound by shared memory: a page's scores
// and values read 4 + 6 KB of operands where the tensor core needs half the time
// for them.  So two CTAs of a cluster work as one (cta_group::2): each holds 64 of
// the 128 rows and gives half of every product's other operand,
//   S [128 rows, 128 tokens]  = Q K^T    each CTA one of two pages: its own tokens
//   O [128 rows, 512]        += P V      each CTA half of the latent elements
// at 32 and 64 clocks a product of 16, 2176 for 128 tokens, where its own operands
// take 4 and 6 KB.  (One SM with 64 rows: 3800 clocks for 128 tokens.)  32 sequences of up
// to 8192 tokens (170 MB), 128 heads: 64 us, 66 among other work; first pieces run at HBM's rate (3300 clocks a step),
// 5 us pass before their first loads and 3 us at each piece's end, most of them 128 KB of
// partials a CTA.  8 trees of up to 8 nodes over up to 16384 tokens: 103 us, 2400 clocks a step, 117
// in long runs, in which the power limit lowers the clock.
//
// A step's keys are read as they arrive, half a page at a time, and their slots freed at
// once; its values, half of the elements of both pages, come again (out of L2) when the
// weights are there.  So four slots of 32 KB keep the products fed.
//
// An accumulator of 128 rows over two CTAs lies in each of them as 64 rows: lanes 0-63
// have the first half of the columns, lanes 64-127 the second.  Warp w has the lanes of
// quadrant w % 4, so rows 32 (w % 2) .. and half (w / 2) % 2 of a step's tokens and of
// O's columns, and of those columns the first or second part by w / 4.
//
// Warps: 0-7 softmax and output, 8 TMA producer; in the first CTA 9 issues the scores'
// MMAs for both, 10 the values'; in the second 11 tells the first of its arrivals.
#pragma once

#include "latent_mma.cuh"

namespace b200kv {
namespace latent {
namespace pair {

constexpr int kStep = 2 * kPageTokens;  // tokens of a step
constexpr int kSlots = 4, kSlot = 2 * kPair;
constexpr int kAhead = 1;  // steps that pages are in L2 before they are loaded (32 sequences: 61.4 us, with 2 64.4, with none 69.5)
constexpr int kOffQ = 3 * 1024;
constexpr int kOffP = kOffQ + kSticks * kStickTile;  // [2 pages][64 rows][64 tokens]
constexpr int kOffRope = kOffP + 2 * kStickTile;
constexpr int kOffSlots = kOffRope + kStickTile;
constexpr int kSmem = kOffSlots + kSlots * kSlot;
static_assert(kSmem <= 227 * 1024, "shared memory per CTA");

// TMEM columns of a CTA: O, 128 for each 256 latent elements, and two score buffers
__device__ __forceinline__ uint32_t col_o(int j) { return uint32_t(j) * 128u; }
__device__ __forceinline__ uint32_t col_s(uint32_t b) { return 256u + b * 64u; }

struct Ctrl {
  // each CTA's own: what has arrived, what is free again, what is computed
  uint64_t full[kSlots], empty[kSlots], rope_empty, q_full, q_empty;
  uint64_t s_full[2], p_free, o_full;
  // the first CTA's: the second's arrivals, and both CTAs' weights and outputs
  uint64_t peer[kSlots], q_peer, p_ready[2], o_empty;
  uint32_t tmem;
  Plan plan;
  float top[4][kTileRows];  // maxima, then sums, of the quarters of a row's tokens
};
static_assert(sizeof(Ctrl) <= kOffQ, "control block");

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// (Relaxed: what has to be seen across the pair is fenced, or has been waited for.  A
// release would wait for the partials' stores as well: 1000 clocks and more.)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
// After a wait that ran out: this thread's arrivals at the other CTA's barriers have landed.
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// An arrival at the first CTA's barrier.  What it tells of lies in shared memory, written
// by the copy engine or behind fence.proxy.async, and is read by the tensor cores: the
// order of shared memory that arrival and wait give is enough.  (A release and an
// acquire of the cluster's scope order global memory too, and cost 1000 to 2000 clocks each.)
__device__ __forceinline__ void arrive_first(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, 0;\n\tmbarrier.arrive.shared::cluster.b64 _, [r];\n\t}" ::"r"(
          smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void commit_both(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(acc), "r"(go)
      : "memory");
}

// The rows of a CTA in the pair's block: nodes from node0 on, heads from head0 on.
struct Rows {
  int node0, nodes, head0;
};
__device__ __forceinline__ Rows rows_of(const Args &a, const Walk<kStep> &w) {
  const int part = static_cast<int>(blockIdx.x) % a.stride;
  Rows r;
  if (a.heads > kTileRows) {  // a node's heads over the CTAs of the share
    r.node0 = w.block;
    r.head0 = part * kTileRows;
  } else {
    r.node0 = w.block * a.block_nodes + part * a.tile_nodes;
    r.head0 = 0;
  }
  r.nodes = min(max(w.s.nodes - r.node0, 0), a.tile_nodes);
  return r;
}

// A piece's copies, in order: two halves of the keys of step t (with the first the
// rotary stick), one step ahead of two halves of the values (so keys of step i > 0 begin
// at slot 2 (2 i - 1) of the piece, values of step i of n at 2 (min(n, i + 2) + i)).
__device__ __forceinline__ void producer(const Args &a, Ctrl &c, uint8_t *smem, const CUtensorMap *qm,
                                         const CUtensorMap *rm, const CUtensorMap *hm, const CUtensorMap *pm,
                                         const CUtensorMap *sm) {
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const uint32_t q_bytes = static_cast<uint32_t>(a.box_nodes * a.head_box * 128);
  bool dead = false;
  uint32_t slots = 0, steps = 0, pieces = 0;  // issued
  Walk<kStep> w;
  w.init(a, c.plan);
  while (!dead && w.next(a)) {
    const int pages = (w.s.ctx + w.s.nodes + kPageTokens - 1) / kPageTokens;
    int window = w.t0 / 16, ids = load_ids(a, w.b, window, pages), ids_next = load_ids(a, w.b, window + 1, pages);
    int ids_before = ids;
    // (a page that these ids do not reach is not brought ahead)
    auto ahead = [&](int t) {
      if (t >= w.t1 || t / 16 > window + 1) return;
      const int id = __shfl_sync(0xffffffffu, t / 16 > window ? ids_next : ids, (2 * t + rank) & 31);
      if (lane == 2 && id >= 0) page_ahead(a, id);
    };
    wait(&c.q_empty, (pieces & 1u) ^ 1u, dead, a.error_flag);
    if ((dead = __any_sync(0xffffffffu, dead))) break;
    const Rows rows = rows_of(a, w);
    if (lane == 0) mbar_arrive_expect_tx(&c.q_full, kSticks * q_bytes);
    __syncwarp();
    if (lane < kSticks)
      tma_3d(smem + kOffQ + lane * kStickTile, lane < kSticks - 1 ? qm : rm, &c.q_full, lane < kSticks - 1 ? lane * 64 : 0,
             rows.head0, w.s.q0 + rows.node0);
    ++pieces;
    // an invalid id, and a page past the sequence's, reads past the last page: zeros
    auto page_of = [&](int have, int p) {
      const int id = __shfl_sync(0xffffffffu, have, p & 31);
      return id < 0 ? a.num_blocks : id;
    };
    // Keys: lane 0 the half `h` of a page, lane 1 with the first the rotary stick.  Values:
    // lanes 0 and 1 two sticks of a page each.
    auto load = [&](bool key, int h, int page) {
      const uint32_t s = slots % kSlots;
      const bool rope = key && h == 0;
      wait_until(
          [&] {
            const bool r = !rope || mbar_test(&c.rope_empty, (steps & 1u) ^ 1u);
            return r & mbar_test(&c.empty[s], (slots / kSlots & 1u) ^ 1u);
          },
          dead, a.error_flag);
      if ((dead = __any_sync(0xffffffffu, dead))) return;
      if (lane == 0) mbar_arrive_expect_tx(&c.full[s], kSlot + (rope ? kStickTile : 0));
      __syncwarp();
      uint8_t *to = smem + kOffSlots + s * kSlot;
      if (key) {
        if (lane == 0)
          tma_3d(to, hm, &c.full[s], 0, h * 4 * kTile, page);
        else if (lane == 1 && rope)
          tma_3d(smem + kOffRope, sm, &c.full[s], 0, (kSticks - 1) * kTile, page);
      } else if (lane < 2) {
        tma_3d(to + lane * kPair, pm, &c.full[s], 0, (4 * h + 2 * rank) * kTile, page);
      }
      __syncwarp();
      ++slots;
      steps += rope;
    };
    auto keys = [&](int t) {
      if (t / 16 > window) {  // keys lead, values follow by a step
        ids_before = ids;
        ids = ids_next;
        ids_next = load_ids(a, w.b, ++window + 1, pages);
      }
      const int page = page_of(ids, 2 * t + rank);
      load(true, 0, page);
      if (!dead) load(true, 1, page);
      ahead(t + kAhead);
    };
    keys(w.t0);
    for (int t = w.t0; t < w.t0 + kAhead; ++t) ahead(t);
    for (int t = w.t0; t < w.t1 && !dead; ++t) {
      if (t + 1 < w.t1) keys(t + 1);
      if (dead) break;
      const int page = page_of(t / 16 == window ? ids : ids_before, 2 * t + (lane & 1));
      load(false, 0, page);
      if (!dead) load(false, 1, page);
    }
    w.advance(a);
  }
  if (dead) {  // the copies under way, with a limit
    bool late = false;
    if (pieces > 0) wait(&c.q_full, (pieces - 1) & 1u, late, a.error_flag);
    for (uint32_t n = slots - min(slots, uint32_t(kSlots)); n < slots; ++n)
      wait(&c.full[n % kSlots], (n / kSlots) & 1u, late, a.error_flag);
  }
  // the last arrival that the MMAs owe this CTA: not before it may the CTA end
  if (lane == 0 && pieces > 0) {
    bool late = false;
    wait(&c.q_empty, (pieces & 1u) ^ 1u, late, a.error_flag);
  }
  __syncwarp();
}

// The second CTA's arrivals, told to the first: a lane for every slot and one for Q,
// each as often as it is filled.
__device__ __forceinline__ void relay(const Args &a, Ctrl &c) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t steps = 0, pieces = 0;
  Walk<kStep> w;
  for (w.init(a, c.plan); w.next(a); w.advance(a)) {
    steps += w.t1 - w.t0;
    ++pieces;
  }
  static_assert(kSlots == 4, "a step fills every slot once");
  uint64_t *from = lane < kSlots ? &c.full[lane] : &c.q_full;
  uint64_t *to = lane < kSlots ? &c.peer[lane] : &c.q_peer;
  uint32_t left = lane < kSlots ? steps : (lane == kSlots ? pieces : 0);
  uint32_t parity = 0, idle = 0;
  uint64_t since = 0;
  while (__any_sync(0xffffffffu, left > 0)) {
    const bool ready = left > 0 && mbar_test(from, parity);
    if (ready) {
      arrive_first(to);
      parity ^= 1u;
      --left;
    }
    if (__any_sync(0xffffffffu, ready)) {
      idle = 0;
    } else if ((++idle & 1023u) == 0) {
      const uint64_t now = global_timer_ns();
      if (idle == 1024u) since = now;
      if (__any_sync(0xffffffffu, now - since > kWaitLimitNs)) {  // (the first CTA's waits run out as well)
        if (lane == 0 && a.error_flag) atomicOr(a.error_flag, B200KV_DEVERR_TIMEOUT);
        fence_cluster();
        break;
      }
    }
  }
}

// The two MMA warps of the first CTA, converged, issue for both CTAs from an elected lane.
template <typename T>
__device__ __forceinline__ void score_issuer(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem_any) {
  const uint32_t go = elect_one(), tmem = uniform(tmem_any);
  const uint32_t idesc = kIdesc<T> | (uint32_t(128 >> 4) << 24) | (uint32_t(kStep >> 3) << 17) |
                         (a.scale < 0.f ? 1u << 13 : 0u);  // a negative scale turns Q's sign
  const uint32_t qd = desc_kmajor(smem_u32(smem + kOffQ)), rd = desc_kmajor(smem_u32(smem + kOffRope));
  const uint32_t kd = desc_kmajor(smem_u32(smem + kOffSlots));
  auto done = [&](uint64_t *bar) {
    if (go) commit_both(bar);
  };
  bool dead = false;
  uint32_t slots = 0, n = 0, pieces = 0;  // slots of the pieces before; steps; pieces
  Walk<kStep> w;
  w.init(a, c.plan);
  while (w.next(a)) {
    const int steps = w.t1 - w.t0;
    for (int i = 0; i < steps; ++i, ++n) {
      const uint32_t odd = uniform(n & 1u), at = slots + 2 * (i + max(i - 1, 0));
      const uint32_t s = tmem + col_s(0) + odd * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t slot = uniform((at + h) % kSlots), parity = (at + h) / kSlots & 1u;
        wait_until(
            [&] {
              bool ok = mbar_test(&c.full[slot], parity) & mbar_test(&c.peer[slot], parity);
              if (h == 0) {
                // this score buffer is free once the step before last has weights
                if (n >= 2) ok = ok & mbar_test(&c.p_ready[odd], ((n - 2) >> 1) & 1u);
                if (i == 0) ok = ok & mbar_test(&c.q_full, pieces & 1u) & mbar_test(&c.q_peer, pieces & 1u);
              }
              return ok;
            },
            dead, a.error_flag);
        fence_after();
        if (h == 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_pair(s, qd + ((kSticks - 1) * kStickTile + k * 32 >> 4), rd + (k * 32 >> 4), idesc, k > 0, go);
          done(&c.rope_empty);
        }
        const uint32_t k0 = kd + (slot * kSlot >> 4);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint32_t off = ((k >> 2) * kStickTile + (k & 3) * 32) >> 4;
          mma_pair(s, qd + (h * 2 * kPair >> 4) + off, k0 + off, idesc, 1, go);
        }
        done(&c.empty[slot]);
      }
      done(&c.s_full[odd]);
    }
    done(&c.q_empty);
    slots += kSlots * steps;
    ++pieces;
    w.advance(a);
  }
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ void value_issuer(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem_any) {
  constexpr uint32_t idesc = kIdesc<T> | (uint32_t(128 >> 4) << 24) | (1u << 16) | (uint32_t(256 >> 3) << 17);  // V: N-major
  const uint32_t go = elect_one(), tmem = uniform(tmem_any);
  const uint32_t pd = desc_kmajor(smem_u32(smem + kOffP));
  const uint32_t vd = (smem_u32(smem + kOffSlots) >> 4) | (uint32_t(kStickTile >> 4) << 16);
  auto done = [&](uint64_t *bar) {
    if (go) commit_both(bar);
  };
  bool dead = false;
  uint32_t slots = 0, n = 0, pieces = 0;
  Walk<kStep> w;
  w.init(a, c.plan);
  while (w.next(a)) {
    const int steps = w.t1 - w.t0;
    for (int i = 0; i < steps; ++i, ++n) {
      const uint32_t later = uniform(i > 0), at = slots + 2 * (min(steps, i + 2) + i);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t slot = uniform((at + j) % kSlots), parity = (at + j) / kSlots & 1u;
        wait_until(
            [&] {
              bool ok = mbar_test(&c.full[slot], parity) & mbar_test(&c.peer[slot], parity);
              if (j == 0) {
                ok = ok & mbar_test(&c.p_ready[n & 1u], (n >> 1) & 1u);
                if (i == 0) ok = ok & mbar_test(&c.o_empty, (pieces & 1u) ^ 1u);
              }
              return ok;
            },
            dead, a.error_flag);
        fence_after();
        const uint32_t v = vd + (slot * kSlot >> 4);
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            mma_pair(tmem + col_o(j), pd + (p * kStickTile + k * 32 >> 4), v + (p * kPair + k * 2048 >> 4), idesc,
                     p + k > 0 ? 1 : later, go);
        done(&c.empty[slot]);
      }
      done(&c.p_free);
    }
    done(&c.o_full);
    slots += kSlots * steps;
    ++pieces;
    w.advance(a);
  }
  // the last arrivals from the other CTA: not before them may this one end
  if (pieces > 0) wait(&c.o_empty, (pieces & 1u) ^ 1u, dead, a.error_flag);
  __syncwarp();
}

// This thread's columns of O, of its row, times `keep`.
static __device__ __noinline__ void rescale(uint32_t at, float keep) {
#pragma unroll 1
  for (int i = 0; i < 128; i += 16) {
    uint32_t r[16];
    tmem_ld16(at + i, r);
    wait_ld(r);
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
    tmem_st16(at + i, r);
  }
  wait_st();
}

// Softmax of the CTA's rows, and their output.
template <typename T>
__device__ __forceinline__ void softmax(const Args &a, Ctrl &c, uint8_t *smem, uint32_t tmem) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = tid & 63, half = (warp >> 1) & 1, part = warp >> 2;  // of the tokens: page `half`, 32 tokens `part`
  const int quarter = 2 * half + part;
  const uint32_t quad = tmem + (uint32_t((warp & 3) * 32) << 16);
  // (a scale of zero: too small to move a score, and -inf stays -inf)
  const float cl = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1e-37f);
  bool dead = false;
  uint32_t n = 0, slots = 0;  // steps; slots of the pieces before
  unsigned piece = 0;
  Walk<kStep> wk;
  wk.init(a, c.plan);
  while (wk.next(a)) {
    ++piece;
    const int len = wk.s.ctx + wk.s.nodes, steps = wk.t1 - wk.t0;
    const Rows r = rows_of(a, wk);
    const int node = r.node0 + row / a.head_box, head = r.head0 + row % a.head_box;
    const bool live = row < r.nodes * a.head_box && head < a.heads;
    const bool warp_live = __any_sync(0xffffffffu, live);
    // tokens before this one are seen by every row of the block
    const int common = wk.s.ctx + (a.mask ? 0 : wk.block * a.block_nodes + 1);
    float m = -CUDART_INF_F, l = 0.f;
    for (int t = wk.t0; t < wk.t1; ++t, ++n) {
      const bool first = t == wk.t0, tail = t * kStep + kStep > common;
      const uint32_t vis = tail && live ? visible32(a, wk.s, node, t * kStep + 32 * quarter) : ~0u;
      wait(&c.s_full[n & 1], (n >> 1) & 1u, dead, a.error_flag);
      fence_after();
      uint32_t s[32];
      float mt = -CUDART_INF_F;
      if (warp_live) {
        tmem_ld32(quad + col_s(n & 1) + 32 * part, s);
        wait_ld(s);
        mt = fmaf(tail ? mask_max<true>(s, vis) : mask_max<false>(s, ~0u), cl, -kWeightLog2<T>);
      }
      // the maximum is that of all quarters of the row; it moves when one has risen far enough
      if (first || any_softmax(live && mt > m + kLazyLog2)) {
        c.top[quarter][row] = mt;
        bar_softmax();
        mt = fmaxf(fmaxf(c.top[0][row], c.top[1][row]), fmaxf(c.top[2][row], c.top[3][row]));
        const bool rise = live && mt > m + (first ? 0.f : kLazyLog2);
        if (!first) {
          // O moves to the new maximum once the values before are in it
          const float keep = rise ? ex2(m - mt) : 1.f;
          l *= keep;
          wait(&c.p_free, (n - 1) & 1u, dead, a.error_flag);
          fence_after();
          if (warp_live) rescale(quad + col_o(part), keep);
        }
        if (rise) m = mt;
        bar_softmax();  // (the maxima are read)
      }
      // P is free once the values of the step before are in O
      if (n >= 1) wait(&c.p_free, (n - 1) & 1u, dead, a.error_flag);
      if (warp_live)
        l += put_weights<T>(s, cl, m, smem + kOffP + half * kStickTile + row * 128, 4 * part, row & 7, true);
      if (t * kStep + kStep > min(common, len)) {
        // (this CTA's values, half of the elements: a slot for each product, both pages)
        const uint32_t vs = slots + 2 * (min(steps, t - wk.t0 + 2) + t - wk.t0) + part;
        wait(&c.full[vs % kSlots], (vs / kSlots) & 1u, dead, a.error_flag);
        for (int p = 0; p < 2; ++p) {
          const int start = t * kStep + p * kTile;
          clean<T, 2>(smem + kOffSlots + vs % kSlots * kSlot + p * kPair, tid & 127, max(common - start, 0), len - start);
        }
      }
      fence_async_smem();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive_first(&c.p_ready[n & 1]);
    }
    slots += kSlots * steps;

    // -------------------------------------------------------- end of piece --
    const bool split = wk.t0 > 0 || wk.t1 < wk.tiles;
    const int64_t pslot = 2 * blockIdx.x + (wk.t0 > 0 ? 0 : 1);  // one of each kind per share
    const int64_t orow = static_cast<int64_t>(wk.s.q0 + node) * a.heads + head;
    c.top[quarter][row] = l;
    bar_softmax();
    l = (c.top[0][row] + c.top[1][row]) + (c.top[2][row] + c.top[3][row]);
    const float inv = split ? 1.f : (l == 0.f ? 0.f : 1.f / l);
    if (live && quarter == 0) {
      if (split)
        a.part_ml[pslot * kTileRows + row] = make_float2(m, l);
      else if (a.lse)
        a.lse[orow] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * 0.69314718055994530942f;
    }
    wait(&c.o_full, (piece - 1) & 1u, dead, a.error_flag);
    fence_after();
    // column x of product `part` is element 256 part + 128 half + x of this lane's row
    if (warp_live) {
      const int d0 = 256 * part + 128 * half;
      // (a lane's own row at a time, a store would touch 32 lines: partials lie by fours of
      // elements, neighbouring rows side by side, and outputs go through P, which is free)
      uint8_t *stage = smem + kOffP + warp * 2048;
      const unsigned lives = __ballot_sync(0xffffffffu, live);
      const int at = static_cast<int>(orow);  // (rows x heads are less than 2^31)
#pragma unroll 1
      for (int x = 0; x < 128; x += 32) {
        uint32_t o[32];
        tmem_ld32(quad + col_o(part) + x, o);
        wait_ld(o);
        if (split) {
          if (live) {
            float4 *to = reinterpret_cast<float4 *>(a.part_o) + (pslot * (kRank / 4) + (d0 + x) / 4) * kTileRows + row;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              to[j * kTileRows] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                                              __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = inv == 0.f ? 0.f : __uint_as_float(o[8 * j + k]) * inv;
            *reinterpret_cast<uint4 *>(stage + lane * 64 + ((j ^ (lane >> 1)) & 3) * 16) = pack8(f, T());
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int from = 8 * k + lane / 4, j = lane % 4;
            const int64_t to = __shfl_sync(0xffffffffu, at, from);
            const uint4 v = *reinterpret_cast<const uint4 *>(stage + from * 64 + ((j ^ (from >> 1)) & 3) * 16);
            if (lives >> from & 1u) *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + to * kRank + d0 + x + 8 * j) = v;
          }
        }
        __syncwarp();
      }
    }
    fence_before();
    bar_softmax();  // (the sums are read)
    if (lane == 0) arrive_first(&c.o_empty);
    // the second share of a split block describes it to the join
    if (wk.t0 > 0 && tid == 0) {
      const int first = wk.share_of(0, c.plan.per), share = static_cast<int>(blockIdx.x) / a.stride;
      if (share == first + 1) {
        Join j;
        j.rows0 = wk.s.q0;
        j.node0 = r.node0;
        j.nodes = r.nodes;
        j.head0 = r.head0;
        j.first = first;
        j.last = wk.share_of(wk.tiles - 1, c.plan.per);
        a.joins[blockIdx.x] = j;
      }
    }
    wk.advance(a);
  }
  if (dead) fence_cluster();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    latent_pair_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap rm,
                       const __grid_constant__ CUtensorMap hm, const __grid_constant__ CUtensorMap pm,
                       const __grid_constant__ CUtensorMap sm, const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Ctrl &c = *reinterpret_cast<Ctrl *>(smem);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    prefetch_tensormap(&qm);
    prefetch_tensormap(&rm);
    prefetch_tensormap(&hm);
    prefetch_tensormap(&pm);
    prefetch_tensormap(&sm);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 1);
      mbar_init(&c.peer[i], 1);
    }
    mbar_init(&c.rope_empty, 1);
    mbar_init(&c.q_full, 1);
    mbar_init(&c.q_empty, 1);
    mbar_init(&c.q_peer, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.s_full[i], 1);
      mbar_init(&c.p_ready[i], 2 * kSoftmaxWarps);
    }
    mbar_init(&c.p_free, 1);
    mbar_init(&c.o_full, 1);
    mbar_init(&c.o_empty, 2 * kSoftmaxWarps);
    fence_mbar_init();  // (of the cluster's scope)
  }
  __syncwarp();
  cluster_arrive();
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) a.joins[blockIdx.x].nodes = 0;  // no block begins to be split here, unless the epilogue says so
  make_plan<T, kStep>(a, c.plan);
  fence_before();
  __syncthreads();
  cluster_wait();  // both CTAs' barriers are there
  fence_after();
  const uint32_t tmem = c.tmem;
  const bool leads = cluster_rank() == 0;
  if (warp < kSoftmaxWarps)
    softmax<T>(a, c, smem, tmem);
  else if (warp == 8)
    producer(a, c, smem, &qm, &rm, &hm, &pm, &sm);
  else if (warp == 9 && leads)
    score_issuer<T>(a, c, smem, tmem);
  else if (warp == 10 && leads)
    value_issuer<T>(a, c, smem, tmem);
  else if (warp == 11 && !leads)
    relay(a, c);
  __syncwarp();
  fence_before();
  __syncthreads();
  cluster_arrive();  // neither CTA ends while the other's operands or barriers may be used
  cluster_wait();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

}  // namespace pair
}  // namespace latent
}  // namespace b200kv
