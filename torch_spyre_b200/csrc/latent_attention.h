// Arguments of the latent-attention kernels.
#pragma once

#include "common.cuh"

namespace b200kv {
namespace latent {

constexpr int kRank = B200KV_LATENT_RANK, kRope = B200KV_LATENT_ROPE, kRow = kRank + kRope;
constexpr int kSticks = kRow / 64;
constexpr int kMaxCtas = 148;  // one CTA per SM of a B200
constexpr int kTileRows = 64;  // rows of q that a CTA holds
constexpr int kMaxHeads = 512;

// A block of rows whose token tiles are spread over shares first .. last; its
// partials are in slot 2 * cta + 1 of the first share's CTA and slots 2 * cta of
// the others'.
struct Join {
  int64_t rows0;  // first row of q of the sequence
  int node0, nodes, head0, first, last, pad;
};

struct Args {
  const int32_t *block_table;
  int64_t bt_stride;
  const int32_t *ctx, *indptr;
  const uint64_t *mask;  // [N, words], null: a chain
  int64_t words;
  const void *pool;
  void *out;  // contiguous [N, H, 512]
  float *lse;
  int total_q, batch, heads, max_blocks, max_nodes, num_blocks;
  int stride;       // CTAs of a share: they walk the same blocks, each with rows of its own
  int head_box;     // heads of a Q tile (a CTA's rows)
  int tile_nodes;   // nodes of a Q tile
  int block_nodes;  // nodes of a block
  int box_nodes;   // nodes of a TMA box of Q (no more than a sequence can have)
  float scale;
  int32_t *error_flag;
  Join *joins;      // [CTAs]
  float2 *part_ml;  // [2 * CTAs][64] (maximum in log2 units, sum)
  float *part_o;    // [2 * CTAs][64][512], from pairs of SMs [2 * CTAs][128][64][4]
};

}  // namespace latent
}  // namespace b200kv
