// Arguments of the tree-attention kernels and their launchers (one translation
// unit per compute type).
#pragma once

#include "common.cuh"

namespace b200kv {
namespace tree {

constexpr int kMaxCtas = 148;  // shares of a launch: one CTA per SM of a B200

// A block of rows whose token tiles are spread over CTAs first_cta .. last_cta;
// its partials are in slot 2 * first_cta + 1 and then in slots 2 * cta.
struct Join {
  int64_t rows0;
  int node0, nodes, kvh, first_cta, last_cta, pad;
};

struct Args {
  const int32_t *block_table;
  int64_t bt_stride;
  const int32_t *ctx, *indptr;
  const uint64_t *mask;  // [N, words], null: a chain
  int64_t words;
  const float *k_scales, *v_scales;
  const void *k_pool, *v_pool;
  void *out;  // contiguous [N, Hq, D]
  float *lse;
  int total_q, batch, hq, hkv, group, max_blocks, max_nodes, num_blocks;
  int tile_nodes;        // nodes of a Q tile: floor(128 / group)
  int box_nodes;         // nodes of a TMA box of Q
  int small_boxes;       // the boxes are of 32 rows, as many as are needed; else one box a tile
  uint32_t q_box_bytes;  // bytes of a box
  float scale;
  int32_t *error_flag;
  Join *joins;      // [CTAs]
  float2 *part_ml;  // [2 * CTAs][256] (maximum in log2 units, sum)
  float *part_o;    // [2 * CTAs][D / 4][256][4] (8-bit caches: divided by the sum)
};

int launch_f16(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, const Args &a, int dim, int cache,
               int ctas, cudaStream_t stream);
int launch_bf16(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, const Args &a, int dim, int cache,
                int ctas, cudaStream_t stream);

}  // namespace tree
}  // namespace b200kv
