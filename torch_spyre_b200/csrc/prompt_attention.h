// Arguments of the prompt-attention kernels (latent attention, expanded form).
#pragma once

#include "common.cuh"

namespace b200kv {
namespace prompt {

constexpr int kMaxCtas = 148;  // shares of a launch: one CTA per SM of a B200
constexpr int kNope = B200KV_LATENT_NOPE, kRope = B200KV_LATENT_ROPE, kDim = B200KV_LATENT_NOPE;

// A block of rows whose token tiles are spread over CTAs first_cta .. last_cta;
// its partials are in slot 2 * first_cta + 1 and then in slots 2 * cta.
struct Join {
  int64_t rows0;
  int row0, rows, head, first_cta, last_cta, pad;
};

struct Args {
  const int32_t *q_indptr, *kv_indptr;
  const void *v;
  int64_t v_st, v_sh;
  void *out;  // contiguous [N, H, 128]
  float *lse;
  int total_q, total_kv, batch, heads, causal;
  float scale;
  int32_t *error_flag;
  Join *joins;      // [CTAs]
  float2 *part_ml;  // [2 * CTAs][256] (maximum in log2 units, sum)
  float *part_o;    // [2 * CTAs][32][256][4]
};

}  // namespace prompt
}  // namespace b200kv
