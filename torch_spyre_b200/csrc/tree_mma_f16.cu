// Tree attention, compute type f16.
#include "tree_mma.cuh"

namespace b200kv {
namespace tree {

int launch_f16(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, const Args &a, int dim, int cache,
              int ctas, cudaStream_t stream) {
  if (cache == B200KV_I8) return launch<__half, 128, B200KV_I8>(qm, km, vm, a, ctas, stream);
  if (cache == B200KV_E4M3) return launch<__half, 128, B200KV_E4M3>(qm, km, vm, a, ctas, stream);
  return dim == 64 ? launch<__half, 64, B200KV_F16>(qm, km, vm, a, ctas, stream)
                   : launch<__half, 128, B200KV_F16>(qm, km, vm, a, ctas, stream);
}

}  // namespace tree
}  // namespace b200kv
