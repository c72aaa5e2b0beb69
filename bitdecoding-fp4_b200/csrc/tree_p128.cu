// Tree attention over 128-token pages.
#include "tree_kernel.cuh"

namespace bdfp4 {

cudaError_t launch_tree_p128(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream) {
  return tree::launch_tile<128>(k_map, v_map, p, stream);
}

}  // namespace bdfp4
