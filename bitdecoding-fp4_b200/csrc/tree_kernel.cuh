// Launch by tile: the instantiations of one page size.
#pragma once

#include "tree_narrow.cuh"
#include "tree_wide.cuh"

namespace bdfp4 {
namespace tree {

template <int PT>
static cudaError_t launch_tile(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream) {
  switch (p.tile) {
    case 16: return narrow::launch<16, PT>(k_map, v_map, p, stream);
    case 32: return narrow::launch<32, PT>(k_map, v_map, p, stream);
    case 64: return wide::launch<64, PT>(k_map, v_map, p, stream);
    case 96: return wide::launch<96, PT>(k_map, v_map, p, stream);
    default: return wide::launch<128, PT>(k_map, v_map, p, stream);
  }
}

}  // namespace tree
}  // namespace bdfp4
