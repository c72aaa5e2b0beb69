// Launch parameters of the tree attention kernel and the entry points of its instantiation units. The kernels.
// Their templates (tree_narrow.cuh, tree_wide.cuh) are instantiated in two translation units (128- and 64-token pages);
// tree.cu holds the C ABI and the merge kernel.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace bdfp4 {

// CTAs of a launch: two per SM of a B200 for tiles of at most kTreeNarrowTile queries, else one. They share
// nothing but the workspace, so any number is correct.
constexpr int kTreeNarrowCtas = 296, kTreeWideCtas = 148;
constexpr int kTreeNarrowTile = 32;
constexpr int kTreeMaxTile = 128;  // query rows (node x query head of one KV head) of a CTA's tile at most

// A unit that begins in CTA c and does not end there: its parts lie in slot 2c + 1 and in slots 2c' of the
// CTAs c < c' <= last.
struct TreeSplit {
  int row, head, tile, last;  // row < 0: none
};

struct TreeParams {
  int rows, nodes, heads_q, heads_kv, ratio;
  int tile;  // query rows per tile
  int ctas;
  const __nv_bfloat16* query;
  int64_t query_row, query_node;
  const __nv_bfloat16* draft_key;
  const __nv_bfloat16* draft_value;
  int64_t draft_key_row, draft_key_node, draft_value_row, draft_value_node;
  const int32_t* parents;
  int64_t parents_row;
  const int32_t* node_counts;
  const uint8_t* codes[2];  // K, V: bulk copies of 64-token pages
  const uint8_t* scales[2];
  int64_t codes_pitch[2], scales_pitch[2];
  int pages;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  int rotate;
  const int32_t* seqused_fp4;
  const __nv_bfloat16* tail_key;
  const __nv_bfloat16* tail_value;
  int64_t tail_slot;
  int tail_slots;
  const int32_t* slot_ids;
  const int32_t* residual;
  const int32_t* sink;
  int sink_rows;  // of a slot, 0 to 16
  const float* key_shift;
  float scale_log2;  // softmax scale in log2 units
  float key_scale;   // key tensor scale of the pages
  float value_scale, inverse_value_scale;
  __nv_bfloat16* out;
  int64_t out_row, out_node;
  float* partial;  // [2 * ctas][tile][128] sums, then [2 * ctas][2][tile] maxima and weights
  float* partial_stat;
  TreeSplit* splits;  // [ctas]
  int32_t* error_word;
};

cudaError_t launch_tree_p128(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream);
cudaError_t launch_tree_p64(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream);

}  // namespace bdfp4
