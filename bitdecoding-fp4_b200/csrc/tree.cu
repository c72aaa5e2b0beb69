// C ABI of the tree attention: argument checks, the tile and its instantiation (tree_p128.cu, tree_p64.cu),
// and the kernel that adds the parts of units that straddle CTAs. The attention itself is
// tree_narrow.cuh and tree_wide.cuh.
#include <algorithm>
#include <cmath>
#include <utility>

#include "common.cuh"
#include "decode_params.h"
#include "host.h"
#include "tree_params.h"

namespace bdfp4 {

// The query rows of one KV head are cut into as few tiles as hold them, and those made as even as the built
// widths allow: a wider tile converts the cache for more queries at once, an empty column costs its share of the
// products and exponentials. Up to 32 queries go to the kernel of two CTAs per SM (331 us against 430 for 16 rows x
// 65536 tokens under 32 queries per KV head), wider tiles to the one of one (82 against 120 us for 16 rows x 8192
// under 64).
static int tree_tile(int queries) {
  const int tiles = (queries + kTreeMaxTile - 1) / kTreeMaxTile;
  const int each = (queries + tiles - 1) / tiles;
  for (int tile : {16, 32, 64, 96})
    if (each <= tile) return tile;
  return kTreeMaxTile;
}

constexpr int kMaxHeads = 65535;  // what a row's query rows are counted in 32 bits for

static int tree_ctas(int tile) { return tile <= kTreeNarrowTile ? kTreeNarrowCtas : kTreeWideCtas; }

// One block per (CTA that a straddling unit begins in, eight query rows). First the parts' weights 2^(their
// maximum - the largest) for each row, by 16 x GROUPS threads; then GROUPS threads per channel add every
// GROUPS-th part each. It is latency that counts: for a single row's 66 parts (one token over 8192) the launch
// took 0.8 us a part with one thread per channel that weighed each part against the ones before, 0.6 us with the
// weights known before, 0.25 us with four. Wide tiles, of fewer parts and more blocks, take two.
constexpr int kMergeRows = 8;

__device__ __forceinline__ float merge_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS) tree_merge_kernel(const TreeParams p) {
  __shared__ float weight[kTreeNarrowCtas][kMergeRows];
  constexpr int kRowThreads = 16 * GROUPS, kRowWarps = GROUPS / 2;
  __shared__ float stat_of[kRowWarps][kMergeRows];  // by warp: maxima, then weights
  __shared__ float sums[GROUPS - 1][kMergeRows][kHeadDim];
  wait_for_prior_kernels();
  const int cta = blockIdx.x;
  const TreeSplit split = p.splits[cta];
  if (split.row < 0) return;
  const int count = p.node_counts ? min(max(p.node_counts[split.row], 0), p.nodes) : p.nodes;
  const int first = blockIdx.y * kMergeRows;
  const int rows = min(min(count * p.ratio - split.tile * p.tile, p.tile) - first, kMergeRows);
  if (rows <= 0) return;
  const int parts = split.last - cta + 1;
  auto part = [&](int i) { return 2 * (cta + i) + (i == 0 ? 1 : 0); };
  float total = 0.0f;
  const int row = threadIdx.x / kRowThreads, lane = threadIdx.x % kRowThreads;  // (rows behind the tile's last repeat it)
  {
    const float* const stat = p.partial_stat + first + min(row, rows - 1);
    float top = -3.0e38f;
    for (int i = lane; i < parts; i += kRowThreads) {
      const float m = __ldcg(stat + (int64_t)(2 * part(i)) * p.tile);
      weight[i][row] = m;
      top = fmaxf(top, m);
    }
    for (int step = 16; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
    if ((lane & 31) == 0) stat_of[lane >> 5][row] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, stat_of[w][row]);
    __syncthreads();
    for (int i = lane; i < parts; i += kRowThreads) {
      const float w = merge_ex2(weight[i][row] - top);
      weight[i][row] = w;
      total += w * __ldcg(stat + (int64_t)(2 * part(i) + 1) * p.tile);
    }
    for (int step = 16; step > 0; step >>= 1) total += __shfl_xor_sync(0xffffffffu, total, step);
    if ((lane & 31) == 0) stat_of[lane >> 5][row] = total;
  }
  __syncthreads();
  const int channel = threadIdx.x & 127, group = threadIdx.x >> 7;
  float acc[kMergeRows];
#pragma unroll
  for (int r = 0; r < kMergeRows; ++r) acc[r] = 0.0f;
#pragma unroll 4
  for (int i = group; i < parts; i += GROUPS) {
    const float* value = p.partial + ((int64_t)part(i) * p.tile + first) * kHeadDim + channel;
#pragma unroll
    for (int r = 0; r < kMergeRows; ++r) acc[r] += __ldcg(value + r * kHeadDim) * weight[i][r];
  }
  if (group > 0) {
#pragma unroll
    for (int r = 0; r < kMergeRows; ++r) sums[group - 1][r][channel] = acc[r];
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int r = 0; r < kMergeRows; ++r) {
    if (r < rows) {
      float weights = 0.0f;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) weights += stat_of[w][r];
      float sum = acc[r];
#pragma unroll
      for (int g = 0; g < GROUPS - 1; ++g) sum += sums[g][r][channel];
      const int query = split.tile * p.tile + first + r;
      p.out[split.row * p.out_row + (query / p.ratio) * p.out_node +
            (int64_t)(split.head * p.ratio + query % p.ratio) * kHeadDim + channel] =
          __float2bfloat16_rn(sum * (weights > 0.0f ? p.value_scale / weights : 0.0f));
    }
  }
}

template <int GROUPS>
static cudaError_t launch_merge(const TreeParams& p, cudaStream_t stream) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(p.ctas, (p.tile + kMergeRows - 1) / kMergeRows);
  config.blockDim = dim3(128 * GROUPS);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, tree_merge_kernel<GROUPS>, p);
}

}  // namespace bdfp4

using namespace bdfp4;

extern "C" int64_t bdfp4_tree_workspace_bytes(int32_t rows, int32_t nodes, int32_t heads_q, int32_t heads_kv) {
  if (rows < 1 || nodes < 1 || nodes > BDFP4_MAX_TREE_NODES || heads_kv < 1 || heads_q < 1 || heads_q % heads_kv ||
      heads_q > kMaxHeads)
    return 0;
  const int64_t tile = tree_tile(nodes * (heads_q / heads_kv));
  return (int64_t)tree_ctas((int)tile) * (2 * tile * (kHeadDim + 2) * (int64_t)sizeof(float) + (int64_t)sizeof(TreeSplit));
}

// Whether the blocks of `size` elements of a two-dimensional grid share none, one dimension wholly inside the other.
static bool apart(int64_t n0, int64_t stride0, int64_t n1, int64_t stride1, int64_t size) {
  if (n0 == 1 || n1 == 1) return n0 * n1 == 1 || (n0 == 1 ? stride1 : stride0) >= size;
  if (stride0 < stride1) std::swap(n0, n1), std::swap(stride0, stride1);
  return stride1 >= size && stride0 >= (n1 - 1) * stride1 + size;
}

extern "C" int bdfp4_tree_decode(const bdfp4_tree_args* a, void* stream_handle) {
  if (!a) return BDFP4_E_ARG;
  if (a->rows < 1 || a->nodes < 1 || a->heads_q < 1 || a->heads_kv < 1 || a->heads_q % a->heads_kv) return BDFP4_E_ARG;
  if (a->nodes > BDFP4_MAX_TREE_NODES || a->rows > 65535 || a->heads_q > kMaxHeads) return BDFP4_E_UNSUPPORTED;
  if (!a->query || !a->draft_key || !a->draft_value || !a->parents || !a->out) return BDFP4_E_ARG;
  if (!a->key_codes || !a->key_scales || !a->value_codes || !a->value_scales || a->pages < 1 ||
      (!a->page_table && a->max_pages_per_row > 0) || !a->seqused_fp4 || a->max_pages_per_row < 0 ||
      a->page_table_stride < a->max_pages_per_row)
    return BDFP4_E_ARG;
  auto misaligned = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) != 0; };
  for (const void* ptr : {a->query, a->draft_key, a->draft_value, a->key_codes, a->key_scales, a->value_codes,
                          a->value_scales, a->tail_key, a->tail_value, (const void*)a->key_shift, (const void*)a->out})
    if (misaligned(ptr)) return BDFP4_E_ARG;
  for (int64_t stride : {a->query_row_stride, a->query_node_stride, a->draft_key_row_stride, a->draft_key_node_stride,
                         a->draft_value_row_stride, a->draft_value_node_stride, a->tail_slot_stride, a->out_row_stride,
                         a->out_node_stride})
    if (stride % 8 || stride < 0) return BDFP4_E_ARG;
  if (a->parents_row_stride < 0 ||
      !apart(a->rows, a->out_row_stride, a->nodes, a->out_node_stride, (int64_t)a->heads_q * kHeadDim))
    return BDFP4_E_ARG;
  const int page_tokens = a->page_tokens == 0 ? kPage : a->page_tokens;
  if (page_tokens != 128 && page_tokens != 64) return BDFP4_E_UNSUPPORTED;
  // the kernel counts one row's and one CTA's steps (128 tokens of one head and tile of queries) in 32 bits
  const int64_t tiles = ((int64_t)a->nodes * (a->heads_q / a->heads_kv) + 15) / 16;
  const int64_t row_steps = ((int64_t)a->max_pages_per_row * page_tokens / kPage + 2) * tiles * a->heads_kv;
  if (row_steps > INT32_MAX || row_steps * a->rows / kTreeWideCtas >= INT32_MAX - 64) return BDFP4_E_UNSUPPORTED;
  const int64_t head_codes = (int64_t)page_tokens * 64, head_scales = (int64_t)page_tokens * 8;
  if (a->key_codes_pitch % 16 || a->key_scales_pitch % 16 || a->value_codes_pitch % 16 || a->value_scales_pitch % 16 ||
      a->key_codes_pitch < a->heads_kv * head_codes || a->value_codes_pitch < a->heads_kv * head_codes ||
      a->key_scales_pitch < a->heads_kv * head_scales || a->value_scales_pitch < a->heads_kv * head_scales)
    return BDFP4_E_ARG;
  if (a->tail_key && (!a->tail_value || !a->tail_slot_ids || !a->seqused_residual || a->tail_slots < 1 ||
                      a->tail_slot_stride < (int64_t)kPage * a->heads_kv * kHeadDim))
    return BDFP4_E_ARG;
  if (!(a->softmax_scale > 0.0f) || !std::isfinite(a->softmax_scale)) return BDFP4_E_ARG;
  auto bad_scale = [](float s) { return s != 0.0f && !(s > 0.0f && std::isfinite(s)); };
  if (bad_scale(a->key_tensor_scale) || bad_scale(a->value_tensor_scale)) return BDFP4_E_ARG;
  const int64_t need = bdfp4_tree_workspace_bytes(a->rows, a->nodes, a->heads_q, a->heads_kv);
  if (need > 0 && (!a->workspace || misaligned(a->workspace) || a->workspace_bytes < need)) return BDFP4_E_ARG;

  TreeParams p{};
  p.rows = a->rows;
  p.nodes = a->nodes;
  p.heads_q = a->heads_q;
  p.heads_kv = a->heads_kv;
  p.ratio = a->heads_q / a->heads_kv;
  p.query = static_cast<const __nv_bfloat16*>(a->query);
  p.query_row = a->query_row_stride;
  p.query_node = a->query_node_stride;
  p.draft_key = static_cast<const __nv_bfloat16*>(a->draft_key);
  p.draft_value = static_cast<const __nv_bfloat16*>(a->draft_value);
  p.draft_key_row = a->draft_key_row_stride;
  p.draft_key_node = a->draft_key_node_stride;
  p.draft_value_row = a->draft_value_row_stride;
  p.draft_value_node = a->draft_value_node_stride;
  p.parents = a->parents;
  p.parents_row = a->parents_row_stride;
  p.node_counts = a->node_counts;
  p.codes[0] = static_cast<const uint8_t*>(a->key_codes);
  p.codes[1] = static_cast<const uint8_t*>(a->value_codes);
  p.scales[0] = static_cast<const uint8_t*>(a->key_scales);
  p.scales[1] = static_cast<const uint8_t*>(a->value_scales);
  p.codes_pitch[0] = a->key_codes_pitch;
  p.codes_pitch[1] = a->value_codes_pitch;
  p.scales_pitch[0] = a->key_scales_pitch;
  p.scales_pitch[1] = a->value_scales_pitch;
  p.pages = a->pages;
  p.table = a->page_table;
  p.table_stride = a->page_table_stride;
  p.max_pages = a->max_pages_per_row;
  p.rotate = a->rotate;
  p.seqused_fp4 = a->seqused_fp4;
  p.tail_key = static_cast<const __nv_bfloat16*>(a->tail_key);
  p.tail_value = static_cast<const __nv_bfloat16*>(a->tail_value);
  p.tail_slot = a->tail_slot_stride;
  p.tail_slots = a->tail_slots;
  p.slot_ids = a->tail_slot_ids;
  p.residual = a->seqused_residual;
  p.sink = a->tail_key ? a->seqused_sink : nullptr;
  p.sink_rows = a->tail_key ? (int)std::min<int64_t>(a->tail_slot_stride / ((int64_t)a->heads_kv * kHeadDim) - kPage, BDFP4_MAX_SINK) : 0;
  p.key_shift = a->key_shift;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.key_scale = a->key_tensor_scale == 0.0f ? 1.0f : a->key_tensor_scale;
  p.value_scale = a->value_tensor_scale == 0.0f ? 1.0f : a->value_tensor_scale;
  p.inverse_value_scale = 1.0f / p.value_scale;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.out_row = a->out_row_stride;
  p.out_node = a->out_node_stride;
  p.error_word = a->error_word;
  p.tile = tree_tile(a->nodes * p.ratio);
  p.ctas = tree_ctas(p.tile);
  p.partial = static_cast<float*>(a->workspace);
  p.partial_stat = p.partial + (int64_t)2 * p.ctas * p.tile * kHeadDim;
  p.splits = reinterpret_cast<TreeSplit*>(p.partial_stat + (int64_t)4 * p.ctas * p.tile);
  CUtensorMap k_map{}, v_map{};
  if (page_tokens == 128 && !cache_tensor_maps(a->key_codes, a->value_codes, a->heads_kv, page_tokens, a->pages,
                                               a->key_codes_pitch, a->value_codes_pitch, &k_map, &v_map))
    return BDFP4_E_CUDA;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  cudaError_t e = page_tokens == 128 ? launch_tree_p128(k_map, v_map, p, stream) : launch_tree_p64(k_map, v_map, p, stream);
  if (e == cudaSuccess) e = p.tile <= kTreeNarrowTile ? launch_merge<4>(p, stream) : launch_merge<2>(p, stream);
  return bdfp4::cuda_status(e);
}
