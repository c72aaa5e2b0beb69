// The accepted path of a drafted tree into the BF16 tail and sink of every layer.
//
// Token p of a sequence lives at row p % 128 of its slot's rolling page, so the a accepted nodes of a row of
// n committed tokens go to rows n % 128 .. (n + a - 1) % 128: a gather of whole K/V rows by node number, with
// K brought into the cache's basis on the way. Bound by HBM (2 x 512 bytes read and written per token and
// head; 64 rows x 32 layers x 8 heads of up to 16 tokens: 27 us, 0.81 of a plain copy's rate), or by the launch for
// small batches. At most 64 nodes make at most one page boundary per row; the
// page that fills is sealed by the page writers between a HEAD and a REST call, since the tokens behind the
// boundary reuse the rows that the seal still has to read.
#include "common.cuh"
#include "host.h"
#include "key_basis.cuh"

namespace bdfp4 {

struct CommitParams {
  int layers, rows, nodes, heads;
  const __nv_bfloat16* key;
  const __nv_bfloat16* value;
  int64_t key_layer, key_row, key_node, value_layer, value_row, value_node;
  const int32_t* accepted;
  int64_t accepted_stride;
  const int32_t* counts;
  const int32_t* seq_lens;
  const int32_t* row_to_slot;
  __nv_bfloat16* tail_key;
  __nv_bfloat16* tail_value;
  int64_t tail_layer, tail_slot;
  int slots, sink, part;
  const float* shift;
  const int32_t* table;
  int64_t table_stride;
  int max_pages, pages, page_tokens;
  int32_t* new_seq_lens;
  int32_t* fp4;
  int32_t* residual;
  int32_t* sink_out;
  int32_t* source_tokens;
  int32_t* destinations;
  int32_t* error_word;
};

constexpr int kCommitThreads = 256;
// Groups of 16 channels per thread: all their loads are issued before the first store. One row of 16
// nodes, 8 heads and both sides is 4096 groups, four CTAs.
constexpr int kCommitPerThread = 4;

// The row's new lengths and its entries of the seal's work table.
__device__ __forceinline__ void commit_lengths(const CommitParams& p, int row, int n, int count, bool live, int slot) {
  const int total = live ? n + count : n;
  const int fp4 = total > 0 ? (total - 1) / kPage * kPage : 0;
  p.new_seq_lens[row] = total;
  p.fp4[row] = fp4;
  p.residual[row] = total - fp4;
  p.sink_out[row] = min(total, p.sink);
  const bool fills = live && total / kPage > n / kPage;
  if (!p.source_tokens) return;
  // (every entry is written, whatever the table holds: the page writers follow what stands here)
  const int entries = kPage / p.page_tokens;
  for (int e = 0; e < entries; ++e) {
    const int column = (total / kPage - 1) * entries + e;
    int page = -1;
    if (fills) {
      if (column < p.max_pages) page = p.table[(int64_t)row * p.table_stride + column];
      if (page < 0 || page >= p.pages) {
        page = -1;
        if (p.error_word) atomicOr(p.error_word, (int)BDFP4_DEV_BAD_PAGE);
      }
    }
    p.source_tokens[row * entries + e] = live ? slot * (kPage + p.sink) + e * p.page_tokens : 0;
    p.destinations[row * entries + e] = page;
  }
}

template <int SHIFT_TYPE, bool ROTATE>
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const CommitParams p) {
  const int row = blockIdx.y, layer = blockIdx.z;
  const int slot = p.row_to_slot[row];
  const int n = p.seq_lens[row];
  const bool live = slot >= 0 && slot < p.slots && n >= 0;
  // The path ends at the first entry that is not a node's number: the tokens behind it have nothing to be written
  // from, and a length that counted them would make old rows of the tail part of the sequence. (Every warp looks for it.)
  const int claimed = min(max(p.counts[row], 0), p.nodes);
  int count = claimed;
#pragma unroll
  for (int half = 1; half >= 0; --half) {
    const int i = 32 * half + (threadIdx.x & 31);
    const int node = i < p.nodes ? p.accepted[(int64_t)row * p.accepted_stride + i] : 0;
    const unsigned bad = __ballot_sync(0xffffffffu, i < claimed && (node < 0 || node >= p.nodes));
    if (bad) count = 32 * half + __ffs(bad) - 1;
  }
  if (blockIdx.x == 0 && layer == 0 && threadIdx.x == 0 && p.part != BDFP4_COMMIT_REST) {
    commit_lengths(p, row, n, count, live, slot);
    if (live && count < claimed && p.error_word) atomicOr(p.error_word, (int)BDFP4_DEV_BAD_NODE);
  }
  if (!live) return;
  const int boundary = (n + count) / kPage * kPage;
  const bool fills = boundary > n / kPage * kPage;
  // accepted tokens this call writes: [first, last)
  int first = 0, last = count;
  if (p.part == BDFP4_COMMIT_HEAD && fills) last = boundary - n;
  if (p.part == BDFP4_COMMIT_REST) first = fills ? boundary - n : count;
  const int groups = p.heads * kGroupsPerVec;  // of one token and side; eight lanes hold one head
  const int items = (last - first) * 2 * groups;
  const int begin = blockIdx.x * kCommitThreads * kCommitPerThread;
  if (begin >= items) return;
  const int64_t row_elems = (int64_t)p.heads * kHeadDim;

  uint4 raw[kCommitPerThread][2];
  int64_t to[kCommitPerThread];  // element offset inside a tail buffer, or -1
  int to_sink[kCommitPerThread];
#pragma unroll
  for (int k = 0; k < kCommitPerThread; ++k) {
    const int item = begin + k * kCommitThreads + threadIdx.x;
    to[k] = -1;
    raw[k][0] = raw[k][1] = make_uint4(0, 0, 0, 0);
    if (item < items) {
      const int token = first + item / (2 * groups);
      const int within = item % (2 * groups);
      const bool is_key = within < groups;
      const int channel = (is_key ? within : within - groups) * kGroup;  // head and channel in one
      const int node = p.accepted[(int64_t)row * p.accepted_stride + token];
      const __nv_bfloat16* src = is_key ? p.key + layer * p.key_layer + row * p.key_row + node * p.key_node
                                        : p.value + layer * p.value_layer + row * p.value_row + node * p.value_node;
      raw[k][0] = __ldg(reinterpret_cast<const uint4*>(src + channel));
      raw[k][1] = __ldg(reinterpret_cast<const uint4*>(src + channel) + 1);
      const int position = n + token;
      to[k] = (int64_t)slot * p.tail_slot + (position % kPage) * row_elems + channel;
      to_sink[k] = position < p.sink ? kPage + position - position % kPage : 0;  // rows between the two places
    }
  }
#pragma unroll
  for (int k = 0; k < kCommitPerThread; ++k) {
    const int item = begin + k * kCommitThreads + threadIdx.x;
    const int within = item % (2 * groups);
    const bool is_key = within < groups;
    uint4 out0 = raw[k][0], out1 = raw[k][1];
    if (ROTATE || SHIFT_TYPE != BDFP4_SHIFT_NONE) {
      // every lane takes part: the rotation exchanges channels among the eight lanes of a head
      float v[16];
      const uint32_t w[8] = {out0.x, out0.y, out0.z, out0.w, out1.x, out1.y, out1.z, out1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
      const int channel = is_key ? within * kGroup : 0;
      cache_basis16<SHIFT_TYPE, ROTATE>(v, within % kGroupsPerVec, p.shift, layer * row_elems + channel);
      if (is_key) {
        out0 = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                          pack_bf16x2(v[6], v[7]));
        out1 = make_uint4(pack_bf16x2(v[8], v[9]), pack_bf16x2(v[10], v[11]), pack_bf16x2(v[12], v[13]),
                          pack_bf16x2(v[14], v[15]));
      }
    }
    if (to[k] >= 0) {
      __nv_bfloat16* dst = (is_key ? p.tail_key : p.tail_value) + layer * p.tail_layer + to[k];
      reinterpret_cast<uint4*>(dst)[0] = out0;
      reinterpret_cast<uint4*>(dst)[1] = out1;
      if (to_sink[k]) {
        dst += to_sink[k] * row_elems;
        reinterpret_cast<uint4*>(dst)[0] = out0;
        reinterpret_cast<uint4*>(dst)[1] = out1;
      }
    }
  }
}

}  // namespace bdfp4

using namespace bdfp4;

extern "C" int bdfp4_commit_drafts(const bdfp4_commit_args* a, void* stream_handle) {
  if (!a) return BDFP4_E_ARG;
  if (a->layers < 1 || a->rows < 1 || a->heads_kv < 1 || a->nodes < 1) return BDFP4_E_ARG;
  if (a->nodes > BDFP4_MAX_TREE_NODES || a->rows > 65535 || a->layers > 65535) return BDFP4_E_UNSUPPORTED;
  if (!a->draft_key || !a->draft_value || !a->accepted || !a->accepted_counts || !a->seq_lens || !a->row_to_slot ||
      !a->tail_key || !a->tail_value)
    return BDFP4_E_ARG;
  if (a->part < BDFP4_COMMIT_ALL || a->part > BDFP4_COMMIT_REST) return BDFP4_E_ARG;
  if (a->sink_tokens < 0 || a->sink_tokens > BDFP4_MAX_SINK || a->tail_slots < 1) return BDFP4_E_ARG;
  auto misaligned = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) != 0; };
  if (misaligned(a->draft_key) || misaligned(a->draft_value) || misaligned(a->tail_key) || misaligned(a->tail_value) ||
      misaligned(a->key_shift))
    return BDFP4_E_ARG;
  for (int64_t stride : {a->key_layer_stride, a->key_row_stride, a->key_node_stride, a->value_layer_stride,
                         a->value_row_stride, a->value_node_stride, a->tail_layer_stride, a->tail_slot_stride})
    if (stride % 8) return BDFP4_E_ARG;
  if (a->part != BDFP4_COMMIT_REST &&
      (!a->new_seq_lens || !a->seqused_fp4 || !a->seqused_residual || !a->seqused_sink))
    return BDFP4_E_ARG;
  const int page_tokens = a->page_tokens == 0 ? kPage : a->page_tokens;
  if (page_tokens != 128 && page_tokens != 64) return BDFP4_E_UNSUPPORTED;
  if (!a->source_tokens != !a->destination_pages) return BDFP4_E_ARG;
  if (a->source_tokens ? a->max_pages_per_row < 0 || a->pages < 1 || (!a->page_table && a->max_pages_per_row > 0)
                       : a->page_table != nullptr)
    return BDFP4_E_ARG;
  CommitParams p{};
  p.layers = a->layers;
  p.rows = a->rows;
  p.nodes = a->nodes;
  p.heads = a->heads_kv;
  p.key = static_cast<const __nv_bfloat16*>(a->draft_key);
  p.value = static_cast<const __nv_bfloat16*>(a->draft_value);
  p.key_layer = a->key_layer_stride;
  p.key_row = a->key_row_stride;
  p.key_node = a->key_node_stride;
  p.value_layer = a->value_layer_stride;
  p.value_row = a->value_row_stride;
  p.value_node = a->value_node_stride;
  p.accepted = a->accepted;
  p.accepted_stride = a->accepted_row_stride;
  p.counts = a->accepted_counts;
  p.seq_lens = a->seq_lens;
  p.row_to_slot = a->row_to_slot;
  p.tail_key = static_cast<__nv_bfloat16*>(a->tail_key);
  p.tail_value = static_cast<__nv_bfloat16*>(a->tail_value);
  p.tail_layer = a->tail_layer_stride;
  p.tail_slot = a->tail_slot_stride;
  p.slots = a->tail_slots;
  p.sink = a->sink_tokens;
  p.part = a->part;
  p.shift = a->key_shift;
  p.table = a->page_table;
  p.table_stride = a->page_table_stride;
  p.max_pages = a->max_pages_per_row;
  p.pages = a->pages;
  p.page_tokens = page_tokens;
  p.new_seq_lens = a->new_seq_lens;
  p.fp4 = a->seqused_fp4;
  p.residual = a->seqused_residual;
  p.sink_out = a->seqused_sink;
  p.source_tokens = a->source_tokens;
  p.destinations = a->destination_pages;
  p.error_word = a->error_word;
  const int64_t items = (int64_t)a->nodes * 2 * a->heads_kv * kGroupsPerVec;
  const int per_cta = kCommitThreads * kCommitPerThread;
  const dim3 grid((unsigned)((items + per_cta - 1) / per_cta), a->rows, a->layers);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (a->rotate && a->key_shift)
    commit_kernel<BDFP4_SHIFT_F32, true><<<grid, kCommitThreads, 0, stream>>>(p);
  else if (a->rotate)
    commit_kernel<BDFP4_SHIFT_NONE, true><<<grid, kCommitThreads, 0, stream>>>(p);
  else if (a->key_shift)
    commit_kernel<BDFP4_SHIFT_F32, false><<<grid, kCommitThreads, 0, stream>>>(p);
  else
    commit_kernel<BDFP4_SHIFT_NONE, false><<<grid, kCommitThreads, 0, stream>>>(p);
  return bdfp4::cuda_status(cudaGetLastError());
}
