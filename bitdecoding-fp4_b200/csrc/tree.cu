// Attention of a tree of drafted tokens over the paged NVFP4 cache.
//
// One CTA holds eight query rows (node x query head) of one (row, KV head) and walks the row's tokens 128 at
// a time: FP4 pages, then the BF16 rolling tail, then drafts and sink together. Thread t scores token t with
// FP32 FMAs, the running maximum and sum are kept per query row, and thread c accumulates channel c.
#include <cmath>

#include "common.cuh"
#include "host.h"
#include "key_basis.cuh"

namespace bdfp4 {

struct TreeParams {
  int rows, nodes, heads_q, heads_kv, ratio;
  const __nv_bfloat16* query;
  int64_t query_row, query_node;
  const __nv_bfloat16* draft_key;
  const __nv_bfloat16* draft_value;
  int64_t draft_key_row, draft_key_node, draft_value_row, draft_value_node;
  const int32_t* parents;
  int64_t parents_row;
  const int32_t* node_counts;
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  int64_t codes_pitch[2], scales_pitch[2];
  int pages, page_tokens;
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
  const float* key_shift;
  float scale_log2;  // softmax scale in log2 units
  float key_scale, value_scale;
  __nv_bfloat16* out;
  int64_t out_row, out_node;
  int32_t* error_word;
};

constexpr int kTreeRows = 8;

__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__global__ void __launch_bounds__(128) tree_kernel(const TreeParams p) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int row = blockIdx.z, head = blockIdx.y, first = blockIdx.x * kTreeRows;
  const int count = p.node_counts ? min(max(p.node_counts[row], 0), p.nodes) : p.nodes;
  const int queries = count * p.ratio;
  if (first >= queries) return;
  __shared__ float q[kTreeRows][kHeadDim];
  __shared__ float prob[kTreeRows][128];
  __shared__ float red[4][kTreeRows];
  __shared__ __nv_bfloat16 drafts[BDFP4_MAX_TREE_NODES][kHeadDim + 8];
  __shared__ uint64_t family[BDFP4_MAX_TREE_NODES];

  {  // eight lanes hold one query row or one draft key
    const int group = t & 7;
    for (int base = 0; base < kTreeRows; base += 16) {
      const int r = base + (t >> 3);
      float v[16];
      const int query = min(first + min(r, kTreeRows - 1), queries - 1);
      load_bf16x16(p.query + row * p.query_row + (query / p.ratio) * p.query_node +
                       (head * p.ratio + query % p.ratio) * kHeadDim + group * kGroup, v);
      if (p.rotate) {
        hadamard_butterflies(v, group);
        for (int j = 0; j < 16; ++j) v[j] *= kInvSqrt128;
      }
      if (r < kTreeRows)
        for (int j = 0; j < 16; ++j) q[r][group * kGroup + j] = v[j];
    }
    for (int base = 0; base < count; base += 16) {
      const int node = base + (t >> 3);
      float v[16];
      load_bf16x16(p.draft_key + row * p.draft_key_row + min(node, count - 1) * p.draft_key_node + head * kHeadDim +
                       group * kGroup, v);
      if (p.rotate && p.key_shift) cache_basis16<BDFP4_SHIFT_F32, true>(v, group, p.key_shift, head * kHeadDim + group * kGroup);
      else if (p.rotate) cache_basis16<BDFP4_SHIFT_NONE, true>(v, group, nullptr, 0);
      else if (p.key_shift) cache_basis16<BDFP4_SHIFT_F32, false>(v, group, p.key_shift, head * kHeadDim + group * kGroup);
      if (node < count) store_bf16x16(&drafts[node][group * kGroup], v);
    }
    if (t == 0) {
      for (int i = 0; i < count; ++i) {
        const int parent = p.parents[row * p.parents_row + i];
        family[i] = (1ull << i) | (parent >= 0 && parent < i ? family[parent] : 0ull);
      }
    }
  }
  __syncthreads();

  const int entries = kPage / p.page_tokens;
  const int fp4 = min(max(p.seqused_fp4[row], 0) / kPage, p.max_pages / entries) * kPage;
  int slot = 0, residual = 0, sink = 0;
  if (p.tail_key) {
    slot = p.slot_ids[row];
    if (slot >= 0 && slot < p.tail_slots) {
      residual = min(max(p.residual[row], 0), kPage);
      sink = p.sink ? min(max(p.sink[row], 0), BDFP4_MAX_SINK) : 0;
    }
  }
  const int64_t tail_row = (int64_t)p.heads_kv * kHeadDim;
  float top[kTreeRows], sum[kTreeRows], acc[kTreeRows];
  for (int r = 0; r < kTreeRows; ++r) top[r] = -INFINITY, sum[r] = 0.0f, acc[r] = 0.0f;
  const int steps = fp4 / kPage + 2;
  for (int step = 0; step < steps; ++step) {
    const int kind = step < fp4 / kPage ? 0 : step == fp4 / kPage ? 1 : 2;
    float s[kTreeRows];
    for (int r = 0; r < kTreeRows; ++r) s[r] = 0.0f;
    bool valid;
    auto page_of = [&](int token) {
      int page = p.table[row * p.table_stride + (int64_t)step * entries + token / p.page_tokens];
      if (page < 0 || page >= p.pages) {
        if (p.error_word) atomicOr(p.error_word, (int)BDFP4_DEV_BAD_PAGE);
        page = 0;
      }
      return (int64_t)page;
    };
    if (kind == 0) {
      valid = step > 0 || t >= sink;
      const int64_t page = page_of(t);
      const int tok = t % p.page_tokens;
      const uint8_t* codes = p.codes[0] + page * p.codes_pitch[0];
      const uint8_t* scales = p.scales[0] + page * p.scales_pitch[0];
      for (int g = 0; g < 8; ++g) {
        uint32_t scale, lo, hi;
        if (p.page_tokens == 128) {
          const uint2 w = *reinterpret_cast<const uint2*>(codes + (tok * p.heads_kv + head) * 64 + g * 8);
          lo = w.x, hi = w.y;
          scale = scales[head * 1024 + scale_tile_offset(tok, g)];
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(codes + head * 4096 + tok * 64 + (((g >> 1) ^ ((tok >> 1) & 3)) * 16) + (g & 1) * 8);
          lo = w.x, hi = w.y;
          scale = scales[head * 512 + (g >> 2) * 256 + (tok & 31) * 8 + (tok >> 5) * 4 + (g & 3)];
        }
        const float f = e4m3_to_float(scale) * p.key_scale;
        for (int b = 0; b < 8; ++b) {
          const float2 k = e2m1x2_to_float2((b < 4 ? lo : hi) >> (8 * (b & 3)));
          for (int r = 0; r < kTreeRows; ++r)
            s[r] = fmaf(k.x * f, q[r][g * 16 + 2 * b], fmaf(k.y * f, q[r][g * 16 + 2 * b + 1], s[r]));
        }
      }
    } else {
      const __nv_bfloat16* key;
      if (kind == 1) {
        valid = t < residual && (fp4 > 0 || t >= sink);
        key = p.tail_key + slot * p.tail_slot + t * tail_row + head * kHeadDim;
      } else if (t < BDFP4_MAX_TREE_NODES) {
        valid = t < count;
        key = drafts[valid ? t : 0];
      } else {
        valid = t - BDFP4_MAX_TREE_NODES < sink;
        key = p.tail_key + slot * p.tail_slot + (kPage + t - BDFP4_MAX_TREE_NODES) * tail_row + head * kHeadDim;
      }
      if (valid)
        for (int c = 0; c < kHeadDim; ++c) {
          const float k = __bfloat162float(key[c]);
          for (int r = 0; r < kTreeRows; ++r) s[r] = fmaf(k, q[r][c], s[r]);
        }
    }
    for (int r = 0; r < kTreeRows; ++r) {
      bool seen = valid;
      if (kind == 2 && t < BDFP4_MAX_TREE_NODES) seen = valid && (family[min((first + r) / p.ratio, count - 1)] >> t & 1);
      s[r] = seen ? s[r] * p.scale_log2 : -INFINITY;
      float m = s[r];
      for (int step2 = 16; step2 > 0; step2 >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, step2));
      if (lane == 0) red[warp][r] = m;
    }
    __syncthreads();
    for (int r = 0; r < kTreeRows; ++r) {
      const float m = fmaxf(fmaxf(fmaxf(red[0][r], red[1][r]), fmaxf(red[2][r], red[3][r])), top[r]);
      const float base = m == -INFINITY ? 0.0f : m;
      const float back = tree_ex2(top[r] - base);
      const float e = tree_ex2(s[r] - base);
      top[r] = m;
      sum[r] = sum[r] * back + e;
      acc[r] *= back;
      prob[r][t] = e;
    }
    __syncthreads();
    if (kind == 0) {
      for (int part = 0; part < entries; ++part) {
        const int64_t page = page_of(part * p.page_tokens);
        const uint8_t* codes = p.codes[1] + page * p.codes_pitch[1];
        const uint8_t* scales = p.scales[1] + page * p.scales_pitch[1];
        for (int g = 0; g < p.page_tokens / 16; ++g) {
          uint2 w;
          uint32_t scale;
          if (p.page_tokens == 128) {
            w = *reinterpret_cast<const uint2*>(codes + (head * kHeadDim + t) * 64 + g * 8);
            scale = scales[head * 1024 + scale_tile_offset(t, g)];
          } else {
            w = *reinterpret_cast<const uint2*>(codes + head * 4096 + t * 32 + (((g >> 1) ^ ((t >> 2) & 1)) * 16) + (g & 1) * 8);
            scale = scales[head * 512 + scale_tile_offset(t, g)];
          }
          const float f = e4m3_to_float(scale) * p.value_scale;
          for (int b = 0; b < 8; ++b) {
            const float2 v = e2m1x2_to_float2((b < 4 ? w.x : w.y) >> (8 * (b & 3)));
            const int token = part * p.page_tokens + g * 16 + 2 * b;
            for (int r = 0; r < kTreeRows; ++r)
              acc[r] = fmaf(v.x * f, prob[r][token], fmaf(v.y * f, prob[r][token + 1], acc[r]));
          }
        }
      }
    } else {
      const int tokens = kind == 1 ? residual : count;
      for (int token = 0; token < tokens; ++token) {
        const __nv_bfloat16* value = kind == 1 ? p.tail_value + slot * p.tail_slot + token * tail_row
                                               : p.draft_value + row * p.draft_value_row + token * p.draft_value_node;
        const float v = __bfloat162float(value[head * kHeadDim + t]);
        for (int r = 0; r < kTreeRows; ++r) acc[r] = fmaf(v, prob[r][token], acc[r]);
      }
      for (int token = 0; kind == 2 && token < sink; ++token) {
        const float v = __bfloat162float(p.tail_value[slot * p.tail_slot + (kPage + token) * tail_row + head * kHeadDim + t]);
        for (int r = 0; r < kTreeRows; ++r) acc[r] = fmaf(v, prob[r][BDFP4_MAX_TREE_NODES + token], acc[r]);
      }
    }
    __syncthreads();
  }
  for (int r = 0; r < kTreeRows; ++r) {
    for (int step = 16; step > 0; step >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], step);
    if (lane == 0) red[warp][r] = sum[r];
  }
  __syncthreads();
  for (int r = 0; r < kTreeRows && first + r < queries; ++r) {
    const float total = red[0][r] + red[1][r] + red[2][r] + red[3][r];
    const int query = first + r;
    p.out[row * p.out_row + (query / p.ratio) * p.out_node + (head * p.ratio + query % p.ratio) * kHeadDim + t] =
        __float2bfloat16_rn(total > 0.0f ? acc[r] / total : 0.0f);
  }
}

}  // namespace bdfp4

using namespace bdfp4;

extern "C" int64_t bdfp4_tree_workspace_bytes(int32_t rows, int32_t nodes, int32_t heads_q, int32_t heads_kv) {
  if (rows < 1 || nodes < 1 || nodes > BDFP4_MAX_TREE_NODES || heads_kv < 1 || heads_q < 1 || heads_q % heads_kv) return 0;
  return 16;
}

extern "C" int bdfp4_tree_decode(const bdfp4_tree_args* a, void* stream_handle) {
  if (!a) return BDFP4_E_ARG;
  if (a->rows < 1 || a->nodes < 1 || a->heads_q < 1 || a->heads_kv < 1 || a->heads_q % a->heads_kv) return BDFP4_E_ARG;
  if (a->nodes > BDFP4_MAX_TREE_NODES || a->rows > 65535 || a->heads_kv > 65535) return BDFP4_E_UNSUPPORTED;
  if (!a->query || !a->draft_key || !a->draft_value || !a->parents || !a->out) return BDFP4_E_ARG;
  if (!a->key_codes || !a->key_scales || !a->value_codes || !a->value_scales || a->pages < 1 || !a->page_table ||
      !a->seqused_fp4 || a->max_pages_per_row < 0 || a->page_table_stride < a->max_pages_per_row)
    return BDFP4_E_ARG;
  auto misaligned = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) != 0; };
  for (const void* ptr : {a->query, a->draft_key, a->draft_value, a->key_codes, a->key_scales, a->value_codes,
                          a->value_scales, a->tail_key, a->tail_value, (const void*)a->key_shift, (const void*)a->out})
    if (misaligned(ptr)) return BDFP4_E_ARG;
  for (int64_t stride : {a->query_row_stride, a->query_node_stride, a->draft_key_row_stride, a->draft_key_node_stride,
                         a->draft_value_row_stride, a->draft_value_node_stride, a->tail_slot_stride, a->out_row_stride,
                         a->out_node_stride})
    if (stride % 8 || stride < 0) return BDFP4_E_ARG;
  if (a->out_node_stride < (int64_t)a->heads_q * kHeadDim || a->parents_row_stride < 0) return BDFP4_E_ARG;
  const int page_tokens = a->page_tokens == 0 ? kPage : a->page_tokens;
  if (page_tokens != 128 && page_tokens != 64) return BDFP4_E_UNSUPPORTED;
  const int64_t head_codes = (int64_t)page_tokens * 64, head_scales = (int64_t)page_tokens * 8;
  if (a->key_codes_pitch % 16 || a->key_scales_pitch % 16 || a->value_codes_pitch % 16 || a->value_scales_pitch % 16 ||
      a->key_codes_pitch < a->heads_kv * head_codes || a->value_codes_pitch < a->heads_kv * head_codes ||
      a->key_scales_pitch < a->heads_kv * head_scales || a->value_scales_pitch < a->heads_kv * head_scales)
    return BDFP4_E_ARG;
  if (a->tail_key && (!a->tail_value || !a->tail_slot_ids || !a->seqused_residual || a->tail_slots < 1 ||
                      a->tail_slot_stride < (int64_t)(kPage + (a->seqused_sink ? BDFP4_MAX_SINK : 0)) * a->heads_kv * kHeadDim))
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
  p.page_tokens = page_tokens;
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
  p.key_shift = a->key_shift;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.key_scale = a->key_tensor_scale == 0.0f ? 1.0f : a->key_tensor_scale;
  p.value_scale = a->value_tensor_scale == 0.0f ? 1.0f : a->value_tensor_scale;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.out_row = a->out_row_stride;
  p.out_node = a->out_node_stride;
  p.error_word = a->error_word;
  const int queries = a->nodes * p.ratio;
  tree_kernel<<<dim3((queries + kTreeRows - 1) / kTreeRows, a->heads_kv, a->rows), 128, 0,
                static_cast<cudaStream_t>(stream_handle)>>>(p);
  return bdfp4::cuda_status(cudaGetLastError());
}
