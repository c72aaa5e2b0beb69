// Raw keys -> the basis the cache stores, shared by every kernel that puts keys into it (the page and tail
// writers, the draft commit) or scores keys that are not in it yet (the tree attention's drafts).
#pragma once

#include "../../include/bdfp4.h"
#include "common.cuh"

namespace bdfp4 {

template <int SHIFT_TYPE>
__device__ __forceinline__ void load_shift16(const void* shift, int64_t offset, float* out) {
  if (SHIFT_TYPE == BDFP4_SHIFT_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(shift) + offset);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldg(p + i);
      out[4 * i] = v.x;
      out[4 * i + 1] = v.y;
      out[4 * i + 2] = v.z;
      out[4 * i + 3] = v.w;
    }
  } else if (SHIFT_TYPE == BDFP4_SHIFT_BF16) {
    load_bf16x16(static_cast<const __nv_bfloat16*>(shift) + offset, out);
  }
}

// Raw K -> the basis the cache stores: rotate, scale by 1/sqrt(128), subtract the shift, round
// to BF16 once. The multiply and the subtract round separately
// (src/nvfp4_decode_kernel/quantize_kv_kernel.py:123-162).
template <int SHIFT_TYPE, bool ROTATE>
__device__ __forceinline__ void cache_basis16(float* v, int group, const void* shift, int64_t shift_offset) {
  if (ROTATE) {
    hadamard_butterflies(v, group);
    const float inverse = (float)0.08838834764831845;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fmul_rn(v[j], inverse);
  }
  if (SHIFT_TYPE != BDFP4_SHIFT_NONE) {
    float centre[16];
    load_shift16<SHIFT_TYPE>(shift, shift_offset, centre);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fsub_rn(v[j], centre[j]);
  }
  if (ROTATE || SHIFT_TYPE != BDFP4_SHIFT_NONE) round_to_bf16(v);
}

// The same with the rotation and an FP32 shift chosen at run time, in one copy of the code. `shift` points at
// this group's sixteen values, or is null.
__device__ __forceinline__ void cache_basis16_any(float* v, int group, bool rotate, const float* shift) {
  if (rotate) {
    hadamard_butterflies(v, group);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fmul_rn(v[j], (float)0.08838834764831845);
  }
  if (shift) {
    float centre[16];
    load_shift16<BDFP4_SHIFT_F32>(shift, 0, centre);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fsub_rn(v[j], centre[j]);
  }
  round_to_bf16(v);
}

}  // namespace bdfp4
