// What the two tree attention kernels share: the work list, waits, tensor-memory and conversion helpers.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "host.h"
#include "key_basis.cuh"
#include "tcgen05.cuh"
#include "tree_params.h"

namespace bdfp4 {
namespace tree {

constexpr int kStage = 18432;  // K codes 8192, V codes 8192, K scales 1024, V scales 1024
constexpr int kVOffset = 8192, kKsOffset = 16384, kVsOffset = 17408;
// A BF16 step (tail, or sink and drafts) takes one stage per 64 tokens for K, then as many for V; a token's
// 256 bytes lie 272 apart, so that eight rows' 16-byte chunks fall on distinct banks.
constexpr int kBf16Pitch = 272, kBf16Rows = 64;
constexpr float kNoMax = -3.0e38f;  // a query that has seen no token yet
constexpr float kShift = 7.0f;      // probabilities carry 2^7
constexpr float kGrowth = 8.0f;     // a maximum is renewed when a score exceeds it by more than this (log2)

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ bool bar_any(int id, bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(out)
      : "r"((uint32_t)pred), "r"(id)
      : "memory");
  return out != 0;
}

// kind::f16 with A in tensor memory (lane = row, a 32-bit column = two neighbouring K values).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// FP32 accumulate; A K-major; B K-major (queries) or MN-major (probabilities, bit 16); operand format 0 FP16, 1 BF16.
__host__ __device__ constexpr uint32_t f16_idesc(int n, int format, bool b_mn_major) {
  return (1u << 4) | ((uint32_t)format << 7) | ((uint32_t)format << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void st16(uint32_t address, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::
          "r"(address),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void st8(uint32_t address, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(address), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t address, float* v) {
  if constexpr (N == 8) tc::tmem_ld8(address, v);
#pragma unroll
  for (int j = 0; j + 16 <= N; j += 16) tc::tmem_ld16(address + j, v + j);
}

__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// Eight E2M1 codes times one FP16 scale -> eight FP16 values in four words, in code order. Exact.
__device__ __forceinline__ void dequantize8(uint32_t codes, __half2 scale, uint32_t* out) {
  uint32_t v[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = h2(__hmul2(*reinterpret_cast<__half2*>(&v[i]), scale));
}

// Two E4M3 bytes -> two FP16 pairs (scale, scale).
__device__ __forceinline__ void scale_pairs(uint32_t bytes, __half2* out) {
  uint32_t both;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(both) : "r"(bytes));
  const __half2 pair = *reinterpret_cast<__half2*>(&both);
  out[0] = __low2half2(pair);
  out[1] = __high2half2(pair);
}

// The power of two that brings `amax` into [2^TO, 2^(TO + 1)), and its inverse. Zero, infinite or NaN: 1.
template <int TO>
__device__ __forceinline__ float scale_to(float amax, float* inverse) {
  const int e = (int)((__float_as_uint(amax) >> 23) & 0xffu);
  if (e == 0 || e == 255) {
    *inverse = 1.0f;
    return 1.0f;
  }
  const int field = min(127 + TO + 127 - e, 253);
  *inverse = __uint_as_float((uint32_t)(254 - field) << 23);
  return __uint_as_float((uint32_t)field << 23);
}

struct RowInfo {
  int count, pages, residual, sink, slot;  // pages: 128-token steps in the FP4 cache
  int steps;                               // of one unit: pages, tail, drafts with sink
  int tiles;
};

__device__ __forceinline__ RowInfo row_info(const TreeParams& p, int row, int page_tokens) {
  RowInfo r;
  r.count = p.node_counts ? min(max(p.node_counts[row], 0), p.nodes) : p.nodes;
  const int entries = kPage / page_tokens;
  r.pages = min(max(p.seqused_fp4[row], 0) / kPage, p.max_pages / entries);
  r.residual = r.sink = r.slot = 0;
  if (p.tail_key) {
    r.slot = p.slot_ids[row];
    if (r.slot >= 0 && r.slot < p.tail_slots) {
      r.residual = min(max(p.residual[row], 0), kPage);
      if (p.sink) r.sink = min(max(p.sink[row], 0), BDFP4_MAX_SINK);
    } else {
      r.slot = 0;
    }
  }
  r.steps = r.pages + (r.residual > 0 ? 1 : 0) + 1;
  r.tiles = (r.count * p.ratio + p.tile - 1) / p.tile;
  return r;
}

struct Unit {
  RowInfo info;
  int row, head, tile, begin, end;  // steps [begin, end) of the unit are this CTA's
};

enum StepKind { kStepPage, kStepTail, kStepDraft };

__device__ __forceinline__ StepKind step_kind(const RowInfo& r, int step) {
  return step < r.pages ? kStepPage : (step == r.pages && r.residual > 0) ? kStepTail : kStepDraft;
}
// Token places of a BF16 step: the tail's tokens, or 16 places of the sink and the drafts behind them.
__device__ __forceinline__ int bf16_places(const RowInfo& r, StepKind kind) {
  return kind == kStepTail ? r.residual : BDFP4_MAX_SINK + r.count;
}
__device__ __forceinline__ int bf16_stages(const RowInfo& r, StepKind kind) {  // of each side
  return (bf16_places(r, kind) + kBf16Rows - 1) / kBf16Rows;
}
// 16-token slices of a step that hold anything.
__device__ __forceinline__ int step_slices(const RowInfo& r, StepKind kind) {
  return kind == kStepPage ? 8 : (bf16_places(r, kind) + 15) / 16;
}

// The units of this CTA in order; every role walks them on its own. Steps are counted in 32 bits within a
// row (the host refuses larger rows).
struct Walker {
  const TreeParams& p;
  int row, page_tokens, offset, left;
  __device__ Walker(const TreeParams& params, int start_row, int start_offset, int steps, int pt)
      : p(params), row(start_row), page_tokens(pt), offset(start_offset), left(steps) {}
  // `known`: u is a unit of this walk, so its row's lengths need not be read again.
  __device__ __forceinline__ bool next(Unit& u, bool known) {
    if (left <= 0) return false;
    while (true) {
      if (!known || u.row != row) u.info = row_info(p, row, page_tokens);
      const int whole = u.info.steps * u.info.tiles * p.heads_kv;
      if (offset < whole) break;
      offset -= whole;
      known = false;
      if (++row >= p.rows) return false;
    }
    const int unit = offset / u.info.steps;
    u.row = row;
    u.head = unit / u.info.tiles;
    u.tile = unit - u.head * u.info.tiles;
    u.begin = offset - unit * u.info.steps;
    u.end = min(u.info.steps, u.begin + left);
    left -= u.end - u.begin;
    offset += u.end - u.begin;
    return true;
  }
};

// Waiting is a dozen instructions, one when the phase is already over. After about two seconds, or once another thread has given
// up, a wait ends without its phase; the roles go through the rest of their motions and the kernel reports it.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, int* abort_flag) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 begin, now;\n\t.reg .b32 given_up;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
      "@p bra OVER;\n\t"
      "mov.u64 begin, %%globaltimer;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
      "@p bra OVER;\n\t"
      "ld.volatile.shared.b32 given_up, [%2];\n\t"
      "setp.ne.b32 p, given_up, 0;\n\t"
      "@p bra OVER;\n\t"
      "mov.u64 now, %%globaltimer;\n\t"
      "sub.u64 now, now, begin;\n\t"
      "setp.lt.u64 p, now, %3;\n\t"
      "@p bra AGAIN;\n\t"
      "st.volatile.shared.b32 [%2], 1;\n"
      "OVER:\n\t}" ::"r"(tc::smem_u32(bar)),
      "r"(parity), "r"(tc::smem_u32(abort_flag)), "n"(tc::kWaitLimitNs)
      : "memory");
}

// One thread of a converged warp. tcgen05.mma takes its descriptors from uniform registers: behind an elected
// predicate the warp's control flow stays uniform for the compiler, and an MMA issues in 32 (N = 64) to 64
// cycles (N = 128), its tensor time; behind a test of the lane number it took 140 whatever its size.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(elected));
  return elected != 0;
}

// Thirty-two codes and the scales of their two groups into sixteen columns of this thread's lane.
__device__ __forceinline__ void store_dequantized(uint32_t a, uint4 chunk, uint32_t scales) {
  __half2 scale[2];
  scale_pairs(scales, scale);
  uint32_t v[16];
  dequantize8(chunk.x, scale[0], v);
  dequantize8(chunk.y, scale[0], v + 4);
  dequantize8(chunk.z, scale[1], v + 8);
  dequantize8(chunk.w, scale[1], v + 12);
  st16(a, v);
}

// Sums of N per-lane columns over the warp: every exchange halves what a lane holds, until it holds N / 32 (at
// least one) columns, which go to `store(column, sum)`.
template <int N, int MASK, typename Store>
__device__ __forceinline__ void reduce_columns(float* v, int lane, int column, Store store) {
  if constexpr (MASK == 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) store(column + j, v[j]);
  } else if constexpr (N % 2 == 0) {
    const bool upper = (lane & MASK) != 0;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const float keep = upper ? v[j + N / 2] : v[j], send = upper ? v[j] : v[j + N / 2];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, send, MASK);
    }
    reduce_columns<N / 2, MASK / 2>(v, lane, column + (upper ? N / 2 : 0), store);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], MASK);
    reduce_columns<N, MASK / 2>(v, lane, column, store);
  }
}

}  // namespace tree
}  // namespace bdfp4
