// The tree attention for tiles of at most 32 queries.
//
// Two CTAs share an SM, and within a CTA the same eight warps convert V and take the softmax, one after the other;
// only the copies and the products have a warp of their own each. What one CTA waits for (a product, a barrier,
// tensor memory) the other fills. With warps of one role each, side by side on every scheduler and one CTA per SM,
// 16 rows x 8 KV heads x 65536 tokens under 32 queries took 430 us; this form took 331.
//
// Thread r (of 128, twice: each half has half of the channels, tokens or queries) owns token r of S^T and channel r
// of V. A step: its scores into registers (the next step's are taken meanwhile), its half of V into tensor memory,
// the vote, the exponentials, P. Now (same case, by box) 321 to 370 us, 3.3 to 3.8 TB/s of FP4 cache, 0.50 to 0.58 of a
// plain copy's rate: some 1500 cycles a step and SM of which the tensor cores work 15% and the schedulers issue half.
// What bounds it is the chain of a step's waits (scores, output, vote; 150 to 250 cycles each), of which an SM has only
// two to overlap; a third CTA's operands do not fit the tensor memory.
#pragma once

#include "tree_common.cuh"

namespace bdfp4 {
namespace tree {
namespace narrow {

// Named barriers: one per half, and all eight working warps.
constexpr int kHalfBarrier = 1, kWorkBarrier = 3;
// How near a unit's end a cut moves there, in steps (10: 16 rows x 8 nodes x 4096 76 us instead of 62).
constexpr int kSnap = 4;
constexpr int kWorkers = kCacheThreads;    // two halves of 128
constexpr int kThreads = kWorkers + 64;    // and a warp each for copies and products
constexpr int kTmemColumns = 256;          // half of what an SM has

template <int NT>
struct Shape {
  static constexpr int kColumns = NT / 2;  // queries per thread
  // tensor memory columns
  // (the keys of a BF16 step lie where a page's product had its scales: pages come first in a unit)
  static constexpr int kS = 0, kO = NT, kV = 2 * NT, kK = kV + 64, kKs = kK, kQs = kKs + 8;
  static_assert(kK + 64 <= kTmemColumns && kQs + 8 * kTerms <= kTmemColumns, "tensor memory");
};

template <int NT>
struct Smem {
  using Sh = Shape<NT>;
  static constexpr int kStages = 4;  // as many as two CTAs' shared memory holds
  alignas(1024) uint8_t ring[kStages][kStage];
  alignas(1024) uint8_t q[2][NT * 128];            // FP16 queries: two halves of 64 channels, K-major, 128-byte swizzle
  alignas(1024) uint8_t q_codes[kTerms][NT * 64];  // FP4 terms, K-major, 64-byte swizzle
  alignas(1024) uint8_t q_scales[kTerms][1024];    // two atoms each
  alignas(1024) uint8_t p[16384];        // MN-major: 128-byte rows of 64 queries per token, swizzled
  uint32_t seen_by[2][BDFP4_MAX_TREE_NODES];  // [half] which of its columns see a draft node
  float base[NT];       // kShift - maximum, 0 while there is none
  float top[NT];        // maximum, log2 units
  float factor[NT], shift[NT];  // what a renewal does to sums and scores (at a unit's end: 1 / weight)
  float col[4][NT];             // a warp's maxima, then sums
  float level[NT];              // what brings a query's scores down to the tile's scale (in uneven tiles)
  float own[NT];
  float2 q_range[8];
  int parents[BDFP4_MAX_TREE_NODES];
  uint64_t full[kStages], empty[kStages];
  uint64_t s_ready, s_full, p_full, o_full, drained;  // s_ready: the scores before are read, BF16 keys in their operand
  long long sums[kThreads / 32];
  Plan plan;
  int start_row;
  long long start_offset, first, last;
  uint32_t tmem;
  int abort_flag, ignored_flag;
};

// The whole warp walks and waits; one thread of it issues.
template <int NT, int PT>
__device__ __forceinline__ void issue(Smem<NT>& sm, Walker walker, int lane) {
  using Sh = Shape<NT>;
  constexpr uint32_t kFp4 = tc::nvf4_idesc(128, NT), kF16 = f16_idesc(NT, 0, false);
  constexpr uint32_t kPages = f16_idesc(NT, 0, true), kBf16 = f16_idesc(NT, 1, true);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const uint32_t q = tc::smem_u32(sm.q), ring = tc::smem_u32(sm.ring);
  const uint64_t q_codes = tc::fp4_tile_desc(tc::smem_u32(sm.q_codes), 0);
  const uint64_t q_scales = tc::sf_atom_desc(tc::smem_u32(sm.q_scales));
  const uint64_t tile = tc::smem_desc(tc::smem_u32(sm.p), tc::kSwizzle128B, 1024, 16384);
  uint32_t k_parity = 0, p_parity = 0;
  Place<Smem<NT>::kStages> at;
  Unit u;
  bool known = false;
#pragma unroll 1
  for (; walker.next(u, known); known = true) {
    // a step's scores go before the output of the one before
#pragma unroll 1
    for (int step = u.begin; step <= u.end; ++step) {
      if (step < u.end) {
        const StepKind kind = step_kind(u.info, step);
        wait(&sm.s_ready, k_parity, &sm.abort_flag);
        k_parity ^= 1;
        if (kind == kStepPage) {
          wait(&sm.full[at.slot], at.turn, &sm.abort_flag);
          if constexpr (PT == 64) interleave_scales(sm.ring[at.slot] + kKsOffset, lane);
          tc::fence_after_sync();
          const uint32_t stage = ring + at.slot * kStage;
          const uint64_t codes = tc::fp4_tile_desc(stage, 0), atoms = tc::sf_atom_desc(stage + kKsOffset);
          if (elect_one()) {
            if (step == u.begin) {
#pragma unroll 1
              for (int i = 0; i < 2 * kTerms; ++i) tc::cp_sf_atom(tmem + Sh::kQs + i * 4, q_scales + i * 32);
            }
            tc::cp_sf_atom(tmem + Sh::kKs, atoms);
            tc::cp_sf_atom(tmem + Sh::kKs + 4, atoms + 32);
#pragma unroll
            for (int s = 0; s < 2; ++s) {  // 64 channels further: 32 bytes of codes, one atom of scales
#pragma unroll
              for (int term = 0; term < kTerms; ++term)
                tc::mma_nvf4(tmem + Sh::kS, codes + 2 * s, q_codes + term * NT * 4 + 2 * s, kFp4,
                             tmem + Sh::kKs + 4 * s, tmem + Sh::kQs + term * 8 + 4 * s, s + term > 0);
            }
            tc::commit(&sm.s_full);
            tc::commit(&sm.empty[at.slot]);
          }
          __syncwarp();
          at.advance();
        } else {
#pragma unroll 1
          for (int i = 2 * bf16_stages(u.info, kind); i > 0; --i) at.advance();
          tc::fence_after_sync();
          if (elect_one()) {
#pragma unroll 1
            for (int s = 0; s < 8; ++s)
              mma_ts(tmem + Sh::kS, tmem + Sh::kK + s * 8, tc::bf16_tile_desc(q + (s >> 2) * NT * 128, s & 3), kF16, s > 0);
            tc::commit(&sm.s_full);
          }
          __syncwarp();
        }
      }
      if (step == u.begin) continue;
      wait(&sm.p_full, p_parity, &sm.abort_flag);  // P, and before it V
      p_parity ^= 1;
      tc::fence_after_sync();
      const StepKind kind = step_kind(u.info, step - 1);
      const bool first = step - 1 == u.begin;
      if (elect_one()) {
        if (kind == kStepPage) {
#pragma unroll
          for (int s = 0; s < 8; ++s)  // 16 tokens further: 2048 bytes of P, 8 columns of V
            mma_ts(tmem + Sh::kO, tmem + Sh::kV + s * 8, tile + s * 128, kPages, !(first && s == 0));
        } else {
          const int slices = step_slices(u.info, kind);
#pragma unroll 1
          for (int s = 0; s < slices; ++s)
            mma_ts(tmem + Sh::kO, tmem + Sh::kV + s * 8, tile + s * 128, kBf16, !(first && s == 0));
        }
        tc::commit(&sm.o_full);
      }
      __syncwarp();
    }
  }
  // also after an abort: tensor memory is freed behind the last product
  if (elect_one()) tc::commit(&sm.drained);
  __syncwarp();
  wait(&sm.drained, 0, &sm.ignored_flag);
}

template <int NT, int PT>
__device__ __forceinline__ void work(const TreeParams& p, Smem<NT>& sm, Walker walker, int thread) {
  using Sh = Shape<NT>;
  constexpr int C = Sh::kColumns;
  const int t = thread & 127, lane = thread & 31, warp = t >> 5, half = thread >> 7;
  const int first_column = half * C;
  const int barrier = kHalfBarrier + half;
  const uint32_t lanes = sm.tmem + ((uint32_t)(t & ~31) << 16);
  const uint32_t scores = lanes + Sh::kS + first_column, k_operand = lanes + Sh::kK, v_operand = lanes + Sh::kV;
  float* base = sm.base + first_column;
  float* top = sm.top + first_column;
  // where this thread's codes and scales lie in a stage: half of channel t's tokens
  const int v_swizzle = (t >> 1) & 3;
  const int v_codes = kVOffset + (PT == 128 ? t * 64 : half * 4096 + t * 32);
  const int v_scales = kVsOffset + half * 512 + (t & 31) * 16 + (t >> 5) * 4;
  const int v_chunk0 = PT == 128 ? ((2 * half) ^ v_swizzle) * 16 : ((t >> 2) & 1) * 16;  // the other one's is 16 off
  uint8_t* const p_row = sm.p + t * 128;
  const int p_chunk = first_column >> 3, p_swizzle = t & 7;
  Place<Smem<NT>::kStages> v_at;
  uint32_t parity = 0;
  bool any = false;  // a step has been taken
  long long done = sm.first;
  Unit u;
  bool known = false;
#pragma unroll 1
  for (; walker.next(u, known); known = true) {
    bool uneven;
    const float q_inverse = load_queries<NT, kWorkers>(p, sm, kWorkBarrier, u, thread, uneven);
    if (t < C) {
      if (uneven) sm.level[first_column + t] = query_level(sm.own[first_column + t], q_inverse);
      top[t] = kNoMax;
      base[t] = 0.0f;  // scores as they are
    }
    if (warp == 0) make_masks(p, u, sm.parents, sm.seen_by[half], u.tile * NT + first_column, lane);
    float2 sum[C / 2];
#pragma unroll
    for (int j = 0; j < C / 2; ++j) sum[j] = make_float2(0.0f, 0.0f);
    bar_sync(barrier, 128);
    const float page_factor = p.scale_log2 * q_inverse * p.key_scale;
    // Lets the scores of a step be taken: those of the step before are in registers. `keys`: where a BF16 step's
    // keys are; they go into their operand first. Returns what turns the step's scores into log2 units.
    auto let_scores = [&](int step, Place<Smem<NT>::kStages> keys) -> float {
      const StepKind kind = step_kind(u.info, step);
      float f = page_factor;
      if (kind != kStepPage) {
        f = p.scale_log2 * q_inverse * bf16_keys(p, sm, kWorkBarrier, u, kind, keys, k_operand, thread);
        tc::tmem_wait_st();
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.s_ready);
      return f;
    };
    float f = let_scores(u.begin, v_at);
#pragma unroll 1
    for (int step = u.begin; step < u.end; ++step) {
      const StepKind kind = step_kind(u.info, step);
      const bool special = kind != kStepPage || (step == 0 && u.info.sink > 0);  // the same in the whole half
      wait(&sm.s_full, parity, &sm.abort_flag);
      tc::fence_after_sync();

      if (uneven) scale_columns<C>(scores, sm.level + first_column);
      float s[C];
      tmem_load<C>(scores, s);
      tc::tmem_wait_ld();
      // scores -> log2 units above the maxima, plus kShift
      const float2 f2 = make_float2(f, f);
#pragma unroll
      for (int j = 0; j < C; j += 4) {
        const float4 b = *reinterpret_cast<const float4*>(base + j);
        const float2 y0 = __ffma2_rn(make_float2(s[j], s[j + 1]), f2, make_float2(b.x, b.y));
        const float2 y1 = __ffma2_rn(make_float2(s[j + 2], s[j + 3]), f2, make_float2(b.z, b.w));
        s[j] = y0.x, s[j + 1] = y0.y, s[j + 2] = y1.x, s[j + 3] = y1.y;
      }
      if (special) {  // (masked behind the scaling: a factor may underflow to zero, and its product with -inf is NaN)
        bool dead;  // no query sees this thread's token
        if (kind == kStepPage) dead = t < u.info.sink;
        else if (kind == kStepTail) dead = t >= u.info.residual || (u.info.pages == 0 && t < u.info.sink);
        else dead = t < BDFP4_MAX_SINK ? t >= u.info.sink : t - BDFP4_MAX_SINK >= u.info.count;
        uint32_t seen = dead ? 0u : ~0u;
        if (kind == kStepDraft && t >= BDFP4_MAX_SINK && !dead) seen = sm.seen_by[half][t - BDFP4_MAX_SINK];
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (!((seen >> j) & 1)) s[j] = -INFINITY;
      }
      float highest = -INFINITY;
#pragma unroll
      for (int j = 0; j < C; j += 4) highest = fmaxf(fmaxf(highest, fmaxf(s[j], s[j + 1])), fmaxf(s[j + 2], s[j + 3]));
      // the next step's scores are taken while this one's probabilities are formed
      float next_f = f;
      if (step + 1 < u.end) {
        Place<Smem<NT>::kStages> keys = v_at;
#pragma unroll 1
        for (int i = kind == kStepPage ? 1 : 2 * bf16_stages(u.info, kind); i > 0; --i) keys.advance();
        next_f = let_scores(step + 1, keys);
      }
      // V, once the product of the step before is done with its operand, P and (for a rescaling) the output
      if (any) wait(&sm.o_full, parity ^ 1, &sm.abort_flag);
      tc::fence_after_sync();
      if (kind == kStepPage) {
        wait(&sm.full[v_at.slot], v_at.turn, &sm.abort_flag);
        const uint8_t* stage = sm.ring[v_at.slot];
        const uint32_t scale = *reinterpret_cast<const uint32_t*>(stage + v_scales);
        const uint4 chunk0 = *reinterpret_cast<const uint4*>(stage + v_codes + v_chunk0);
        const uint4 chunk1 = *reinterpret_cast<const uint4*>(stage + v_codes + (v_chunk0 ^ 16));
        store_dequantized(v_operand + 32 * half, chunk0, scale);
        store_dequantized(v_operand + 32 * half + 16, chunk1, scale >> 16);
        release(sm, v_at, thread, false);
      } else {
        bf16_values(sm, u, kind, v_at, v_operand, thread);
      }
      // Maxima are taken in a unit's first step, in one that could be the first with anything to see (a tail may
      // hold nothing but sink), and when a score exceeds its query's by too much.
      const bool forced = step == u.begin || (kind == kStepDraft && u.info.pages == 0);
      if (bar_any(barrier, forced || highest > kShift + kGrowth)) {
        float mine = 0.0f;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const float m = warp_max(s[j]);
          if (lane == j) mine = m;
        }
        if (lane < C) sm.col[warp][first_column + lane] = mine;
        bar_sync(barrier, 128);
        if (t < C) {
          // The new maximum is taken from the scores as they stand, above the old one, and all move by the same
          // difference: between a score and a maximum that were rounded apart, differences beyond FP16's range open
          // up as soon as scores exceed 2^27.
          const int col = first_column + t;
          const float m = fmaxf(fmaxf(sm.col[0][col], sm.col[1][col]), fmaxf(sm.col[2][col], sm.col[3][col]));
          const bool none = top[t] == kNoMax;
          float move = 0.0f, factor = 1.0f;
          if (none ? m > -INFINITY : m > kShift) {
            move = kShift - m;
            factor = none ? 0.0f : ex2(move);
            base[t] += move;
            top[t] = kShift - base[t];
          }
          sm.shift[col] = move;
          sm.factor[col] = factor;
        }
        bar_sync(barrier, 128);
#pragma unroll
        for (int j = 0; j < C / 2; ++j) {
          s[2 * j] += sm.shift[first_column + 2 * j];
          s[2 * j + 1] += sm.shift[first_column + 2 * j + 1];
          sum[j].x *= sm.factor[first_column + 2 * j];
          sum[j].y *= sm.factor[first_column + 2 * j + 1];
        }
        if (step > u.begin) {  // what O^T holds is of the old maxima
#pragma unroll 1
          for (int j = 0; j < C; j += 8) {
            float o[8];
            const uint32_t column = lanes + Sh::kO + first_column + j;
            tc::tmem_ld8(column, o);
            tc::tmem_wait_ld();
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(o[i] * sm.factor[first_column + j + i]);
            st8(column, w);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < C; j += 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[j + i] = ex2(s[j + i]);
        if (kind == kStepPage) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = h2(__floats2half2_rn(s[j + 2 * i], s[j + 2 * i + 1]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = pack_bf16x2(s[j + 2 * i] * p.inverse_value_scale, s[j + 2 * i + 1] * p.inverse_value_scale);
        }
        *reinterpret_cast<uint4*>(p_row + (((p_chunk + (j >> 3)) ^ p_swizzle) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.p_full);
#pragma unroll
      for (int j = 0; j < C / 2; ++j) sum[j] = __fadd2_rn(sum[j], make_float2(s[2 * j], s[2 * j + 1]));
      f = next_f;
      parity ^= 1;
      any = true;
    }

    {  // each query's weight: first over a warp's 32 tokens, then (below) over the four warps
      float v[C];
#pragma unroll
      for (int j = 0; j < C / 2; ++j) v[2 * j] = sum[j].x, v[2 * j + 1] = sum[j].y;
      reduce_columns<C, 16>(v, lane, 0, [&](int j, float total) { sm.col[warp][first_column + j] = total; });
    }
    bar_sync(barrier, 128);
    const bool whole = u.begin == 0 && u.end == u.info.steps;
    const long long at_step = done - u.begin;  // where the unit begins in the launch's steps
    done += u.end - u.begin;
    // a part that begins a unit goes to the CTA's second slot, one that continues it to the first
    const int part = 2 * blockIdx.x + (u.begin == 0 ? 1 : 0);
    if (t < C) {
      const int col = first_column + t;
      const float total = (sm.col[0][col] + sm.col[1][col]) + (sm.col[2][col] + sm.col[3][col]);
      if (whole) {
        sm.factor[col] = total > 0.0f ? p.value_scale / total : 0.0f;
      } else {
        p.partial_stat[(int64_t)(2 * part) * NT + col] = top[t];
        p.partial_stat[(int64_t)(2 * part + 1) * NT + col] = total;
      }
    }
    bar_sync(barrier, 128);
    wait(&sm.o_full, parity ^ 1, &sm.abort_flag);
    tc::fence_after_sync();
    store_output(p, sm, u, lanes + Sh::kO + first_column, NT, first_column, C, whole, part, t);
    tc::fence_before_sync();
    if (!whole && u.begin == 0 && thread == 0) {
      TreeSplit split;
      split.row = u.row;
      split.head = u.head;
      split.tile = u.tile;
      split.last = sm.plan.owner_of_last(at_step, at_step + u.info.steps);
      p.splits[blockIdx.x] = split;
    }
  }
}

template <int NT, int PT>
__global__ void __launch_bounds__(kThreads, 2)
tree_narrow_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const TreeParams p) {
  extern __shared__ uint8_t raw_smem[];
  // (an offset, not a masked pointer: the compiler has to see that this is shared memory)
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(raw_smem + (-tc::smem_u32(raw_smem) & 1023u));
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  dependents_may_launch();

  if (thread == 0) {
#pragma unroll 1
    for (int i = 0; i < Smem<NT>::kStages; ++i) {
      tc::mbar_init(&sm.full[i], 1);
      tc::mbar_init(&sm.empty[i], 9);  // the workers' warps and the score product
    }
    tc::mbar_init(&sm.s_ready, 8);
    tc::mbar_init(&sm.s_full, 1);
    tc::mbar_init(&sm.p_full, 8);
    tc::mbar_init(&sm.o_full, 1);
    tc::mbar_init(&sm.drained, 1);
    tc::fence_barrier_init();
    sm.abort_flag = sm.ignored_flag = 0;
    TreeSplit none;
    none.row = -1;
    none.head = none.tile = none.last = 0;
    p.splits[blockIdx.x] = none;
  }
  make_plan<PT, kThreads, kSnap>(p, sm, thread);
  if (warp == 0) {
    tc::tmem_alloc(&sm.tmem, kTmemColumns);
    tc::tmem_relinquish();
    tc::fence_before_sync();
  }
  __syncthreads();
  tc::fence_after_sync();
  if (sm.first < sm.last) {
    const Walker walker(p, sm.start_row, (int)sm.start_offset, (int)(sm.last - sm.first), PT);
    if (warp < kWorkers / 32) work<NT, PT>(p, sm, walker, thread);
    else if (warp == kWorkers / 32) produce<PT>(p, sm, walker, &k_map, &v_map, lane);
    else issue<NT, PT>(sm, walker, lane);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (thread == 0 && sm.abort_flag && p.error_word) atomicOr(p.error_word, (int)BDFP4_DEV_WAIT_TIMEOUT);
  if (warp == 0) tc::tmem_dealloc(sm.tmem, kTmemColumns);
}

template <int NT, int PT>
static cudaError_t launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream) {
  const int smem = (int)sizeof(Smem<NT>) + 1024;
  static PerDeviceOnce configured;
  const int slot = current_device_slot();
  if (slot < 0 || !configured.done[slot]) {
    cudaError_t e = cudaFuncSetAttribute(tree_narrow_kernel<NT, PT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (slot >= 0) configured.done[slot] = true;
  }
  tree_narrow_kernel<NT, PT><<<kTreeNarrowCtas, kThreads, smem, stream>>>(k_map, v_map, p);
  return cudaGetLastError();
}

}  // namespace narrow
}  // namespace tree
}  // namespace bdfp4
