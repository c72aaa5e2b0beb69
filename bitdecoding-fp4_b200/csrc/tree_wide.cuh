// The tree attention for tiles of 64 to 128 queries: warps of one role each, one CTA per SM. A step's values are
// converted once for up to 128 queries, so what bounds it is the softmax: 128 x NT exponentials (8 cycles a step and
// query on an SM) and their surroundings, up to four groups of 128 threads with at most 32 queries per thread. One
// row of 262145 tokens under 256 query rows per KV head takes 418 to 425 us, 650 TFLOP/s of FP16 products or 0.41 of a
// library product's rate: tensor cores 31% busy, issue slots 57%. (Before scores of any magnitude were served, 403 to
// 420 on the same boxes, and 367 on another: 2750 cycles a step of 128 queries.) With 64 queries (16 rows x 16 nodes, up
// to 8192) 87 us; by two CTAs per SM (tree_narrow.cuh's form) 120.
#pragma once

#include "tree_common.cuh"

namespace bdfp4 {
namespace tree {
namespace wide {

// Named barriers: one per softmax group (four at most), all softmax threads, the key threads.
constexpr int kCtas = kTreeWideCtas;
// How near a unit's end a cut moves there, in steps (3, 6, 10, 16 measured: 16 rows x 16 nodes x 2048 51, 49, 41, 41 us,
// 24 rows x 61 nodes x 2048 218, 214, 201, 201, a ragged batch of 16 rows up to 8192 80, 82, 84, 89).
constexpr int kSnap = 10;
constexpr int kGroupBarrier = 1, kSoftmaxBarrier = 5, kCacheBarrier = 6;

// A softmax thread holds at most 32 queries: their sums stay in registers for a whole unit, and with 64 (256 threads
// for NT = 128) the kernel spilled, into an L1 that shared memory has left little of. Sixteen, as many threads as a
// tile of 64 leaves, let it keep the scores too (82 us for 16 rows x 16 nodes x 8192 against 87 with 32). With 32,
// half of them are read twice, for the vote and after it (all of them: 385 us for one row x 262145 against 367; forming
// the probabilities first and keeping them, packed, until the vote is over: 413).
template <int NT>
struct Shape {
  static constexpr int kColumns = NT < 96 ? 16 : 32;        // queries per softmax thread
  static constexpr int kGroups = NT / kColumns;             // softmax groups of 128 threads
  static constexpr int kBlocks = (NT + 63) / 64;            // 128-byte rows of P per token
  static constexpr int kVBuffers = NT > 96 ? 1 : 2;         // operand buffers in tensor memory, as many as it holds
  static constexpr int kStages = NT > 96 ? 4 : NT > 64 ? 5 : 7;
  static constexpr int kSoftmaxThreads = 128 * kGroups;
  static constexpr int kThreads = kCacheThreads + kSoftmaxThreads + 128;  // cache side, softmax, control (two of its warps idle)
  // Registers per thread at launch and after the warpgroups have traded them: the sum over the warpgroups
  // must not exceed what the launch was given.
  static constexpr int kLaunchRegs = kGroups == 4 ? 72 : kGroups == 3 ? 80 : kGroups == 2 ? 96 : 128;
  static constexpr int kSoftmaxRegs = kGroups == 4 ? 80 : kGroups == 3 ? 96 : kGroups == 2 ? 112 : 144;
  static constexpr int kCacheRegs = kGroups == 4 ? 72 : kGroups == 3 ? 72 : kGroups == 2 ? 96 : 128;
  static constexpr int kControlRegs = kGroups == 4 ? 40 : kGroups == 3 ? 40 : kGroups == 2 ? 56 : 88;
  static_assert(kSoftmaxRegs * kGroups + 2 * kCacheRegs + kControlRegs <= kLaunchRegs * (3 + kGroups), "registers");
  static_assert(kLaunchRegs * kThreads <= 65536, "registers");
  static constexpr bool kHold = kColumns <= 16;  // a thread's scores stay in registers between the vote and the exponentials
  // tensor memory columns
  // (the keys of a BF16 step lie where the pages' products had their scales: pages come first in a unit)
  static constexpr int kS = 0, kO = 2 * NT, kV = 3 * NT, kK = kV + 64 * kVBuffers, kKs = kK, kQs = kKs + 16;
  static_assert(kK + 64 <= 512 && kQs + 8 * kTerms <= kK + 64, "tensor memory");
};

template <int FROM, int TO>
__device__ __forceinline__ void trade_registers() {
  if constexpr (TO > FROM) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TO));
  if constexpr (TO < FROM) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TO));
}

template <int NT>
struct Smem {
  using Sh = Shape<NT>;
  static constexpr int kStages = Sh::kStages;
  alignas(1024) uint8_t ring[kStages][kStage];
  alignas(1024) uint8_t q[2][NT * 128];            // FP16 queries: two halves of 64 channels, K-major, 128-byte swizzle
  alignas(1024) uint8_t q_codes[kTerms][NT * 64];  // FP4 terms, K-major, 64-byte swizzle
  alignas(1024) uint8_t q_scales[kTerms][1024];    // two atoms each
  alignas(1024) uint8_t p[2][Sh::kBlocks * 16384];  // MN-major: 128-byte rows of 64 queries per token, swizzled
  uint32_t seen_by[Sh::kGroups][BDFP4_MAX_TREE_NODES];  // which of a group's columns see a draft node
  float base[NT];       // kShift - maximum
  float top[NT];        // maximum, log2 units
  float factor[NT];     // what a renewal does to sums (at a unit's end: 1 / weight)
  float level[NT];      // power of two that a column's scores are multiplied by as they come, where a group has any
  float squeeze[NT];    // undoes what renewals made of it
  float lower[NT];      // what the last renewal did
  bool lowered[Sh::kGroups];
  float col[4][NT];     // a warp's maxima, then sums
  float key_factor[8][128];  // what undoes the scaling of a BF16 step's keys, by step number
  float own[NT];
  float2 q_range[16];
  int parents[BDFP4_MAX_TREE_NODES];
  uint64_t full[kStages], empty[kStages];
  uint64_t ka_full, ka_empty, va_full[2], va_empty[2];  // operands: BF16 keys, values
  uint64_t s_full[2], s_empty[2], p_full[2], p_empty[2];
  uint64_t q_full, o_full, o_empty, drained;
  long long sums[Sh::kThreads / 32];
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
  const uint32_t q = tc::smem_u32(sm.q), prob = tc::smem_u32(sm.p), ring = tc::smem_u32(sm.ring);
  const uint64_t q_codes = tc::fp4_tile_desc(tc::smem_u32(sm.q_codes), 0);
  const uint64_t q_scales = tc::sf_atom_desc(tc::smem_u32(sm.q_scales));
  int n = 0, unit = 0;
  uint32_t ka_turn = 0;
  Place<Sh::kStages> at;
  Unit u;
  bool known = false;
#pragma unroll 1
  for (; walker.next(u, known); known = true) {
    auto output = [&](int step, int j) {  // O^T += V^T P^T of step `step` of the unit, the CTA's j-th
      const StepKind kind = step_kind(u.info, step);
      const int a = j % Sh::kVBuffers;
      wait(&sm.va_full[a], (j / Sh::kVBuffers) & 1, &sm.abort_flag);
      wait(&sm.p_full[j & 1], (j >> 1) & 1, &sm.abort_flag);
      const bool first = step == u.begin;
      if (first) wait(&sm.o_empty, (unit & 1) ^ 1, &sm.abort_flag);
      tc::fence_after_sync();
      const uint64_t tile = tc::smem_desc(prob + (j & 1) * Sh::kBlocks * 16384, tc::kSwizzle128B, 1024, 16384);
      const uint32_t operand = tmem + Sh::kV + a * 64;
      if (elect_one()) {
        if (kind == kStepPage) {
#pragma unroll
          for (int s = 0; s < 8; ++s)  // 16 tokens further: 2048 bytes of P, 8 columns of V
            mma_ts(tmem + Sh::kO, operand + s * 8, tile + s * 128, kPages, !(first && s == 0));
        } else {
          const int slices = step_slices(u.info, kind);
          for (int s = 0; s < slices; ++s)
            mma_ts(tmem + Sh::kO, operand + s * 8, tile + s * 128, kBf16, !(first && s == 0));
        }
        tc::commit(&sm.va_empty[a]);
        tc::commit(&sm.p_empty[j & 1]);
      }
      __syncwarp();
    };
    wait(&sm.q_full, unit & 1, &sm.abort_flag);
#pragma unroll 1
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      const uint32_t scores = tmem + Sh::kS + (n & 1) * NT;
      wait(&sm.s_empty[n & 1], ((n >> 1) & 1) ^ 1, &sm.abort_flag);
      if (kind == kStepPage) {
        wait(&sm.full[at.slot], at.turn, &sm.abort_flag);
        if constexpr (PT == 64) interleave_scales(sm.ring[at.slot] + kKsOffset, lane);
        tc::fence_after_sync();
        const uint32_t stage = ring + at.slot * kStage;
        const uint64_t codes = tc::fp4_tile_desc(stage, 0), atoms = tc::sf_atom_desc(stage + kKsOffset);
        const uint32_t scales = tmem + Sh::kKs + (n & 1) * 8;
        if (elect_one()) {
          if (step == u.begin) {
#pragma unroll 1
            for (int i = 0; i < 2 * kTerms; ++i) tc::cp_sf_atom(tmem + Sh::kQs + i * 4, q_scales + i * 32);
          }
          tc::cp_sf_atom(scales, atoms);
          tc::cp_sf_atom(scales + 4, atoms + 32);
#pragma unroll
          for (int s = 0; s < 2; ++s) {  // 64 channels further: 32 bytes of codes, one atom of scales
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
              tc::mma_nvf4(scores, codes + 2 * s, q_codes + term * NT * 4 + 2 * s, kFp4, scales + 4 * s,
                           tmem + Sh::kQs + term * 8 + 4 * s, s + term > 0);
          }
          tc::commit(&sm.s_full[n & 1]);
          tc::commit(&sm.empty[at.slot]);
        }
        __syncwarp();
        at.advance();
      } else {
#pragma unroll 1
        for (int i = 2 * bf16_stages(u.info, kind); i > 0; --i) at.advance();
        if (elect_one()) tc::commit(&sm.ka_empty);  // behind every product that reads scales or keys there
        __syncwarp();
        wait(&sm.ka_full, ka_turn, &sm.abort_flag);
        ka_turn ^= 1;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll 1
          for (int s = 0; s < 8; ++s)
            mma_ts(scores, tmem + Sh::kK + s * 8, tc::bf16_tile_desc(q + (s >> 2) * NT * 128, s & 3), kF16, s > 0);
          tc::commit(&sm.s_full[n & 1]);
        }
        __syncwarp();
      }
      if (step > u.begin) output(step - 1, n - 1);
    }
    output(u.end - 1, n - 1);
    if (elect_one()) tc::commit(&sm.o_full);
    __syncwarp();
    ++unit;
  }
  // also after an abort: tensor memory is freed behind the last product
  if (elect_one()) tc::commit(&sm.drained);
  __syncwarp();
  wait(&sm.drained, 0, &sm.ignored_flag);
}

// The cache side: half h of the threads converts tokens 64 h to 64 h + 63 of channel c of every step.
template <int NT, int PT>
__device__ __forceinline__ void cache(const TreeParams& p, Smem<NT>& sm, Walker walker, int thread) {
  using Sh = Shape<NT>;
  const int c = thread & 127, half = thread >> 7, lane = thread & 31;
  const uint32_t lanes = sm.tmem + ((uint32_t)(c & ~31) << 16);
  const int codes = kVOffset + (PT == 128 ? c * 64 : half * 4096 + c * 32);
  const int chunk = PT == 128 ? ((2 * half) ^ ((c >> 1) & 3)) * 16 : ((c >> 2) & 1) * 16;  // the other one's is 16 off
  const int scales = kVsOffset + half * 512 + (c & 31) * 16 + (c >> 5) * 4;
  Place<Sh::kStages> at;
  int n = 0;
  uint32_t ka_turn = 0;
  Unit u;
  bool known = false;
#pragma unroll 1
  for (; walker.next(u, known); known = true) {
#pragma unroll 1
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      const int buffer = n % Sh::kVBuffers;
      const uint32_t operand = lanes + Sh::kV + buffer * 64;
      const uint32_t empty_parity = ((n / Sh::kVBuffers) & 1) ^ 1;
      if (kind == kStepPage) {
        wait(&sm.full[at.slot], at.turn, &sm.abort_flag);
        const uint8_t* stage = sm.ring[at.slot];
        const uint32_t scale = *reinterpret_cast<const uint32_t*>(stage + scales);
        const uint4 chunk0 = *reinterpret_cast<const uint4*>(stage + codes + chunk);
        const uint4 chunk1 = *reinterpret_cast<const uint4*>(stage + codes + (chunk ^ 16));
        release(sm, at, thread, false);
        wait(&sm.va_empty[buffer], empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
        store_dequantized(operand + 32 * half, chunk0, scale);
        store_dequantized(operand + 32 * half + 16, chunk1, scale >> 16);
      } else {
        wait(&sm.ka_empty, ka_turn, &sm.abort_flag);
        ka_turn ^= 1;
        tc::fence_after_sync();
        const float inverse = bf16_keys(p, sm, kCacheBarrier, u, kind, at, lanes + Sh::kK, thread);
        if (half == 0) sm.key_factor[n & 7][c] = inverse;
        tc::tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.ka_full);
        wait(&sm.va_empty[buffer], empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
        bf16_values(sm, u, kind, at, operand, thread);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.va_full[buffer]);
    }
  }
}

template <int NT>
__device__ __forceinline__ float bring_queries(const TreeParams& p, Smem<NT>& sm, const Unit& u, int thread, bool& uneven) {
  const float inverse = load_queries<NT, Shape<NT>::kSoftmaxThreads>(p, sm, kSoftmaxBarrier, u, thread, uneven);
  __syncwarp();
  if ((thread & 31) == 0) tc::mbar_arrive(&sm.q_full);
  return inverse;
}

template <int NT>
__device__ __forceinline__ void softmax(const TreeParams& p, Smem<NT>& sm, Walker walker, int thread) {
  using Sh = Shape<NT>;
  constexpr int C = Sh::kColumns;
  const int t = thread & 127, lane = thread & 31, warp = t >> 5, group = thread >> 7;
  const int first_column = group * C;
  const int barrier = kGroupBarrier + group;
  const uint32_t lanes = (uint32_t)(t & ~31) << 16;
  float* base = sm.base + first_column;
  float* top = sm.top + first_column;
  int n = 0, unit = 0;
  long long done = sm.first;
  Unit u;
  if (!walker.next(u, false)) return;
  bool more = true;
  bool leveled;  // the group's scores are brought down as they come
  float q_inverse = bring_queries<NT>(p, sm, u, thread, leveled);
  while (more) {
    for (int j = t; j < C; j += 128) {
      top[j] = kNoMax;
      base[j] = kShift - kNoMax;
      sm.level[first_column + j] = leveled ? query_level(sm.own[first_column + j], q_inverse) : 1.0f;
      sm.squeeze[first_column + j] = 1.0f;
    }
    if (warp == 0) make_masks(p, u, sm.parents, sm.seen_by[group], u.tile * NT + first_column, lane);
    float2 sum[C / 2];
#pragma unroll
    for (int j = 0; j < C / 2; ++j) sum[j] = make_float2(0.0f, 0.0f);
    bar_sync(barrier, 128);
    const float page_factor = p.scale_log2 * q_inverse * p.key_scale;
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      bool dead;  // no query sees this thread's token
      if (kind == kStepPage) dead = step == 0 && t < u.info.sink;
      else if (kind == kStepTail) dead = t >= u.info.residual || (u.info.pages == 0 && t < u.info.sink);
      else dead = t < BDFP4_MAX_SINK ? t >= u.info.sink : t - BDFP4_MAX_SINK >= u.info.count;
      const bool masked = kind == kStepDraft && t >= BDFP4_MAX_SINK && !dead;
      const uint32_t seen = masked ? sm.seen_by[group][t - BDFP4_MAX_SINK] : ~0u;
      wait(&sm.s_full[n & 1], (n >> 1) & 1, &sm.abort_flag);
      tc::fence_after_sync();
      float f = page_factor;
      if (kind != kStepPage) f = p.scale_log2 * q_inverse * sm.key_factor[n & 7][t];
      f = fmaxf(f, 1.0e-38f);  // (where it underflows to zero, its product with a mask's -inf would be NaN)
      const float2 f2 = make_float2(f, f);
      const uint32_t scores = sm.tmem + Sh::kS + (n & 1) * NT + first_column + lanes;
      if (leveled) scale_columns<C>(scores, sm.level + first_column);
      auto load16 = [&](int j, float* s) {
        tc::tmem_ld16(scores + j, s);
        tc::tmem_wait_ld();
        if (kind == kStepDraft) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((seen >> (j + i)) & 1)) s[i] = -INFINITY;
        }
      };
      // scores -> log2 units above the maxima, plus kShift
      auto above16 = [&](int j, float* s) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 b = *reinterpret_cast<const float4*>(base + j + i);
          const float2 y0 = __ffma2_rn(make_float2(s[i], s[i + 1]), f2, make_float2(b.x, b.y));
          const float2 y1 = __ffma2_rn(make_float2(s[i + 2], s[i + 3]), f2, make_float2(b.z, b.w));
          s[i] = y0.x, s[i + 1] = y0.y, s[i + 2] = y1.x, s[i + 3] = y1.y;
        }
      };
      float held[Sh::kHold ? C : 16];
      float highest = -INFINITY;
#pragma unroll
      for (int j = 0; j < C; j += 16) {
        float* s = Sh::kHold ? held + j : held;
        load16(j, s);
        above16(j, s);
#pragma unroll
        for (int i = 0; i < 16; ++i) highest = fmaxf(highest, s[i]);
      }
      if (bar_any(barrier, highest > kGrowth + kShift && !dead)) {
#pragma unroll
        for (int j = 0; j < C; j += 16) {
          float s[16];
          load16(j, s);
          float mine = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float m = warp_max(dead ? -INFINITY : s[i] * f);
            if (lane == i) mine = m;
          }
          if (lane < 16) sm.col[warp][first_column + j + lane] = mine;
        }
        if (t == 0) sm.lowered[group] = false;
        bar_sync(barrier, 128);
        for (int j = t; j < C; j += 128) {
          const int col = first_column + j;
          const float before = top[j];
          float now = fmaxf(fmaxf(fmaxf(sm.col[0][col], sm.col[1][col]),
                                  fmaxf(sm.col[2][col], sm.col[3][col])), before);
          sm.factor[col] = ex2((before - now) * sm.squeeze[col]);
          // A score's product is not rounded before the maximum, which was, is taken off: above 2^27 the two stand
          // further apart than FP16's exponents reach. Such a query's scores are brought down to 2^22 by a power of two:
          // what then differs by less than 64 (log2) did so by less than 2^-16 of the scores, which is what the
          // rounding of their products and sums may come to.
          float lower = 1.0f;
          if (fabsf(now) >= 8388608.0f && now > kNoMax) {
            float back;
            lower = scale_to<22>(fabsf(now), &back);
            now *= lower;
            sm.level[col] *= lower;
            sm.squeeze[col] *= back;
            sm.lowered[group] = true;
          }
          sm.lower[col] = lower;
          top[j] = now;
          base[j] = kShift - now;
        }
        bar_sync(barrier, 128);
        if (sm.lowered[group]) {
          leveled = true;
          scale_columns<C>(scores, sm.lower + first_column);
        }
#pragma unroll
        for (int j = 0; j < C / 2; ++j) {
          sum[j].x *= sm.factor[first_column + 2 * j];
          sum[j].y *= sm.factor[first_column + 2 * j + 1];
        }
        if (step > u.begin) {  // what O^T holds is of the old maxima
          wait(&sm.p_empty[(n - 1) & 1], ((n - 1) >> 1) & 1, &sm.abort_flag);
          tc::fence_after_sync();
#pragma unroll 1
          for (int j = 0; j < C; j += 16) {
            float o[16];
            const uint32_t at = sm.tmem + Sh::kO + first_column + j + lanes;
            tc::tmem_ld16(at, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= sm.factor[first_column + j + i];
            tc::tmem_st16(at, o);
          }
          tc::tmem_wait_st();
        }
#pragma unroll
        for (int j = Sh::kHold ? 0 : C - 16; j < C; j += 16) {
          load16(j, held + (Sh::kHold ? j : 0));
          above16(j, held + (Sh::kHold ? j : 0));
        }
      }
      if constexpr (Sh::kHold) {  // the scores are in registers: the next but one may come
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.s_empty[n & 1]);
      }
      // P of this step goes where the one before the last was
      wait(&sm.p_empty[n & 1], ((n >> 1) & 1) ^ 1, &sm.abort_flag);
#pragma unroll
      for (int j = C - 16; j >= 0; j -= 16) {  // (the last sixteen are there in any case)
        float* s = Sh::kHold ? held + j : held;
        if (!Sh::kHold && j < C - 16) {
          load16(j, s);
          above16(j, s);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = ex2(s[i]);
        if (dead) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = 0.0f;
        }
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[j / 2 + i] = __fadd2_rn(sum[j / 2 + i], make_float2(s[2 * i], s[2 * i + 1]));
        if (kind == kStepPage) {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = h2(__floats2half2_rn(s[2 * i], s[2 * i + 1]));
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = pack_bf16x2(s[2 * i] * p.inverse_value_scale, s[2 * i + 1] * p.inverse_value_scale);
        }
        const int column = first_column + j;
        uint8_t* row = sm.p[n & 1] + (column >> 6) * 16384 + t * 128;
        const int chunk = (column & 63) >> 3;
        *reinterpret_cast<uint4*>(row + ((chunk ^ (t & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ (t & 7)) * 16)) = make_uint4(w[4], w[5], w[6], w[7]);
      }
      tc::fence_before_sync();
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if constexpr (!Sh::kHold) tc::mbar_arrive(&sm.s_empty[n & 1]);
        tc::mbar_arrive(&sm.p_full[n & 1]);
      }
    }

    {  // each query's weight: first over a warp's 32 tokens, then (below) over the four warps
      float v[C];
#pragma unroll
      for (int j = 0; j < C / 2; ++j) v[2 * j] = sum[j].x, v[2 * j + 1] = sum[j].y;
      reduce_columns<C, 16>(v, lane, 0, [&](int j, float total) { sm.col[warp][first_column + j] = total; });
    }
    // the next unit's queries go in while this one's last product runs: all its scores are done
    Unit following = u;
    more = walker.next(following, true);
    float next_inverse = 1.0f;
    bool next_leveled = false;
    bar_sync(kSoftmaxBarrier, Sh::kSoftmaxThreads);  // both groups have seen their last scores; the parents are free
    if (more) next_inverse = bring_queries<NT>(p, sm, following, thread, next_leveled);
    bar_sync(barrier, 128);
    const bool whole = u.begin == 0 && u.end == u.info.steps;
    const long long at_step = done - u.begin;  // where the unit begins in the launch's steps
    done += u.end - u.begin;
    // a part that begins a unit goes to the CTA's second slot, one that continues it to the first
    const int part = 2 * blockIdx.x + (u.begin == 0 ? 1 : 0);
    for (int j = t; j < C; j += 128) {
      const int col = first_column + j;
      const float total = (sm.col[0][col] + sm.col[1][col]) + (sm.col[2][col] + sm.col[3][col]);
      if (whole) {
        sm.factor[col] = total > 0.0f ? p.value_scale / total : 0.0f;
      } else {
        p.partial_stat[(int64_t)(2 * part) * NT + col] = top[j] * sm.squeeze[col];
        p.partial_stat[(int64_t)(2 * part + 1) * NT + col] = total;
      }
    }
    bar_sync(barrier, 128);
    wait(&sm.o_full, unit & 1, &sm.abort_flag);
    tc::fence_after_sync();
    store_output(p, sm, u, sm.tmem + Sh::kO + first_column + lanes, NT, first_column, C, whole, part, t);
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.o_empty);
    bar_sync(barrier, 128);  // base, top and total are written anew
    if (!whole && u.begin == 0 && thread == 0) {
      TreeSplit split;
      split.row = u.row;
      split.head = u.head;
      split.tile = u.tile;
      split.last = sm.plan.owner_of_last(at_step, at_step + u.info.steps);
      p.splits[blockIdx.x] = split;
    }
    q_inverse = next_inverse;
    leveled = next_leveled;
    u = following;
    ++unit;
  }
}

template <int NT, int PT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
tree_wide_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const TreeParams p) {
  using Sh = Shape<NT>;
  extern __shared__ uint8_t raw_smem[];
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(raw_smem + (-tc::smem_u32(raw_smem) & 1023u));
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  dependents_may_launch();

  if (thread == 0) {
#pragma unroll 1
    for (int i = 0; i < Sh::kStages; ++i) {
      tc::mbar_init(&sm.full[i], 1);
      tc::mbar_init(&sm.empty[i], 9);  // the cache side's warps and the score product
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sm.va_full[i], 8);
      tc::mbar_init(&sm.va_empty[i], 1);
      tc::mbar_init(&sm.s_full[i], 1);
      tc::mbar_init(&sm.s_empty[i], 4 * Sh::kGroups);
      tc::mbar_init(&sm.p_full[i], 4 * Sh::kGroups);
      tc::mbar_init(&sm.p_empty[i], 1);
    }
    tc::mbar_init(&sm.ka_full, 8);
    tc::mbar_init(&sm.ka_empty, 1);
    tc::mbar_init(&sm.q_full, 4 * Sh::kGroups);
    tc::mbar_init(&sm.o_full, 1);
    tc::mbar_init(&sm.o_empty, 4 * Sh::kGroups);
    tc::mbar_init(&sm.drained, 1);
    tc::fence_barrier_init();
    sm.abort_flag = sm.ignored_flag = 0;
    TreeSplit none;
    none.row = -1;
    none.head = none.tile = none.last = 0;
    p.splits[blockIdx.x] = none;
  }
  make_plan<PT, Sh::kThreads, kSnap>(p, sm, thread);
  if (warp == 0) {
    tc::tmem_alloc(&sm.tmem, 512);
    tc::tmem_relinquish();
    tc::fence_before_sync();
  }
  __syncthreads();
  tc::fence_after_sync();
  if (sm.first < sm.last) {
    const Walker walker(p, sm.start_row, (int)sm.start_offset, (int)(sm.last - sm.first), PT);
    if (warp < 8) {
      trade_registers<Sh::kLaunchRegs, Sh::kCacheRegs>();
      cache<NT, PT>(p, sm, walker, thread);
    } else if (warp < 8 + 4 * Sh::kGroups) {
      trade_registers<Sh::kLaunchRegs, Sh::kSoftmaxRegs>();
      softmax<NT>(p, sm, walker, thread - 256);
    } else {
      trade_registers<Sh::kLaunchRegs, Sh::kControlRegs>();
      if (warp == 8 + 4 * Sh::kGroups) produce<PT>(p, sm, walker, &k_map, &v_map, lane);
      if (warp == 9 + 4 * Sh::kGroups) issue<NT, PT>(sm, walker, lane);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (thread == 0 && sm.abort_flag && p.error_word) atomicOr(p.error_word, (int)BDFP4_DEV_WAIT_TIMEOUT);
  if (warp == 0) tc::tmem_dealloc(sm.tmem, 512);
}

template <int NT, int PT>
static cudaError_t launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream) {
  const int smem = (int)sizeof(Smem<NT>) + 1024;
  static PerDeviceOnce configured;
  const int slot = current_device_slot();
  if (slot < 0 || !configured.done[slot]) {
    cudaError_t e = cudaFuncSetAttribute(tree_wide_kernel<NT, PT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (slot >= 0) configured.done[slot] = true;
  }
  tree_wide_kernel<NT, PT><<<kCtas, Shape<NT>::kThreads, smem, stream>>>(k_map, v_map, p);
  return cudaGetLastError();
}

}  // namespace wide
}  // namespace tree
}  // namespace bdfp4
