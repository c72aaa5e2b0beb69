// The tree attention for tiles of 64 to 128 queries: the same products as tree_narrow.cuh's with warps of one role
// each, one CTA per SM. A step's keys and values are converted once for up to 128 queries, so what bounds it is
// the softmax: 128 x NT exponentials and their surroundings, four groups of 128 threads with at most 32 queries
// per thread. Both products are kind::f16 with the converted cache side in tensor memory.
#pragma once

#include "tree_common.cuh"

namespace bdfp4 {
namespace tree {
namespace wide {

// Named barriers: one per softmax group (four at most), all softmax threads, the key threads.
constexpr int kCtas = kTreeWideCtas;
constexpr int kGroupBarrier = 1, kSoftmaxBarrier = 5, kKeysBarrier = 6;

// A softmax thread holds at most 32 queries: their sums stay in registers for a whole unit, and with 64 (128
// threads for NT = 64, 256 for 128) the kernel spilled, into an L1 that shared memory has left 24 KB of.
template <int NT>
struct Shape {
  static constexpr int kColumns = NT < 32 ? NT : 32;        // queries per softmax thread
  static constexpr int kGroups = NT / kColumns;             // softmax groups of 128 threads
  static constexpr int kBlocks = (NT + 63) / 64;            // 128-byte rows of P per token
  static constexpr int kKBuffers = NT > 96 ? 1 : 2;         // operand buffers in tensor memory, as many as it holds
  static constexpr int kVBuffers = NT > 64 ? 1 : 2;
  static constexpr int kStages = NT > 96 ? 5 : NT > 64 ? 6 : 8;
  static constexpr int kSoftmaxThreads = 128 * kGroups;
  static constexpr int kThreads = 256 + kSoftmaxThreads + 128;  // keys, values, softmax, control (two of its warps idle)
  // Registers per thread at launch and after the warpgroups have traded them: the sum over the warpgroups
  // must not exceed what the launch was given.
  static constexpr int kLaunchRegs = kGroups == 4 ? 72 : kGroups == 3 ? 80 : kGroups == 2 ? 96 : 128;
  static constexpr int kSoftmaxRegs = kGroups == 4 ? 80 : kGroups == 3 ? 96 : kGroups == 2 ? 112 : 144;
  static constexpr int kKeyRegs = kGroups == 4 ? 80 : kGroups == 3 ? 88 : kGroups == 2 ? 112 : 152;
  static constexpr int kValueRegs = kGroups == 4 ? 64 : kGroups == 3 ? 64 : kGroups == 2 ? 88 : 128;
  static constexpr int kControlRegs = kGroups == 4 ? 40 : kGroups == 3 ? 40 : kGroups == 2 ? 56 : 88;
  static_assert(kSoftmaxRegs * kGroups + kKeyRegs + kValueRegs + kControlRegs <= kLaunchRegs * (3 + kGroups), "registers");
  static_assert(kLaunchRegs * kThreads <= 65536, "registers");
  static constexpr bool kHold = kGroups <= 2;  // a thread's scores stay in registers between the vote and the exponentials
  // tensor memory columns
  static constexpr int kS = 0, kO = 2 * NT, kK = 3 * NT, kV = kK + 64 * kKBuffers;
  static_assert(kV + 64 * kVBuffers <= 512, "tensor memory");
};

template <int FROM, int TO>
__device__ __forceinline__ void trade_registers() {
  if constexpr (TO > FROM) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TO));
  if constexpr (TO < FROM) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TO));
}

template <int NT>
struct Smem {
  using Sh = Shape<NT>;
  alignas(1024) uint8_t ring[Sh::kStages][kStage];
  alignas(1024) uint8_t q[2][NT * 128];  // two halves of 64 channels, K-major, 128-byte swizzle
  alignas(1024) uint8_t p[2][Sh::kBlocks * 16384];  // MN-major: 128-byte rows of 64 queries per token, swizzled
  uint64_t family[NT];  // draft nodes each query sees
  float base[NT];       // kShift - maximum
  float top[NT];        // maximum, log2 units
  float factor[NT];
  float total[NT];
  float col_max[4][NT];
  float col_sum[4][NT];
  float key_factor[8][128];  // what undoes the scaling of a BF16 step's keys, by step number
  float q_max[16];
  int parents[BDFP4_MAX_TREE_NODES];
  uint64_t full_k[Sh::kStages], full_v[Sh::kStages], empty[Sh::kStages];
  uint64_t ka_full[2], ka_empty[2], va_full[2], va_empty[2];
  uint64_t s_full[2], s_empty[2], p_full[2], p_empty[2];
  uint64_t q_full, o_full, o_empty, drained;
  long long sums[Sh::kThreads / 32];
  int start_row;
  long long start_offset, first, last, per_cta;
  uint32_t tmem;
  int abort_flag, ignored_flag;
};

template <int NT, int PT>
__device__ __forceinline__ void produce(const TreeParams& p, Smem<NT>& sm, Walker walker, const CUtensorMap* k_map,
                                        const CUtensorMap* v_map, int lane) {
  using Sh = Shape<NT>;
  constexpr int kEntries = kPage / PT;
  const int64_t tail_row = (int64_t)p.heads_kv * kHeadDim;
  int slot = 0, issued = 0;
  uint32_t turn = 0;
  auto advance = [&] {
    ++issued;
    if (++slot == Sh::kStages) slot = 0, turn ^= 1;
  };
  Unit u;
  bool known = false;
  for (; walker.next(u, known); known = true) {
    const int32_t* table = p.table + u.row * p.table_stride;
    const int stop = min(u.end, u.info.pages);
    for (int batch = u.begin; batch < stop; batch += 32 / kEntries) {
      const int entry = batch * kEntries + lane;
      int mine = 0;
      if (entry < stop * kEntries) {
        mine = table[entry];
        if (mine < 0 || mine >= p.pages) {
          if (p.error_word) atomicOr(p.error_word, (int)BDFP4_DEV_BAD_PAGE);
          mine = 0;
        }
      }
      const int steps = min(32 / kEntries, stop - batch);
      for (int i = 0; i < steps; ++i) {
        int page[kEntries];
#pragma unroll
        for (int e = 0; e < kEntries; ++e) page[e] = __shfl_sync(0xffffffffu, mine, i * kEntries + e);
        wait(&sm.empty[slot], turn ^ 1, &sm.abort_flag);
        if (elect_one()) {
          uint8_t* stage = sm.ring[slot];
          tc::mbar_expect_tx(&sm.full_k[slot], 9216);
          tc::mbar_expect_tx(&sm.full_v[slot], 9216);
          if constexpr (PT == 128) {
            tc::tma_load_4d(stage, k_map, &sm.full_k[slot], 0, u.head, 0, page[0]);
            tc::bulk_load(stage + kKsOffset, p.scales[0] + page[0] * p.scales_pitch[0] + u.head * 1024, 1024, &sm.full_k[slot]);
            tc::tma_load_3d(stage + kVOffset, v_map, &sm.full_v[slot], 0, u.head * kHeadDim, page[0]);
            tc::bulk_load(stage + kVsOffset, p.scales[1] + page[0] * p.scales_pitch[1] + u.head * 1024, 1024, &sm.full_v[slot]);
          } else {
#pragma unroll
            for (int e = 0; e < kEntries; ++e) {
              tc::bulk_load(stage + e * 4096, p.codes[0] + page[e] * p.codes_pitch[0] + u.head * 4096, 4096, &sm.full_k[slot]);
              tc::bulk_load(stage + kKsOffset + e * 512, p.scales[0] + page[e] * p.scales_pitch[0] + u.head * 512, 512,
                            &sm.full_k[slot]);
              tc::bulk_load(stage + kVOffset + e * 4096, p.codes[1] + page[e] * p.codes_pitch[1] + u.head * 4096, 4096,
                            &sm.full_v[slot]);
              tc::bulk_load(stage + kVsOffset + e * 512, p.scales[1] + page[e] * p.scales_pitch[1] + u.head * 512, 512,
                            &sm.full_v[slot]);
            }
          }
        }
        __syncwarp();
        advance();
      }
    }
    for (int step = max(u.begin, u.info.pages); step < u.end; ++step) {
      const StepKind kind = step_kind(u.info, step);
      const int places = bf16_places(u.info, kind);
      for (int side = 0; side < 2; ++side) {
        const __nv_bfloat16* tail = (side ? p.tail_value : p.tail_key) + u.info.slot * p.tail_slot + u.head * kHeadDim;
        const __nv_bfloat16* draft = side ? p.draft_value + u.row * p.draft_value_row + u.head * kHeadDim
                                          : p.draft_key + u.row * p.draft_key_row + u.head * kHeadDim;
        const int64_t draft_node = side ? p.draft_value_node : p.draft_key_node;
        for (int first = 0; first < places; first += kBf16Rows) {
          const int end = min(first + kBf16Rows, places);
          uint64_t* full = side ? &sm.full_v[slot] : &sm.full_k[slot];
          wait(&sm.empty[slot], turn ^ 1, &sm.abort_flag);
          if (elect_one()) {
            // the sink's places behind its length stay empty
            const int absent = kind == kStepDraft && first == 0 ? BDFP4_MAX_SINK - u.info.sink : 0;
            tc::mbar_expect_tx(full, (end - first - absent) * 256);
            tc::mbar_arrive(side ? &sm.full_k[slot] : &sm.full_v[slot]);  // the other side only passes the stage on
          }
          __syncwarp();
          for (int i = first + lane; i < end; i += 32) {
            const __nv_bfloat16* source = nullptr;
            if (kind == kStepTail) source = tail + i * tail_row;
            else if (i >= BDFP4_MAX_SINK) source = draft + (i - BDFP4_MAX_SINK) * draft_node;
            else if (i < u.info.sink) source = tail + (kPage + i) * tail_row;
            if (source) tc::bulk_load(sm.ring[slot] + (i - first) * kBf16Pitch, source, 256, full);
          }
          __syncwarp();
          advance();
        }
      }
    }
  }
  // After an abort nobody else waits for the copies still in flight: no CTA may end under them.
  if (lane == 0 && *static_cast<volatile int*>(&sm.abort_flag)) {
    for (int back = min(issued, Sh::kStages); back > 0; --back) {
      const int at = issued - back;
      wait(&sm.full_k[at % Sh::kStages], (at / Sh::kStages) & 1, &sm.ignored_flag);
      wait(&sm.full_v[at % Sh::kStages], (at / Sh::kStages) & 1, &sm.ignored_flag);
    }
  }
  __syncwarp();
}

// The whole warp walks and waits; one thread of it issues.
template <int NT>
__device__ __forceinline__ void issue(Smem<NT>& sm, Walker walker) {
  using Sh = Shape<NT>;
  constexpr uint32_t kScores = f16_idesc(NT, 0, false), kPages = f16_idesc(NT, 0, true), kBf16 = f16_idesc(NT, 1, true);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const uint32_t q = tc::smem_u32(sm.q), prob = tc::smem_u32(sm.p);
  int n = 0, unit = 0;
  Unit u;
  bool known = false;
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
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const int a = n % Sh::kKBuffers;
      wait(&sm.ka_full[a], (n / Sh::kKBuffers) & 1, &sm.abort_flag);
      wait(&sm.s_empty[n & 1], ((n >> 1) & 1) ^ 1, &sm.abort_flag);
      tc::fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          mma_ts(tmem + Sh::kS + (n & 1) * NT, tmem + Sh::kK + a * 64 + s * 8,
                 tc::bf16_tile_desc(q + (s >> 2) * NT * 128, s & 3), kScores, s > 0);
        tc::commit(&sm.s_full[n & 1]);
        tc::commit(&sm.ka_empty[a]);
      }
      __syncwarp();
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

// One side of the ring as its consumers (four warps) see it.
template <int NT>
struct Ring {
  Smem<NT>& sm;
  uint64_t* full;
  int lane, slot;
  uint32_t turn;
  __device__ Ring(Smem<NT>& s, uint64_t* f, int l) : sm(s), full(f), lane(l), slot(0), turn(0) {}
  __device__ __forceinline__ const uint8_t* arrived() {
    wait(&full[slot], turn, &sm.abort_flag);
    return sm.ring[slot];
  }
  __device__ __forceinline__ void release() {
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.empty[slot]);
    if (++slot == Shape<NT>::kStages) slot = 0, turn ^= 1;
  }
  __device__ __forceinline__ void pass(int stages) {
    for (int i = 0; i < stages; ++i) {
      arrived();
      release();
    }
  }
};

// Keys: thread t holds token t of every step.
template <int NT, int PT>
__device__ __forceinline__ void keys(const TreeParams& p, Smem<NT>& sm, Walker walker, int t) {
  using Sh = Shape<NT>;
  const int lane = t & 31;
  const uint32_t tmem = sm.tmem + Sh::kK + ((uint32_t)(t & ~31) << 16);
  Ring<NT> ring(sm, sm.full_k, lane);
  int n = 0;
  Unit u;
  bool known = false;
  for (; walker.next(u, known); known = true) {
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      const uint32_t operand = tmem + (n % Sh::kKBuffers) * 64;
      uint64_t* operand_empty = &sm.ka_empty[n % Sh::kKBuffers];
      const uint32_t empty_parity = ((n / Sh::kKBuffers) & 1) ^ 1;
      if (kind == kStepPage) {
        const uint8_t* stage = ring.arrived();
        uint4 chunk[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) chunk[j] = *reinterpret_cast<const uint4*>(stage + t * 64 + ((j ^ ((t >> 1) & 3)) * 16));
        const uint8_t* at = PT == 128 ? stage + kKsOffset + (t & 31) * 16 + (t >> 5) * 4
                                      : stage + kKsOffset + (t >> 6) * 512 + (t & 31) * 8 + ((t >> 5) & 1) * 4;
        const uint32_t scales[2] = {*reinterpret_cast<const uint32_t*>(at),
                                    *reinterpret_cast<const uint32_t*>(at + (PT == 128 ? 512 : 256))};
        ring.release();
        wait(operand_empty, empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
#pragma unroll
        for (int j = 0; j < 4; ++j) store_dequantized(operand + 16 * j, chunk[j], scales[j >> 1] >> (16 * (j & 1)));
      } else {
        const int places = bf16_places(u.info, kind);
        const int stages = (places + kBf16Rows - 1) / kBf16Rows;
        // a step's stages are held together; both have arrived when each has been waited for
        ring.arrived();
        uint8_t* const stage0 = sm.ring[ring.slot];
        uint8_t* stage1 = stage0;
        if (stages > 1) {
          const bool wraps = ring.slot + 1 == Sh::kStages;
          const int next = wraps ? 0 : ring.slot + 1;
          wait(&sm.full_k[next], ring.turn ^ (wraps ? 1u : 0u), &sm.abort_flag);
          stage1 = sm.ring[next];
        }
        auto row_of = [&](int place) { return (place < kBf16Rows ? stage0 : stage1) + (place & (kBf16Rows - 1)) * kBf16Pitch; };
        bool there = t < places;
        if (kind == kStepDraft) {
          if (t < BDFP4_MAX_SINK) there = t < u.info.sink;
          if (p.rotate || p.key_shift) {  // eight threads bring one draft key into the cache's basis, in place
            const int group = t & 7;
            const float* shift = p.key_shift ? p.key_shift + u.head * kHeadDim + group * kGroup : nullptr;
            for (int first = 0; first < u.info.count; first += 16) {
              // (threads past the last draft follow along for the exchange; what they make of it goes nowhere)
              const int node = min(first + (t >> 3), u.info.count - 1);
              uint4* at = reinterpret_cast<uint4*>(row_of(BDFP4_MAX_SINK + node) + group * 32);
              const uint4 raw[2] = {at[0], at[1]};
              const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
              float v[16];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
              }
              cache_basis16_any(v, group, p.rotate != 0, shift);
              if (first + (t >> 3) < u.info.count) store_bf16x16(reinterpret_cast<__nv_bfloat16*>(at), v);
            }
            tc::fence_proxy_async_smem();  // the stage is overwritten by copies next
            bar_sync(kKeysBarrier, 128);
          }
        }
        const uint4* row = reinterpret_cast<const uint4*>(row_of(min(t, places - 1)));
        float amax = 0.0f;
        if (there) {
#pragma unroll 4
          for (int j = 0; j < 16; ++j) {
            const uint4 r = row[j];
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
          }
        }
        float inverse;
        const float scale = scale_to<14>(amax, &inverse);
        sm.key_factor[n & 7][t] = inverse;
        wait(operand_empty, empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
#pragma unroll 1
        for (int quarter = 0; quarter < 4; ++quarter) {
          uint32_t v[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 r = make_uint4(0, 0, 0, 0);
            if (there) r = row[quarter * 4 + j];
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[4 * j + i] = h2(__floats2half2_rn(__uint_as_float(w[i] << 16) * scale, __uint_as_float(w[i] & 0xffff0000u) * scale));
          }
          st16(operand + quarter * 16, v);
        }
        for (int i = 0; i < stages; ++i) ring.release();
        ring.pass(stages);  // the values'
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.ka_full[n % Sh::kKBuffers]);
    }
  }
}

// Values: thread c holds channel c of every step.
template <int NT, int PT>
__device__ __forceinline__ void values(const TreeParams& p, Smem<NT>& sm, Walker walker, int c) {
  using Sh = Shape<NT>;
  const int lane = c & 31;
  const uint32_t tmem = sm.tmem + Sh::kV + ((uint32_t)(c & ~31) << 16);
  Ring<NT> ring(sm, sm.full_v, lane);
  int n = 0;
  Unit u;
  bool known = false;
  for (; walker.next(u, known); known = true) {
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      const uint32_t operand = tmem + (n % Sh::kVBuffers) * 64;
      uint64_t* operand_empty = &sm.va_empty[n % Sh::kVBuffers];
      const uint32_t empty_parity = ((n / Sh::kVBuffers) & 1) ^ 1;
      if (kind == kStepPage) {
        const uint8_t* stage = ring.arrived();
        uint4 chunk[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* at = PT == 128 ? stage + kVOffset + c * 64 + ((j ^ ((c >> 1) & 3)) * 16)
                                        : stage + kVOffset + (j >> 1) * 4096 + c * 32 + (((j & 1) ^ ((c >> 2) & 1)) * 16);
          chunk[j] = *reinterpret_cast<const uint4*>(at);
        }
        const uint8_t* at = stage + kVsOffset + (c & 31) * 16 + (c >> 5) * 4;
        const uint32_t scales[2] = {*reinterpret_cast<const uint32_t*>(at), *reinterpret_cast<const uint32_t*>(at + 512)};
        ring.release();
        wait(operand_empty, empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
#pragma unroll
        for (int j = 0; j < 4; ++j) store_dequantized(operand + 16 * j, chunk[j], scales[j >> 1] >> (16 * (j & 1)));
      } else {
        const int places = bf16_places(u.info, kind);
        ring.pass((places + kBf16Rows - 1) / kBf16Rows);  // the keys'
        wait(operand_empty, empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
        for (int first = 0; first < places; first += kBf16Rows) {
          const uint8_t* stage = ring.arrived() + 2 * c;
          const int slices = (min(places - first, kBf16Rows) + 15) / 16;
          for (int s = 0; s < slices; ++s) {
            const int place = first + s * 16;
            const int stop = kind == kStepDraft && place == 0 ? u.info.sink : places;
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint32_t lo = 0, hi = 0;
              if (place + 2 * i < stop) lo = *reinterpret_cast<const uint16_t*>(stage + (s * 16 + 2 * i) * kBf16Pitch);
              if (place + 2 * i + 1 < stop) hi = *reinterpret_cast<const uint16_t*>(stage + (s * 16 + 2 * i + 1) * kBf16Pitch);
              v[i] = lo | (hi << 16);
            }
            st8(operand + (place >> 4) * 8, v);
          }
          ring.release();
        }
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.va_full[n % Sh::kVBuffers]);
    }
  }
}

// The tile's queries into shared memory: rotated if asked, scaled by one power of two into FP16's range
// (rows of the tile whose largest value is 2^-29 of the tile's keep full precision). Returns what undoes it.
template <int NT>
__device__ __forceinline__ float load_queries(const TreeParams& p, Smem<NT>& sm, const Unit& u, int thread) {
  using Sh = Shape<NT>;
  constexpr int kPerPass = Sh::kSoftmaxThreads / 8, kPasses = NT / kPerPass;
  const int group = thread & 7;
  const int queries = u.info.count * p.ratio;
  float v[kPasses][16];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int query = u.tile * NT + i * kPerPass + (thread >> 3);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[i][j] = 0.0f;
    if (query < queries)
      load_bf16x16(p.query + u.row * p.query_row + (query / p.ratio) * p.query_node +
                       (int64_t)(u.head * p.ratio + query % p.ratio) * kHeadDim + group * kGroup, v[i]);
  }
  if (thread < BDFP4_MAX_TREE_NODES) sm.parents[thread] = thread < u.info.count ? p.parents[u.row * p.parents_row + thread] : -1;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    if (p.rotate) {
      hadamard_butterflies(v[i], group);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[i][j] *= kInvSqrt128;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (fabsf(v[i][j]) < INFINITY) amax = fmaxf(amax, fabsf(v[i][j]));
  }
  amax = warp_max(amax);
  if ((thread & 31) == 0) sm.q_max[thread >> 5] = amax;
  bar_sync(kSoftmaxBarrier, Sh::kSoftmaxThreads);
#pragma unroll
  for (int w = 0; w < Sh::kSoftmaxThreads / 32; ++w) amax = fmaxf(amax, sm.q_max[w]);
  float inverse;
  const float scale = scale_to<14>(amax, &inverse);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kPerPass + (thread >> 3);
    uint8_t* row = sm.q[group >> 2] + r * 128;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = h2(__floats2half2_rn(v[i][2 * j] * scale, v[i][2 * j + 1] * scale));
    const int chunk = (group & 3) * 2;
    *reinterpret_cast<uint4*>(row + ((chunk ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ (r & 7)) * 16)) = make_uint4(w[4], w[5], w[6], w[7]);
  }
  tc::fence_proxy_async_smem();
  bar_sync(kSoftmaxBarrier, Sh::kSoftmaxThreads);
  if (thread == 0) tc::mbar_arrive(&sm.q_full);
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
  Unit u;
  if (!walker.next(u, false)) return;
  bool more = true;
  float q_inverse = load_queries<NT>(p, sm, u, thread);
  while (more) {
    for (int j = t; j < C; j += 128) {
      top[j] = kNoMax;
      base[j] = kShift - kNoMax;
      // the draft nodes the query of column j sees
      const int query = u.tile * NT + first_column + j;
      uint64_t seen = 0;
      for (int node = min(query / p.ratio, u.info.count - 1); node >= 0;) {
        seen |= 1ull << node;
        const int parent = sm.parents[node];
        node = parent < node ? parent : -1;
      }
      sm.family[first_column + j] = seen;
    }
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
      const int node = t - BDFP4_MAX_SINK;
      wait(&sm.s_full[n & 1], (n >> 1) & 1, &sm.abort_flag);
      tc::fence_after_sync();
      float f = page_factor;
      if (kind != kStepPage) f = p.scale_log2 * q_inverse * sm.key_factor[n & 7][t];
      const float2 f2 = make_float2(f, f);
      const uint32_t scores = sm.tmem + Sh::kS + (n & 1) * NT + first_column + lanes;
      auto load16 = [&](int j, float* s) {
        tc::tmem_ld16(scores + j, s);
        tc::tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((sm.family[first_column + j + i] >> node) & 1)) s[i] = -INFINITY;
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
          if (lane < 16) sm.col_max[warp][first_column + j + lane] = mine;
        }
        bar_sync(barrier, 128);
        for (int j = t; j < C; j += 128) {
          const int col = first_column + j;
          const float before = top[j];
          const float now = fmaxf(fmaxf(fmaxf(sm.col_max[0][col], sm.col_max[1][col]),
                                        fmaxf(sm.col_max[2][col], sm.col_max[3][col])), before);
          top[j] = now;
          base[j] = kShift - now;
          sm.factor[col] = ex2(before - now);
        }
        bar_sync(barrier, 128);
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
        if constexpr (Sh::kHold) {
#pragma unroll
          for (int j = 0; j < C; j += 16) {
            load16(j, held + j);
            above16(j, held + j);
          }
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
      for (int j = 0; j < C; j += 16) {
        float* s = Sh::kHold ? held + j : held;
        if constexpr (!Sh::kHold) {
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
      reduce_columns<C, 16>(v, lane, 0, [&](int j, float total) { sm.col_sum[warp][first_column + j] = total; });
    }
    // the next unit's queries go in while this one's last product runs: all its scores are done
    Unit following = u;
    more = walker.next(following, true);
    float next_inverse = 1.0f;
    bar_sync(kSoftmaxBarrier, Sh::kSoftmaxThreads);  // both groups have seen their last scores; the parents are free
    if (more) next_inverse = load_queries<NT>(p, sm, following, thread);
    bar_sync(barrier, 128);
    const bool whole = u.begin == 0 && u.end == u.info.steps;
    // a part that begins a unit goes to the CTA's second slot, one that continues it to the first
    const int part = 2 * blockIdx.x + (u.begin == 0 ? 1 : 0);
    for (int j = t; j < C; j += 128) {
      const int col = first_column + j;
      const float total = (sm.col_sum[0][col] + sm.col_sum[1][col]) + (sm.col_sum[2][col] + sm.col_sum[3][col]);
      if (whole) {
        sm.total[col] = total > 0.0f ? p.value_scale / total : 0.0f;
      } else {
        p.partial_stat[(int64_t)(2 * part) * NT + col] = top[j];
        p.partial_stat[(int64_t)(2 * part + 1) * NT + col] = total;
      }
    }
    bar_sync(barrier, 128);
    wait(&sm.o_full, unit & 1, &sm.abort_flag);
    tc::fence_after_sync();
    const int queries = min(u.info.count * p.ratio - u.tile * NT - first_column, C);
    int query = u.tile * NT + first_column;
    int out_node = query / p.ratio, out_head = query % p.ratio;
    __nv_bfloat16* out = p.out + u.row * p.out_row + (int64_t)u.head * p.ratio * kHeadDim + t;
    float* partial = p.partial + ((int64_t)part * NT + first_column) * kHeadDim + t;
#pragma unroll
    for (int j = 0; j < C; j += 16) {
      float o[16];
      tc::tmem_ld16(sm.tmem + Sh::kO + first_column + j + lanes, o);
      tc::tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (j + i < queries) {
          if (whole) {
            out[out_node * p.out_node + out_head * kHeadDim] = __float2bfloat16_rn(o[i] * sm.total[first_column + j + i]);
            if (++out_head == p.ratio) out_head = 0, ++out_node;
          } else {
            partial[(int64_t)(j + i) * kHeadDim] = o[i];
          }
        }
      }
    }
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.o_empty);
    bar_sync(barrier, 128);  // base, top and total are written anew
    if (!whole && u.begin == 0 && thread == 0) {
      TreeSplit split;
      split.row = u.row;
      split.head = u.head;
      split.tile = u.tile;
      // the unit's last step, counted over the whole launch, names the CTA it ends in
      split.last = (int)((sm.last + (u.info.steps - u.end) - 1) / sm.per_cta);
      p.splits[blockIdx.x] = split;
    }
    q_inverse = next_inverse;
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

  // all steps of the launch, and where this CTA's run begins
  long long mine = 0;
  for (int row = thread; row < p.rows; row += Sh::kThreads) {
    const RowInfo r = row_info(p, row, PT);
    mine += (long long)r.steps * r.tiles * p.heads_kv;
  }
  for (int step = 16; step > 0; step >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, step);
  if (lane == 0) sm.sums[warp] = mine;
  if (thread == 0) {
    for (int i = 0; i < Sh::kStages; ++i) {
      tc::mbar_init(&sm.full_k[i], 1);
      tc::mbar_init(&sm.full_v[i], 1);
      tc::mbar_init(&sm.empty[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sm.ka_full[i], 4);
      tc::mbar_init(&sm.va_full[i], 4);
      tc::mbar_init(&sm.ka_empty[i], 1);
      tc::mbar_init(&sm.va_empty[i], 1);
      tc::mbar_init(&sm.s_full[i], 1);
      tc::mbar_init(&sm.s_empty[i], 4 * Sh::kGroups);
      tc::mbar_init(&sm.p_full[i], 4 * Sh::kGroups);
      tc::mbar_init(&sm.p_empty[i], 1);
    }
    tc::mbar_init(&sm.q_full, 1);
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
  __syncthreads();
  if (warp == 0) {
    long long all = 0;
    for (int w = 0; w < Sh::kThreads / 32; ++w) all += sm.sums[w];
    const long long per = max((all + gridDim.x - 1) / gridDim.x, 1ll);
    const long long first = per * blockIdx.x, last = min(first + per, all);
    if (lane == 0) {
      sm.per_cta = per;
      sm.first = first;
      sm.last = last;
    }
    long long before = 0;
    for (int row0 = 0; row0 < p.rows && first < last; row0 += 32) {
      long long steps = 0;
      if (row0 + lane < p.rows) {
        const RowInfo r = row_info(p, row0 + lane, PT);
        steps = (long long)r.steps * r.tiles * p.heads_kv;
      }
      long long upto = steps;
      for (int step = 1; step < 32; step <<= 1) {
        const long long left = __shfl_up_sync(0xffffffffu, upto, step);
        if (lane >= step) upto += left;
      }
      const unsigned holds = __ballot_sync(0xffffffffu, before + upto > first);
      if (holds) {
        if (lane == __ffs(holds) - 1) {
          sm.start_row = row0 + lane;
          sm.start_offset = first - (before + upto - steps);
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    __syncwarp();
    tc::tmem_alloc(&sm.tmem, 512);
    tc::tmem_relinquish();
    tc::fence_before_sync();
  }
  __syncthreads();
  tc::fence_after_sync();
  if (sm.first < sm.last) {
    const Walker walker(p, sm.start_row, (int)sm.start_offset, (int)(sm.last - sm.first), PT);
    if (warp < 4) {
      trade_registers<Sh::kLaunchRegs, Sh::kKeyRegs>();
      keys<NT, PT>(p, sm, walker, thread);
    } else if (warp < 8) {
      trade_registers<Sh::kLaunchRegs, Sh::kValueRegs>();
      values<NT, PT>(p, sm, walker, thread - 128);
    } else if (warp < 8 + 4 * Sh::kGroups) {
      trade_registers<Sh::kLaunchRegs, Sh::kSoftmaxRegs>();
      softmax<NT>(p, sm, walker, thread - 256);
    } else {
      trade_registers<Sh::kLaunchRegs, Sh::kControlRegs>();
      if (warp == 8 + 4 * Sh::kGroups) produce<NT, PT>(p, sm, walker, &k_map, &v_map, lane);
      if (warp == 9 + 4 * Sh::kGroups) issue<NT>(sm, walker);
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
