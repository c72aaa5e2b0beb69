// Attention of a tree of drafted tokens over the paged NVFP4 cache, on the tensor cores: what its two kernels share.
//
// Per (row, KV head) the queries are one matrix of nodes x ratio rows, cut into tiles of NT. Against 128
// tokens at a time,
//     S^T [token, query]   = K   [token, channel]  * Q^T
//     O^T [channel, query] = V^T [channel, token] * P^T
//
// S^T over a page is the block-scaled FP4 product of the codes as they lie in the cache (kind::mxf4nvf4, no
// conversion) with the query written as a sum of four FP4 terms, each the rounding of what the ones before left: a
// term leaves at most 0.178 of its group's largest value (half the widest E2M1 step of amax / 6, with the E4M3
// scale's rounding), four leave 10^-3 of it: a quarter of what BF16 rounding may cost the group's largest value, four
// times what it may cost one a sixteenth as large. Four terms of K = 64 take the tensor time of FP16's K = 16.
// (Converting K to FP16 instead cost a third of the conversions and a chain of waits: 350 us where the terms take 331,
// 120 against 99 for tiles of 64.)
//
// O^T over a page is a kind::f16 product with V^T in tensor memory: E2M1 x E4M3 has at most six significant bits and
// lies in [2^-10, 2688], so a page's values are exact in FP16. A thread reads its own channel's code bytes, converts
// and scales them in registers and stores them straight into its tensor-memory lane; the converted tile never passes
// through shared memory. P is stored as the softmax threads hold it, one token per thread with its queries
// contiguous, which is the MN-major form of operand B; it is not rounded to FP4, but to FP16.
//
// Softmax maxima are per query, in shared memory, and lazy: probabilities are formed against them at once, and only
// when a score exceeds its query's by more than 8 (log2; the step's barrier carries that vote) are the maxima taken
// anew and O^T rescaled. (Where scores are so large that what rounding does to a maximum counts, above 2^24, the two
// kernels see to it in their own ways that the largest still gets its weight and no more.) Sums are FP32, per thread
// until the unit ends, of the probabilities as they are before their rounding. Probabilities carry a factor 2^7, so in
// FP16 they stay below 2^15 and lose nothing above 2^-31 of the largest.
//
// The rolling tail and the drafts with the sink are two more steps over BF16 values, both products kind::f16 with the
// cache side in tensor memory: K is scaled per token by a power of two into FP16's range (the softmax thread of the
// token undoes it), V and P are BF16. P has to have V's type, and V has no scale that would bring it into FP16's
// range: one per channel cannot be undone in a sum that runs on over the pages, one per step would cost a channel that
// is quiet beside another its values. So the probabilities of these up to 208 tokens are rounded to 2^-8, the pages' to
// 2^-11; for short rows that is as much as the output's own rounding.
//
// Work is the sequence of all steps of all (row, head, tile) units, cut into runs, one per CTA, so any mix of lengths
// is balanced; a unit that straddles CTAs leaves unnormalised parts that a second kernel adds.
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
      if (p.sink) r.sink = min(max(p.sink[row], 0), p.sink_rows);
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

// C columns of this thread's lane in tensor memory times `by` of each, in place. (Out of the way of the loops that read
// scores: a second branch there cost 3.4% of one long row's time, a factor per column 16%, this form 1.7%.)
template <int C>
__device__ __forceinline__ void scale_columns(uint32_t at, const float* by) {
#pragma unroll 1
  for (int j = 0; j < C; j += 8) {
    float s[8];
    tc::tmem_ld8(at + j, s);
    tc::tmem_wait_ld();
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(s[i] * by[j + i]);
    st8(at + j, w);
  }
  tc::tmem_wait_st();
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

// The launch's steps in a row, cut into equal runs, one per CTA: who does which.
//
// A cut within `snap` steps of a unit's end moves there. A unit that straddles a cut costs a second set-up, parts
// through memory and the merge, together about as much as that many steps.
struct Plan {
  long long steps;  // all of them
  long long per;    // of one CTA, before a cut moves
  int snap;

  // Where the cut at `x` within the unit [begin, end) goes.
  __device__ __forceinline__ long long moved(long long x, long long begin, long long end) const {
    const long long down = x - begin, up = end - x;
    if (min(down, up) > snap) return x;
    return down <= up ? begin : end;
  }
  // The CTA that does the last step of the unit [begin, end).
  __device__ __forceinline__ int owner_of_last(long long begin, long long end) const {
    long long cta = (end - 1) / per;
    while (cta * per > begin && moved(cta * per, begin, end) >= end) --cta;
    return (int)cta;
  }
};

// All threads of a CTA. Fills sm.plan, sm.start_row, sm.start_offset, sm.first and sm.last (valid after the next
// barrier of the CTA).
template <int PT, int THREADS, int SNAP, typename Smem>
__device__ __forceinline__ void make_plan(const TreeParams& p, Smem& sm, int thread) {
  const int lane = thread & 31, warp = thread >> 5;
  long long mine = 0;
#pragma unroll 1
  for (int row = thread; row < p.rows; row += THREADS) {
    const RowInfo r = row_info(p, row, PT);
    mine += (long long)r.steps * r.tiles * p.heads_kv;
  }
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, step);
  if (lane == 0) sm.sums[warp] = mine;
  __syncthreads();
  if (warp != 0) return;
  Plan plan;
  plan.steps = 0;
  for (int w = 0; w < THREADS / 32; ++w) plan.steps += sm.sums[w];
  plan.per = max((plan.steps + gridDim.x - 1) / gridDim.x, 1ll);
  plan.snap = (int)min((long long)SNAP, plan.per - 1);
  const long long cut[2] = {min(plan.per * blockIdx.x, plan.steps), min(plan.per * (blockIdx.x + 1), plan.steps)};
  if (lane == 0) {
    sm.plan = plan;
    sm.first = sm.last = plan.steps;
    sm.start_row = p.rows;
    sm.start_offset = 0;
  }
  __syncwarp();
  long long before = 0;
#pragma unroll 1
  for (int row0 = 0; row0 < p.rows && before <= cut[1] && cut[0] < plan.steps; row0 += 32) {
    RowInfo r;
    long long steps = 0;
    if (row0 + lane < p.rows) {
      r = row_info(p, row0 + lane, PT);
      steps = (long long)r.steps * r.tiles * p.heads_kv;
    }
    long long upto = steps;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const long long left = __shfl_up_sync(0xffffffffu, upto, step);
      if (lane >= step) upto += left;
    }
    const long long begin = before + upto - steps;  // of this lane's row
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (steps > 0 && cut[i] >= begin && cut[i] < begin + steps) {
        const long long unit = begin + (cut[i] - begin) / r.steps * r.steps;
        const long long at = plan.moved(cut[i], unit, unit + r.steps);
        if (i == 0) {
          sm.first = at;
          sm.start_row = row0 + lane;
          sm.start_offset = at - begin;  // (the walk goes on to the next row from a row's end)
        } else {
          sm.last = at;
        }
      }
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  __syncwarp();
}

constexpr int kTerms = 4;  // FP4 terms of a query
constexpr int kCacheThreads = 256;  // that bring the cache side: two halves of 128

// A place in the ring of stages; everyone who keeps one visits every stage in order.
template <int STAGES>
struct Place {
  int slot = 0;
  uint32_t turn = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == STAGES) slot = 0, turn ^= 1;
  }
};

// The copies into the ring, by one warp. A page's step takes one stage, a BF16 step one per 64 tokens for K and then
// as many for V.
template <int PT, typename Smem>
__device__ __forceinline__ void produce(const TreeParams& p, Smem& sm, Walker walker, const CUtensorMap* k_map,
                                        const CUtensorMap* v_map, int lane) {
  constexpr int kEntries = kPage / PT;
  const int64_t tail_row = (int64_t)p.heads_kv * kHeadDim;
  Place<Smem::kStages> at;
  // No CTA may end under copies in flight, also when nobody waits for them any more. (A stage that was never filled,
  // or whose last use is over, is in a phase whose predecessor has ended.)
  auto drain = [&] {
#pragma unroll 1
    for (int i = 0; i < Smem::kStages; ++i) {
      wait(&sm.full[at.slot], at.turn ^ 1, &sm.ignored_flag);
      at.advance();
    }
  };
  // A stage's turn to be filled. False once somebody has given up: no barrier may be armed twice in a phase.
  auto emptied = [&]() -> bool {
    wait(&sm.empty[at.slot], at.turn ^ 1, &sm.abort_flag);
    return __all_sync(0xffffffffu, *static_cast<volatile int*>(&sm.abort_flag) == 0);
  };
  Unit u;
  bool known = false;
#pragma unroll 1
  for (; walker.next(u, known); known = true) {
    const int32_t* table = p.table + u.row * p.table_stride;
    const int stop = min(u.end, u.info.pages);
#pragma unroll 1
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
#pragma unroll 1
      for (int i = 0; i < steps; ++i) {
        int page[kEntries];
#pragma unroll
        for (int e = 0; e < kEntries; ++e) page[e] = __shfl_sync(0xffffffffu, mine, i * kEntries + e);
        if (!emptied()) return drain();
        uint64_t* const full = &sm.full[at.slot];
        if (elect_one()) {
          uint8_t* stage = sm.ring[at.slot];
          tc::mbar_expect_tx(full, 18432);
          if constexpr (PT == 128) {
            tc::tma_load_4d(stage, k_map, full, 0, u.head, 0, page[0]);
            tc::bulk_load(stage + kKsOffset, p.scales[0] + page[0] * p.scales_pitch[0] + u.head * 1024, 1024, full);
            tc::tma_load_3d(stage + kVOffset, v_map, full, 0, u.head * kHeadDim, page[0]);
            tc::bulk_load(stage + kVsOffset, p.scales[1] + page[0] * p.scales_pitch[1] + u.head * 1024, 1024, full);
          } else {
#pragma unroll
            for (int e = 0; e < kEntries; ++e) {
              tc::bulk_load(stage + e * 4096, p.codes[0] + page[e] * p.codes_pitch[0] + u.head * 4096, 4096, full);
              tc::bulk_load(stage + kKsOffset + e * 512, p.scales[0] + page[e] * p.scales_pitch[0] + u.head * 512, 512, full);
              tc::bulk_load(stage + kVOffset + e * 4096, p.codes[1] + page[e] * p.codes_pitch[1] + u.head * 4096, 4096, full);
              tc::bulk_load(stage + kVsOffset + e * 512, p.scales[1] + page[e] * p.scales_pitch[1] + u.head * 512, 512, full);
            }
          }
        }
        __syncwarp();
        at.advance();
      }
    }
#pragma unroll 1
    for (int step = max(u.begin, u.info.pages); step < u.end; ++step) {
      const StepKind kind = step_kind(u.info, step);
      const int places = bf16_places(u.info, kind);
#pragma unroll 1
      for (int side = 0; side < 2; ++side) {
        const __nv_bfloat16* tail = (side ? p.tail_value : p.tail_key) + u.info.slot * p.tail_slot + u.head * kHeadDim;
        const __nv_bfloat16* draft = side ? p.draft_value + u.row * p.draft_value_row + u.head * kHeadDim
                                          : p.draft_key + u.row * p.draft_key_row + u.head * kHeadDim;
        const int64_t draft_node = side ? p.draft_value_node : p.draft_key_node;
#pragma unroll 1
        for (int first = 0; first < places; first += kBf16Rows) {
          const int end = min(first + kBf16Rows, places);
          if (!emptied()) return drain();
          uint64_t* const full = &sm.full[at.slot];
          // the sink's places behind its length stay empty
          const int absent = kind == kStepDraft && first == 0 ? BDFP4_MAX_SINK - u.info.sink : 0;
          if (elect_one()) tc::mbar_expect_tx(full, (end - first - absent) * 256);
          __syncwarp();
#pragma unroll 1
          for (int i = first + lane; i < end; i += 32) {
            const __nv_bfloat16* source = nullptr;
            if (kind == kStepTail) source = tail + i * tail_row;
            else if (i >= BDFP4_MAX_SINK) source = draft + (i - BDFP4_MAX_SINK) * draft_node;
            else if (i < u.info.sink) source = tail + (kPage + i) * tail_row;
            if (source) tc::bulk_load(sm.ring[at.slot] + (i - first) * kBf16Pitch, source, 256, full);
          }
          __syncwarp();
          at.advance();
        }
      }
    }
  }
  drain();
  __syncwarp();
}

// The key scales of two 64-token pages into whole atoms, in place, by one warp.
__device__ __forceinline__ void interleave_scales(uint8_t* scales, int lane) {
  uint2 part[2][2];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    part[e & 1][e >> 1] = *reinterpret_cast<const uint2*>(scales + (e >> 1) * 512 + (e & 1) * 256 + lane * 8);
  __syncwarp();
#pragma unroll
  for (int atom = 0; atom < 2; ++atom)
    *reinterpret_cast<uint4*>(scales + atom * 512 + lane * 16) =
        make_uint4(part[atom][0].x, part[atom][0].y, part[atom][1].x, part[atom][1].y);
  tc::fence_proxy_async_smem();
  __syncwarp();
}

// The tile's queries into shared memory, a group of sixteen values per thread and pass: as kTerms FP4 terms for the
// pages, and as FP16 for the BF16 steps. Rotated if asked, and scaled by one power of two: a query whose largest
// value is 2^-5 of the tile's still has all four terms above E4M3's smallest normal scale. Where one's is less, every
// query is scaled by its own power of two instead (`uneven`), and its scores are brought down to the tile's
// (query_level): what is lost of a query goes by its own values, whatever the others of its tile are. Returns what
// undoes the tile's scale. sm.own: each query's largest value.
template <int NT, int THREADS, typename Smem>
__device__ __forceinline__ float load_queries(const TreeParams& p, Smem& sm, int barrier, const Unit& u, int thread,
                                              bool& uneven) {
  constexpr int kPerPass = THREADS / 8, kPasses = (NT + kPerPass - 1) / kPerPass;
  const int group = thread & 7;
  const int queries = min(u.info.count * p.ratio - u.tile * NT, NT);
  float v[kPasses][16];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kPerPass + (thread >> 3), query = u.tile * NT + r;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[i][j] = 0.0f;
    if (r < queries)
      load_bf16x16(p.query + u.row * p.query_row + (query / p.ratio) * p.query_node +
                       (int64_t)(u.head * p.ratio + query % p.ratio) * kHeadDim + group * kGroup, v[i]);
  }
  if (thread < BDFP4_MAX_TREE_NODES) sm.parents[thread] = thread < u.info.count ? p.parents[u.row * p.parents_row + thread] : -1;
  float amax = 0.0f, amin = INFINITY;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kPerPass + (thread >> 3);
    if (p.rotate) {
      hadamard_butterflies(v[i], group);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[i][j] *= kInvSqrt128;
    }
    float own = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (fabsf(v[i][j]) < INFINITY) own = fmaxf(own, fabsf(v[i][j]));
#pragma unroll
    for (int step = 4; step > 0; step >>= 1) own = fmaxf(own, __shfl_xor_sync(0xffffffffu, own, step));
    if (group == 0 && r < NT) sm.own[r] = own;
    amax = fmaxf(amax, own);
    if (own > 0.0f) amin = fminf(amin, own);
  }
  amax = warp_max(amax);
  amin = -warp_max(-amin);
  if ((thread & 31) == 0) sm.q_range[thread >> 5] = make_float2(amax, amin);
  bar_sync(barrier, THREADS);
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    amax = fmaxf(amax, sm.q_range[i].x);
    amin = fminf(amin, sm.q_range[i].y);
  }
  uneven = amin * 32.0f < amax;
  float inverse;
  const float scale = scale_to<10>(amax, &inverse);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kPerPass + (thread >> 3);
    if (kPasses * kPerPass > NT && r >= NT) break;
    float by = scale, ignored;
    if (uneven) by = scale_to<10>(sm.own[min(r, NT - 1)], &ignored);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[i][j] *= by;
    {
      uint8_t* row = sm.q[group >> 2] + r * 128;
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = h2(__floats2half2_rn(v[i][2 * j], v[i][2 * j + 1]));
      const int chunk = (group & 3) * 2;
      *reinterpret_cast<uint4*>(row + ((chunk ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ (r & 7)) * 16)) = make_uint4(w[4], w[5], w[6], w[7]);
    }
    const int at = r * 64 + group * 8;
#pragma unroll 1
    for (int term = 0; term < kTerms; ++term) {
      float largest = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) largest = fmaxf(largest, fabsf(v[i][j]));
      const uint32_t byte = cvt_e4m3(largest * (1.0f / 6.0f));
      GroupCodes codes;
      codes.scale = e4m3_to_float(byte);
      // (an approximate reciprocal: what it rounds otherwise is left to the next term)
      float inverse_scale;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse_scale) : "f"(fmaxf(codes.scale, 1.0e-30f)));
      float scaled[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) scaled[j] = v[i][j] * inverse_scale;
      codes.lo = pack_e2m1x8(scaled);
      codes.hi = pack_e2m1x8(scaled + 8);
      *reinterpret_cast<uint2*>(sm.q_codes[term] + (at ^ (((at >> 7) & 3) << 4))) = make_uint2(codes.lo, codes.hi);
      sm.q_scales[term][scale_tile_offset(r, group)] = (uint8_t)byte;
      float rest[16];
      group_residual16(v[i], codes, rest);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[i][j] = rest[j];
    }
  }
  tc::fence_proxy_async_smem();
  return inverse;
}

// What brings the scores of a query of an uneven tile, whose largest value is `own`, down to the tile's scale, which
// `inverse` undoes.
__device__ __forceinline__ float query_level(float own, float inverse) {
  float mine;
  scale_to<10>(own, &mine);
  return own > 0.0f ? mine / inverse : 1.0f;
}

// Channel t of a tile's queries out of tensor memory: `columns` of them from column `at` (of the tile's
// `first_column`) on, normalised to the output when the unit is whole, as they are to its part when not.
template <typename Smem>
__device__ __forceinline__ void store_output(const TreeParams& p, const Smem& sm, const Unit& u, uint32_t at, int tile,
                                             int first_column, int columns, bool whole, int part, int t) {
  const int query = u.tile * tile + first_column;
  int head = query % p.ratio;
  columns = min(columns, u.info.count * p.ratio - query);
  __nv_bfloat16* out = p.out + u.row * p.out_row + (query / p.ratio) * p.out_node +
                       ((int64_t)u.head * p.ratio + head) * kHeadDim + t;
  float* partial = p.partial + ((int64_t)part * tile + first_column) * kHeadDim + t;
  const int64_t next_node = p.out_node - (int64_t)(p.ratio - 1) * kHeadDim;
#pragma unroll 1
  for (int j = 0; j < columns; j += 8) {
    float o[8];
    tc::tmem_ld8(at + j, o);
    tc::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (j + i >= columns) break;
      if (whole) {
        *out = __float2bfloat16_rn(o[i] * sm.factor[first_column + j + i]);
        const bool wraps = ++head == p.ratio;
        out += wraps ? next_node : (int64_t)kHeadDim;
        if (wraps) head = 0;
      } else {
        *partial = o[i];
        partial += kHeadDim;
      }
    }
  }
}

// Which of up to 32 columns see each draft node: bit j of seen_by[node] is column j's. By one warp, lane j for
// column j of the tile's queries from `query` on. A column sees its own node and that node's ancestors.
__device__ __forceinline__ void make_masks(const TreeParams& p, const Unit& u, const int* parents, uint32_t* seen_by, int query,
                                           int lane) {
  uint64_t seen = 0;
#pragma unroll 1
  for (int node = min((query + lane) / p.ratio, u.info.count - 1); node >= 0;) {
    seen |= 1ull << node;
    const int parent = parents[node];
    node = parent < node ? parent : -1;
  }
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const uint32_t word = (uint32_t)(seen >> (32 * half));
    uint32_t mine = 0;
#pragma unroll 4
    for (int node = 0; node < 32; ++node) {
      const uint32_t all = __ballot_sync(0xffffffffu, (word >> node) & 1);
      if (lane == node) mine = all;
    }
    seen_by[32 * half + lane] = mine;
  }
}

// One stage's release, by a whole warp. A page's stage waits for its score product too; for a BF16 step's one
// warp arrives in its place.
template <typename Smem>
__device__ __forceinline__ void release(Smem& sm, Place<Smem::kStages>& at, int thread, bool bf16) {
  __syncwarp();
  if ((thread & 31) == 0) tc::mbar_arrive(&sm.empty[at.slot]);
  if (bf16 && thread == 0) tc::mbar_arrive(&sm.empty[at.slot]);
  at.advance();
}

// The keys of a BF16 step: thread r of either half brings its half of token r's channels. Returns what undoes
// the token's scaling.
template <typename Smem>
__device__ __forceinline__ float bf16_keys(const TreeParams& p, Smem& sm, int barrier, const Unit& u, StepKind kind,
                                           Place<Smem::kStages> at, uint32_t operand, int thread) {
  const int r = thread & 127, half = thread >> 7;
  const int places = bf16_places(u.info, kind);
  const bool two = places > kBf16Rows;
  // a step's stages are held together
  Place<Smem::kStages> second = at;
  wait(&sm.full[at.slot], at.turn, &sm.abort_flag);
  if (two) {
    second.advance();
    wait(&sm.full[second.slot], second.turn, &sm.abort_flag);
  }
  uint8_t* const stage0 = sm.ring[at.slot];
  uint8_t* const stage1 = sm.ring[second.slot];
  auto row_of = [&](int place) { return (place < kBf16Rows ? stage0 : stage1) + (place & (kBf16Rows - 1)) * kBf16Pitch; };
  bool there = r < places;
  if (kind == kStepDraft) {
    if (r < BDFP4_MAX_SINK) there = r < u.info.sink;
    if (p.rotate || p.key_shift) {  // eight threads bring one draft key into the cache's basis, in place
      const int group = thread & 7;
      const float* shift = p.key_shift ? p.key_shift + u.head * kHeadDim + group * kGroup : nullptr;
#pragma unroll 1
      for (int first = 0; first < u.info.count; first += kCacheThreads / 8) {
        // (threads past the last draft follow along for the exchange; what they make of it goes nowhere)
        const int node = first + (thread >> 3);
        uint4* at16 = reinterpret_cast<uint4*>(row_of(BDFP4_MAX_SINK + min(node, u.info.count - 1)) + group * 32);
        const uint4 raw[2] = {at16[0], at16[1]};
        const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
        __syncwarp();  // a thread that follows along may read the row that another of its warp writes
        cache_basis16_any(v, group, p.rotate != 0, shift);
        if (node < u.info.count) store_bf16x16(reinterpret_cast<__nv_bfloat16*>(at16), v);
      }
      tc::fence_proxy_async_smem();  // the stage is overwritten by copies next
      bar_sync(barrier, kCacheThreads);
    }
  }
  const uint4* row = reinterpret_cast<const uint4*>(row_of(min(r, places - 1)));
  float amax = 0.0f;
  if (there) {
#pragma unroll 4
    for (int j = 0; j < 16; ++j) {
      const uint4 q = row[j];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
    }
  }
  float inverse;
  const float scale = scale_to<14>(amax, &inverse);
#pragma unroll 1
  for (int quarter = 2 * half; quarter < 2 * half + 2; ++quarter) {
    uint32_t v[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (there) q = row[quarter * 4 + j];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[4 * j + i] = h2(__floats2half2_rn(__uint_as_float(w[i] << 16) * scale, __uint_as_float(w[i] & 0xffff0000u) * scale));
    }
    st16(operand + quarter * 16, v);
  }
  release(sm, at, thread, true);
  if (two) release(sm, at, thread, true);
  return inverse;
}

// The values of a BF16 step: half h brings the tokens of the step's stage h into channel r's lane.
template <typename Smem>
__device__ __forceinline__ void bf16_values(Smem& sm, const Unit& u, StepKind kind, Place<Smem::kStages>& at,
                                            uint32_t operand, int thread) {
  const int c = thread & 127, half = thread >> 7;
  const int places = bf16_places(u.info, kind);
  at.advance();  // the keys'
  if (places > kBf16Rows) at.advance();
#pragma unroll 1
  for (int first = 0; first < places; first += kBf16Rows) {
    wait(&sm.full[at.slot], at.turn, &sm.abort_flag);
    if ((first > 0) == (half > 0)) {
      const uint8_t* stage = sm.ring[at.slot] + 2 * c;
      const int slices = (min(places - first, kBf16Rows) + 15) / 16;
#pragma unroll 1
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
    }
    release(sm, at, thread, true);
  }
}

}  // namespace tree
}  // namespace bdfp4
