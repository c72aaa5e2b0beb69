// Attention of a tree of drafted tokens over the paged NVFP4 cache, on the tensor cores.
//
// Per (row, KV head) the queries are one matrix of nodes x ratio rows, cut into tiles of NT. Against 128
// tokens at a time,
//     S^T [token, query]   = K   [token, channel]  * Q^T
//     O^T [channel, query] = V^T [channel, token] * P^T
//
// S^T over a page is the block-scaled FP4 product of the codes as they lie in the cache (kind::mxf4nvf4, no
// dequantization) with the query written as a sum of four FP4 terms, each the rounding of what the ones
// before left: a term leaves at most 0.177 of its group's largest value (half a step of 2/6, the E4M3
// scale's rounding included), four leave 10^-3, less than the BF16 rounding the query came with. Four terms
// of K = 64 take the tensor time of one FP16 product.
//
// O^T over a page is a kind::f16 product with V^T in tensor memory: E2M1 x E4M3 has at most six significant
// bits and lies in [2^-10, 2688], so a page's values are exact in FP16. A thread reads its own channel's 64
// code bytes, converts and scales them in registers and stores them straight into its tensor-memory lane; the
// dequantized tile never passes through shared memory. P is stored as the softmax threads hold it, one token
// per thread with its queries contiguous, which is the MN-major form of operand B.
//
// Softmax thread t owns token t of S^T. Maxima are per query, in shared memory, and lazy: after a unit's first
// block (of two steps) probabilities are formed against them at once, and only when one comes out more than
// 2^8 above its maximum (the barrier that ends a block carries that vote) are the maxima taken anew, O^T
// rescaled and the block formed again. Sums stay per thread until the unit ends. Probabilities carry a factor
// 2^7, so in FP16 they stay below 2^15 and lose nothing above 2^-31 of the largest.
//
// What bounds it: five roles run side by side on every scheduler, and the sum of their code is larger than its
// instruction cache. Code that runs once per unit is kept in rolled loops, and the common path short.
//
// The rolling tail and the drafts with the sink are two more steps over BF16 values, both products kind::f16
// with the cache side in tensor memory: K is scaled per token by a power of two into FP16's range (the softmax
// thread of the token undoes it), V and P are BF16. Queries are scaled per tile the same way.
//
// Work is the sequence of all steps of all (row, head, tile) units, cut into equal runs, one per CTA, so any
// mix of lengths is balanced; a unit that straddles CTAs leaves unnormalised parts that a second kernel adds.
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
// Named barriers: the softmax threads, each stream of them, each half of the values' threads.
constexpr int kSoftmaxBarrier = 1, kStreamBarrier = 2, kValuesBarrier = 4;
constexpr int kTerms = 4;             // FP4 terms of a query
constexpr float kNoMax = -3.0e38f;  // a query that has seen no token yet
constexpr float kShift = 7.0f;      // probabilities carry 2^7
constexpr float kHighest = 32768.0f;  // ... and their queries' maxima are renewed when one exceeds this, 2^8 above

// A unit's blocks of two steps go alternately to two streams, each a softmax of its own (maxima, sums, output)
// in a warpgroup of its own, joined when the unit ends: one stream's block is a chain of latencies (scores out
// of tensor memory, exponentials, stores, fences, a barrier) that the other fills. The values' two warpgroups
// take even and odd steps. Tiles of 64 queries were built too and lost: their sums and scores leave no registers
// for a second stream, and a step cost 2000 cycles against 2 x 600.
template <int NT>
struct Shape {
  static constexpr int kOut = NT / 2;  // queries whose output a warpgroup writes
  static constexpr int kStages = 7;
  static constexpr int kThreads = 256 + 256 + 128;  // values, softmax, control
  // Registers per thread at launch and after the warpgroups have traded them: the sum over the warpgroups
  // must not exceed what the launch was given.
  static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 136, kValueRegs = 72, kControlRegs = 64;
  static_assert(2 * kSoftmaxRegs + 2 * kValueRegs + kControlRegs <= 5 * kLaunchRegs, "registers");
  static_assert(kLaunchRegs * kThreads <= 65536, "registers");
  static constexpr int kRow = NT * 2;  // bytes of a token's probabilities: the swizzle span of P
  static constexpr uint64_t kSwizzle = NT == 32 ? tc::kSwizzle64B : tc::kSwizzle32B;
  // tensor memory columns: scores [stream][set][step], output [stream], values (two steps; a BF16 step's keys
  // before its values), scales of the keys (two steps) and of the query terms
  static constexpr int kS = 0, kO = 8 * NT, kV = 10 * NT, kKs = kV + 128, kQs = kKs + 16;
  static_assert(kQs + 8 * kTerms <= 512, "tensor memory");
};

template <int FROM, int TO>
__device__ __forceinline__ void trade_registers() {
  if constexpr (TO > FROM) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TO));
  if constexpr (TO < FROM) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TO));
}

// A value the compiler may not reason about: in a rolled loop a condition on it is not hoisted out (which would
// make one copy of the loop per outcome).
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+r"(x));
  return x;
}

struct RowInfo {
  int count, pages, residual, sink, slot;  // pages: 128-token steps in the FP4 cache
  int steps;                               // of one unit: pages, tail, drafts with sink
  int tiles;
};

// A run of steps of one (row, head, tile).
struct Unit {
  RowInfo info;
  int row, head, tile, begin, end;  // steps [begin, end) are this CTA's; begin < 0: no more units
};
constexpr int kUnits = 4;  // of the ring through which the key producer hands them to the other roles
constexpr int kUnitReaders = 8 + 8 + 3;  // warps: values, softmax, value producer, score issuer, output issuer

template <int NT>
struct Smem {
  using Sh = Shape<NT>;
  alignas(1024) uint8_t ring[Sh::kStages][kStage];
  alignas(1024) uint8_t q[2][NT * 128];          // FP16: two halves of 64 channels, K-major, 128-byte swizzle
  alignas(1024) uint8_t q_codes[kTerms][NT * 64];  // FP4 terms, K-major, 64-byte swizzle
  alignas(1024) uint8_t q_scales[kTerms][1024];    // two atoms each
  alignas(1024) uint8_t p[2][2][2][128 * Sh::kRow];  // [stream][set][step] MN-major: a row of queries per token, swizzled
  uint64_t family[NT];  // draft nodes each query sees
  // by stream: kShift - maximum; maximum, log2 units; what a renewal scales by; weights of not plain blocks
  float base[2][NT], top[2][NT], factor[2][NT], extra[2][NT];
  float share[2][NT];   // what a stream's output is multiplied by
  float warp_value[2][4][NT];   // a block's maxima, a unit's sums, by warp
  float step_sum[2][2][4][NT];  // [stream][set] a not plain block's weights, by warp
  float key_factor[8][128];  // what undoes the scaling of a BF16 step's keys, by step number
  float q_max[8];
  int parents[BDFP4_MAX_TREE_NODES];
  Unit units[kUnits];
  uint64_t unit_full[kUnits], unit_empty[kUnits];
  uint64_t full_k[Sh::kStages], full_v[Sh::kStages], empty[Sh::kStages];
  uint64_t k_ready[Sh::kStages];  // 64-token pages: the stage's key scales are whole atoms
  uint64_t ka_full[2], ka_empty[2], va_full[2], va_empty[2];  // by step
  uint64_t s_full[2][2][2], s_empty[2][2], p_full[2][2], p_empty[2][2];  // [stream][set], s_full by step too
  uint64_t q_full, o_full, o_empty, drained;
  long long sums[Sh::kThreads / 32];
  int start_row;
  long long start_offset, first, last;
  int per_cta;
  uint32_t tmem;
  int abort_flag, ignored_flag;
};

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

__device__ __forceinline__ void softmax_sync() { bar_sync(kSoftmaxBarrier, 256); }

__device__ __forceinline__ bool bar_any(int id, int threads, bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(out)
      : "r"((uint32_t)pred), "r"(id), "r"(threads)
      : "memory");
  return out != 0;
}
__device__ __forceinline__ bool softmax_any(bool pred) { return bar_any(kSoftmaxBarrier, 256, pred); }

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

// The power of two that brings `amax` into [2^10, 2^11), where FP16 has 25 binades below and the FP4 terms'
// E4M3 scales (up to 448 = 2688 / 6) reach their fourth, and its inverse. Zero, infinite or NaN: 1.
__device__ __forceinline__ float fp16_scale(float amax, float* inverse) {
  const int e = (int)((__float_as_uint(amax) >> 23) & 0xffu);
  if (e == 0 || e == 255) {
    *inverse = 1.0f;
    return 1.0f;
  }
  const int field = min(127 + 10 + 127 - e, 253);
  *inverse = __uint_as_float((uint32_t)(254 - field) << 23);
  return __uint_as_float((uint32_t)field << 23);
}

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

enum StepKind { kStepPage, kStepTail, kStepDraft };

__device__ __forceinline__ StepKind step_kind(const RowInfo& r, int step) {
  return step < r.pages ? kStepPage : (step == r.pages && r.residual > 0) ? kStepTail : kStepDraft;
}
// Token places of a BF16 step: the tail's tokens, or 16 places of the sink and the drafts behind them.
__device__ __forceinline__ int bf16_places(const RowInfo& r, StepKind kind) {
  return kind == kStepTail ? r.residual : BDFP4_MAX_SINK + r.count;
}
// 16-token slices of a step that hold anything.
__device__ __forceinline__ int step_slices(const RowInfo& r, StepKind kind) {
  return kind == kStepPage ? 8 : (bf16_places(r, kind) + 15) / 16;
}

// The units of this CTA in order. Steps are counted in 32 bits within a row (the host refuses larger rows).
struct Walker {
  const TreeParams& p;
  int row, page_tokens, offset, left;
  __device__ Walker(const TreeParams& params, int start_row, int start_offset, int steps, int pt)
      : p(params), row(start_row), page_tokens(pt), offset(start_offset), left(steps) {}
  // `known`: u is a unit of this walk, so its row's lengths need not be read again.
  __device__ __forceinline__ bool next(Unit& u, bool known) {
    if (left <= 0) return false;
#pragma unroll 1
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

// ---- roles -----------------------------------------------------------------------------------------

// The roles' loops run side by side on every scheduler and share its instruction cache, so waiting is a dozen
// instructions, one when the phase is already over. After about two seconds, or once another thread has given
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

// One thread of a converged warp. tcgen05.mma and the bulk copies take their operands from uniform registers:
// behind an elected predicate the warp's control flow stays uniform for the compiler, and an MMA issues in 32
// (N = 64) to 64 cycles (N = 128), its tensor time; behind a test of the lane number it took 140 whatever its
// size, and the copies of a step were longer than its HBM time.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(elected));
  return elected != 0;
}

// A role's view of the ring of units.
template <int NT>
struct Units {
  Smem<NT>& sm;
  int next_unit;
  __device__ explicit Units(Smem<NT>& s) : sm(s), next_unit(0) {}
  // The whole warp: the next unit into `u`; false when there is none, or when a wait has been given up (then `u`
  // may hold anything). Roles whose warps meet at barriers have to agree on the answer.
  __device__ __forceinline__ bool next(Unit& u) {
    const int at = next_unit % kUnits;
    wait(&sm.unit_full[at], (next_unit / kUnits) & 1, &sm.abort_flag);
    u = sm.units[at];
    ++next_unit;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&sm.unit_empty[at]);
    return __all_sync(0xffffffffu, u.begin >= 0 && *static_cast<volatile int*>(&sm.abort_flag) == 0);
  }
};

// One side's copies: SIDE 0 brings a page's key codes and scales, SIDE 1 its values' and the rows of the BF16
// steps. Two warps, because a copy keeps its issuer for 80 cycles and a step of 64-token pages has eight.
template <int NT, int PT, int SIDE>
__device__ __forceinline__ void produce(const TreeParams& p, Smem<NT>& sm, const CUtensorMap* map, int lane) {
  using Sh = Shape<NT>;
  constexpr int kEntries = kPage / PT;
  const int64_t tail_row = (int64_t)p.heads_kv * kHeadDim;
  const int64_t codes_pitch = p.codes_pitch[SIDE], scales_pitch = p.scales_pitch[SIDE];
  uint64_t* full = SIDE ? sm.full_v : sm.full_k;
  int slot = 0, issued = 0;
  uint32_t turn = 0;
  auto advance = [&] {
    ++issued;
    if (++slot == Sh::kStages) slot = 0, turn ^= 1;
  };
  // the key producer walks the units and publishes each before the one in front of it is produced
  Units<NT> units(sm);
  Walker walker(p, sm.start_row, (int)sm.start_offset, (int)(sm.last - sm.first), PT);
  Unit u, following;
  bool known = false, more = true;
  int published = 0;
  auto publish = [&] {
    more = more && walker.next(following, known);
    known = true;
    wait(&sm.unit_empty[published % kUnits], ((published / kUnits) & 1) ^ 1, &sm.abort_flag);
    if (lane == 0) {
      if (!more) following.begin = -1;
      sm.units[published % kUnits] = following;
      tc::mbar_arrive(&sm.unit_full[published % kUnits]);
    }
    __syncwarp();
    ++published;
  };
  if (SIDE == 0) publish();
#pragma unroll 1
  while (true) {
    if (SIDE == 0) {
      if (!more) break;
      u = following;
      publish();
    } else if (!units.next(u)) {
      break;
    }
    const int32_t* table = p.table + u.row * p.table_stride;
    const uint8_t* codes = p.codes[SIDE] + u.head * (PT == 128 ? 8192 : 4096);
    const uint8_t* scales = p.scales[SIDE] + u.head * (PT == 128 ? 1024 : 512);
    if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&sm.abort_flag) != 0)) break;
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
        wait(&sm.empty[slot], turn ^ 1, &sm.abort_flag);
        if (elect_one()) {
          uint8_t* stage = sm.ring[slot];
          tc::mbar_expect_tx(&full[slot], 9216);
          if constexpr (PT == 128) {
            if constexpr (SIDE == 0) tc::tma_load_4d(stage, map, &full[slot], 0, u.head, 0, page[0]);
            else tc::tma_load_3d(stage + kVOffset, map, &full[slot], 0, u.head * kHeadDim, page[0]);
            tc::bulk_load(stage + (SIDE ? kVsOffset : kKsOffset), scales + page[0] * scales_pitch, 1024, &full[slot]);
          } else {
#pragma unroll
            for (int e = 0; e < kEntries; ++e) {
              tc::bulk_load(stage + (SIDE ? kVOffset : 0) + e * 4096, codes + page[e] * codes_pitch, 4096, &full[slot]);
              tc::bulk_load(stage + (SIDE ? kVsOffset : kKsOffset) + e * 512, scales + page[e] * scales_pitch, 512, &full[slot]);
            }
          }
        }
        __syncwarp();
        advance();
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
          wait(&sm.empty[slot], turn ^ 1, &sm.abort_flag);
          if (SIDE == 0) {
            if (lane == 0) tc::mbar_arrive(&full[slot]);  // nothing for the FP4 product here
          } else {
            const int end = min(first + kBf16Rows, places);
            // the sink's places behind its length stay empty
            const int absent = kind == kStepDraft && first == 0 ? BDFP4_MAX_SINK - u.info.sink : 0;
            if (lane == 0) tc::mbar_expect_tx(&full[slot], (end - first - absent) * 256);
            __syncwarp();
#pragma unroll 1
            for (int i = first + lane; i < end; i += 32) {
              const __nv_bfloat16* source = nullptr;
              if (kind == kStepTail) source = tail + i * tail_row;
              else if (i >= BDFP4_MAX_SINK) source = draft + (i - BDFP4_MAX_SINK) * draft_node;
              else if (i < u.info.sink) source = tail + (kPage + i) * tail_row;
              if (source) tc::bulk_load(sm.ring[slot] + (i - first) * kBf16Pitch, source, 256, &full[slot]);
            }
          }
          __syncwarp();
          advance();
        }
      }
    }
  }
  // After an abort nobody else waits for the copies still in flight: no CTA may end under them.
  if (lane == 0 && *static_cast<volatile int*>(&sm.abort_flag)) {
#pragma unroll 1
    for (int back = min(issued, Sh::kStages); back > 0; --back) {
      const int at = issued - back;
      wait(&full[at % Sh::kStages], (at / Sh::kStages) & 1, &sm.ignored_flag);
    }
  }
  __syncwarp();
}

// The products are issued by two warps, one for the scores and one for the output: an MMA keeps its issuer
// for 40 to 60 cycles, and the sixteen of a step one after another were longer than the step's HBM time. The
// whole warp walks and waits; one thread of it issues.
template <int NT, int PT>
__device__ __forceinline__ void issue_scores(Smem<NT>& sm) {
  using Sh = Shape<NT>;
  constexpr uint32_t kFp4 = tc::nvf4_idesc(128, NT), kF16 = f16_idesc(NT, 0, false);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const uint32_t q = tc::smem_u32(sm.q), ring = tc::smem_u32(sm.ring);
  const uint64_t q_codes = tc::fp4_tile_desc(tc::smem_u32(sm.q_codes), 0);
  const uint64_t q_scales = tc::sf_atom_desc(tc::smem_u32(sm.q_scales));
  int n = 0, block = 0, unit = 0, slot = 0;
  uint32_t turn = 0, bf16_turn = 0;  // bf16_turn: one bit per half of the values' threads
  Units<NT> units(sm);
  Unit u;
#pragma unroll 1
  while (units.next(u)) {
    wait(&sm.q_full, unit & 1, &sm.abort_flag);
    tc::fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int i = 0; i < 2 * kTerms; ++i) tc::cp_sf_atom(tmem + Sh::kQs + i * 4, q_scales + i * 32);
    }
    __syncwarp();
#pragma unroll 1
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      const int within = (step - u.begin) & 1, stream = block & 1, set = (block >> 1) & 1;
      const uint32_t scores = tmem + Sh::kS + (4 * stream + 2 * set + within) * NT;
      uint64_t* full = &sm.s_full[stream][set][within];
      if (within == 0) wait(&sm.s_empty[stream][set], ((block >> 2) & 1) ^ 1, &sm.abort_flag);
      if (kind == kStepPage) {
        wait(PT == 64 ? &sm.k_ready[slot] : &sm.full_k[slot], turn, &sm.abort_flag);
        tc::fence_after_sync();
        const uint32_t stage = ring + slot * kStage;
        const uint64_t codes = tc::fp4_tile_desc(stage, 0), atoms = tc::sf_atom_desc(stage + kKsOffset);
        const uint32_t scales = tmem + Sh::kKs + (n & 1) * 8;
        if (elect_one()) {
          tc::cp_sf_atom(scales, atoms);
          tc::cp_sf_atom(scales + 4, atoms + 32);
#pragma unroll 1
          for (int s = 0; s < 2; ++s) {  // 64 channels further: 32 bytes of codes, one atom of scales
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
              tc::mma_nvf4(scores, codes + 2 * s, q_codes + term * NT * 4 + 2 * s, kFp4, scales + 4 * s,
                           tmem + Sh::kQs + term * 8 + 4 * s, s + term > 0);
          }
          tc::commit(full);
          tc::commit(&sm.empty[slot]);
        }
        __syncwarp();
        if (++slot == Sh::kStages) slot = 0, turn ^= 1;
      } else {
#pragma unroll 1
        for (int i = 2 * ((bf16_places(u.info, kind) + kBf16Rows - 1) / kBf16Rows); i > 0; --i) {
          wait(&sm.full_k[slot], turn, &sm.abort_flag);  // the stage is not this product's
          if (elect_one()) tc::mbar_arrive(&sm.empty[slot]);
          __syncwarp();
          if (++slot == Sh::kStages) slot = 0, turn ^= 1;
        }
        wait(&sm.ka_full[n & 1], (bf16_turn >> (n & 1)) & 1, &sm.abort_flag);
        bf16_turn ^= 1u << (n & 1);
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 8; ++s)
            mma_ts(scores, tmem + Sh::kV + (n & 1) * 64 + s * 8, tc::bf16_tile_desc(q + (s >> 2) * NT * 128, s & 3), kF16, s > 0);
          tc::commit(full);
          tc::commit(&sm.ka_empty[n & 1]);
        }
        __syncwarp();
      }
      if (within == 1 || step + 1 == u.end) {
        if (within == 0 && elect_one()) tc::mbar_arrive(&sm.s_full[stream][set][1]);  // a block of one step
        __syncwarp();
        ++block;
      }
    }
    ++unit;
  }
  // also after an abort: tensor memory is freed behind the last product
  if (elect_one()) tc::commit(&sm.drained);
  __syncwarp();
  wait(&sm.drained, 0, &sm.ignored_flag);
}

template <int NT>
__device__ __forceinline__ void issue_output(Smem<NT>& sm) {
  using Sh = Shape<NT>;
  constexpr uint32_t kPages = f16_idesc(NT, 0, true), kBf16 = f16_idesc(NT, 1, true);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  // eight tokens' rows are one swizzle atom, a tile is one atom wide
  const uint64_t prob = tc::smem_desc(tc::smem_u32(sm.p), Sh::kSwizzle, 8 * Sh::kRow, 8 * Sh::kRow);
  int n = 0, block = 0, unit = 0;
  Units<NT> units(sm);
  Unit u;
#pragma unroll 1
  while (units.next(u)) {
    wait(&sm.o_empty, (unit & 1) ^ 1, &sm.abort_flag);
#pragma unroll 1
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      const int within = (step - u.begin) & 1, stream = block & 1, set = (block >> 1) & 1;
      wait(&sm.va_full[n & 1], (n >> 1) & 1, &sm.abort_flag);
      if (within == 0) wait(&sm.p_full[stream][set], (block >> 2) & 1, &sm.abort_flag);
      tc::fence_after_sync();
      const bool first = within == 0 && step - u.begin < 4;  // of its stream in this unit
      const bool closes = within == 1 || step + 1 == u.end;
      const uint64_t tile = prob + (4 * stream + 2 * set + within) * (128 * Sh::kRow / 16);
      const uint32_t operand = tmem + Sh::kV + (n & 1) * 64, output = tmem + Sh::kO + stream * NT;
      if (elect_one()) {
        const uint32_t idesc = kind == kStepPage ? kPages : kBf16;
        const int slices = step_slices(u.info, kind);
#pragma unroll 1
        for (int s = 0; s < slices; ++s)  // 16 tokens further: 16 rows of P, 8 columns of V
          mma_ts(output, operand + s * 8, tile + s * Sh::kRow, idesc, !(first && s == 0));
        tc::commit(&sm.va_empty[n & 1]);
        if (closes) tc::commit(&sm.p_empty[stream][set]);
        if (step + 1 == u.end) tc::commit(&sm.o_full);
      }
      __syncwarp();
      if (closes) ++block;
    }
    ++unit;
  }
  if (elect_one()) tc::commit(&sm.drained);
  __syncwarp();
  wait(&sm.drained, 0, &sm.ignored_flag);
}

// 64-token pages: the key scales of a step's two pages come as half atoms (32 rows of 8 bytes); one warp
// interleaves them, in place, into the two whole atoms the MMA reads.
__device__ __forceinline__ void interleave_scales(uint8_t* scales, int lane) {
  uint2 part[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) part[i & 1][i >> 1] = *reinterpret_cast<const uint2*>(scales + (i >> 1) * 512 + (i & 1) * 256 + lane * 8);
  __syncwarp();
#pragma unroll
  for (int atom = 0; atom < 2; ++atom)
    *reinterpret_cast<uint4*>(scales + atom * 512 + lane * 16) = make_uint4(part[atom][0].x, part[atom][0].y, part[atom][1].x, part[atom][1].y);
  tc::fence_proxy_async_smem();
  __syncwarp();
}

// Thirty-two codes and the scales of their two groups into sixteen columns of this thread's lane. The caller's
// loop over a channel's four chunks stays rolled: three roles run side by side on every scheduler, and with
// the 300 instructions of the unrolled form the warps waited for instructions a third of the time.
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

// The values' warps: thread c of a half holds channel c of its steps' V^T, and token c of a BF16 step's K.
template <int NT, int PT>
__device__ __forceinline__ void values(const TreeParams& p, Smem<NT>& sm, int thread) {
  const int c = thread & 127, lane = c & 31, half = thread >> 7;
  using Sh = Shape<NT>;
  const uint32_t lanes = (uint32_t)(c & ~31) << 16;
  int slot = 0, n = 0;
  uint32_t turn = 0, bf16_turn = 0;
  auto pass = [&](int stages) {  // the other half's
    slot += stages;
    if (slot >= Sh::kStages) slot -= Sh::kStages, turn ^= 1;
  };
  auto arrived = [&]() -> uint8_t* {
    wait(&sm.full_v[slot], turn, &sm.abort_flag);
    return sm.ring[slot];
  };
  const bool interleaves = PT == 64 && (c >> 5) == 3;
  auto release = [&] {
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sm.empty[slot]);
    pass(1);
  };
  Units<NT> units(sm);
  Unit u;
#pragma unroll 1
  while (!bar_any(kValuesBarrier + half, 128, !units.next(u))) {
#pragma unroll 1
    for (int step = u.begin; step < u.end; ++step, ++n) {
      const StepKind kind = step_kind(u.info, step);
      if ((n & 1) != half) {
        pass(kind == kStepPage ? 1 : 2 * ((bf16_places(u.info, kind) + kBf16Rows - 1) / kBf16Rows));
        continue;
      }
      const uint32_t operand = sm.tmem + Sh::kV + (n & 1) * 64 + lanes;
      uint64_t* operand_empty = &sm.va_empty[n & 1];
      const uint32_t empty_parity = ((n >> 1) & 1) ^ 1;
      if (kind == kStepPage) {
        if (interleaves) {
          wait(&sm.full_k[slot], turn, &sm.abort_flag);
          interleave_scales(sm.ring[slot] + kKsOffset, lane);
          if (lane == 0) tc::mbar_arrive(&sm.k_ready[slot]);
        }
        const uint8_t* stage = arrived();
        const uint8_t* scales = stage + kVsOffset + (c & 31) * 16 + (c >> 5) * 4;
        wait(operand_empty, empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          const uint8_t* at = PT == 128 ? stage + kVOffset + c * 64 + ((j ^ ((c >> 1) & 3)) * 16)
                                        : stage + kVOffset + (j >> 1) * 4096 + c * 32 + (((j & 1) ^ ((c >> 2) & 1)) * 16);
          store_dequantized(operand + 16 * j, *reinterpret_cast<const uint4*>(at),
                            *reinterpret_cast<const uint16_t*>(scales + (j >> 1) * 512 + (j & 1) * 2));
        }
        release();
      } else {
        const int places = bf16_places(u.info, kind);
        const int stages = (places + kBf16Rows - 1) / kBf16Rows;
        // keys first, through the buffer that takes the values after the score product
        wait(operand_empty, empty_parity, &sm.abort_flag);
        tc::fence_after_sync();
        {  // a step's stages are held together
          uint8_t* const stage0 = arrived();
          uint8_t* stage1 = stage0;
          if (stages > 1) {
            const bool wraps = slot + 1 == Sh::kStages;
            const int next = wraps ? 0 : slot + 1;
            wait(&sm.full_v[next], turn ^ (wraps ? 1u : 0u), &sm.abort_flag);
            stage1 = sm.ring[next];
          }
          auto row_of = [&](int place) { return (place < kBf16Rows ? stage0 : stage1) + (place & (kBf16Rows - 1)) * kBf16Pitch; };
          bool there = c < places;
          if (kind == kStepDraft) {
            if (c < BDFP4_MAX_SINK) there = c < u.info.sink;
            if (p.rotate || p.key_shift) {  // eight threads bring one draft key into the cache's basis, in place
              const int group = c & 7;
              const float* shift = p.key_shift ? p.key_shift + u.head * kHeadDim + group * kGroup : nullptr;
#pragma unroll 1
              for (int first = 0; first < u.info.count; first += 16) {
                // (threads past the last draft follow along for the exchange; what they make of it goes nowhere)
                const int node = min(first + (c >> 3), u.info.count - 1);
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
                if (first + (c >> 3) < u.info.count) store_bf16x16(reinterpret_cast<__nv_bfloat16*>(at), v);
              }
              tc::fence_proxy_async_smem();  // the stage is overwritten by copies next
              bar_sync(kValuesBarrier + half, 128);
            }
          }
          const uint4* row = reinterpret_cast<const uint4*>(row_of(min(c, places - 1)));
          float amax = 0.0f;
          if (there) {
#pragma unroll 2
            for (int j = 0; j < 16; ++j) {
              const uint4 r = row[j];
              const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
            }
          }
          float inverse;
          const float scale = fp16_scale(amax, &inverse);
          sm.key_factor[n & 7][c] = inverse;
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
#pragma unroll 1
          for (int i = 0; i < stages; ++i) {
            if (interleaves && lane == 0) tc::mbar_arrive(&sm.k_ready[slot]);  // its phases follow the stage's uses
            release();
          }
          tc::tmem_wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sm.ka_full[half]);
          wait(&sm.ka_empty[half], bf16_turn, &sm.abort_flag);
          tc::fence_after_sync();
          bf16_turn ^= 1;
        }
#pragma unroll 1
        for (int first = 0; first < places; first += kBf16Rows) {
          const uint8_t* stage = arrived() + 2 * c;
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
          if (interleaves && lane == 0) tc::mbar_arrive(&sm.k_ready[slot]);
          release();
        }
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.va_full[n & 1]);
    }
  }
}

// The tile's queries into shared memory: rotated if asked, scaled by one power of two, as FP16 for the BF16 steps
// and as FP4 terms for the pages. One scale for the tile: a query whose largest value is 2^-8 of the tile's
// still has all four terms above E4M3's smallest scale. Returns what undoes the scaling.
template <int NT>
__device__ __forceinline__ float load_queries(const TreeParams& p, Smem<NT>& sm, const Unit& u, int thread) {
  const int group = thread & 7;  // eight threads hold one query
  const int queries = u.info.count * p.ratio;
  if (thread < BDFP4_MAX_TREE_NODES) sm.parents[thread] = thread < u.info.count ? p.parents[u.row * p.parents_row + thread] : -1;
  float scale = 1.0f, inverse = 1.0f;
#pragma unroll 1
  for (int phase = 0; phase < 2; ++phase) {  // the tile's largest value, then the operands
    float amax = 0.0f;
#pragma unroll 1
    for (int r = thread >> 3; r < (NT < 32 ? 32 : NT); r += 32) {
      const int query = u.tile * NT + r;
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = 0.0f;
      if (query < queries && r < NT)
        load_bf16x16(p.query + u.row * p.query_row + (query / p.ratio) * p.query_node +
                         (int64_t)(u.head * p.ratio + query % p.ratio) * kHeadDim + group * kGroup, v);
      if (opaque(p.rotate)) {
        hadamard_butterflies(v, group);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] *= kInvSqrt128;
      }
      if (opaque(phase) == 0) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (fabsf(v[j]) < INFINITY) amax = fmaxf(amax, fabsf(v[j]));
      } else if (r < NT) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] *= scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = h2(__floats2half2_rn(v[2 * j], v[2 * j + 1]));
        uint8_t* row = sm.q[group >> 2] + r * 128;
        const int chunk = (group & 3) * 2;
        *reinterpret_cast<uint4*>(row + ((chunk ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ (r & 7)) * 16)) = make_uint4(w[4], w[5], w[6], w[7]);
        const int at = r * 64 + group * 8;
#pragma unroll 1
        for (int term = 0; term < kTerms; ++term) {
          float largest = 0.0f;
#pragma unroll
          for (int j = 0; j < 16; ++j) largest = fmaxf(largest, fabsf(v[j]));
          const uint32_t byte = cvt_e4m3(largest * (1.0f / 6.0f));
          GroupCodes codes;
          codes.scale = e4m3_to_float(byte);
          // (an approximate reciprocal: what it rounds otherwise is left to the next term)
          float inverse_scale;
          asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse_scale) : "f"(fmaxf(codes.scale, 1.0e-30f)));
          float scaled[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) scaled[j] = v[j] * inverse_scale;
          codes.lo = pack_e2m1x8(scaled);
          codes.hi = pack_e2m1x8(scaled + 8);
          *reinterpret_cast<uint2*>(sm.q_codes[term] + (at ^ (((at >> 7) & 3) << 4))) = make_uint2(codes.lo, codes.hi);
          sm.q_scales[term][scale_tile_offset(r, group)] = (uint8_t)byte;
          float rest[16];
          group_residual16(v, codes, rest);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = rest[j];
        }
      }
    }
    if (phase == 0) {
      amax = warp_max(amax);
      if ((thread & 31) == 0) sm.q_max[thread >> 5] = amax;
      softmax_sync();
#pragma unroll
      for (int w = 0; w < 8; ++w) amax = fmaxf(amax, sm.q_max[w]);
      scale = fp16_scale(amax, &inverse);
    }
  }
  tc::fence_proxy_async_smem();
  softmax_sync();
  if (thread == 0) tc::mbar_arrive(&sm.q_full);
  return inverse;
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

template <int NT>
__device__ __forceinline__ void softmax(const TreeParams& p, Smem<NT>& sm, int thread) {
  using Sh = Shape<NT>;
  const int t = thread & 127, lane = thread & 31, warp = t >> 5, stream = thread >> 7;
  const uint32_t lanes = (uint32_t)(t & ~31) << 16;
  const float* base = sm.base[stream];
  const int barrier = kStreamBarrier + stream;
  const uint32_t output = sm.tmem + Sh::kO + stream * NT + lanes;
  int blocks = 0, unit = 0;  // of the CTA so far
  int n = 0;
  float q_inverse = 1.0f;
  float2 sum[NT / 2];
  Units<NT> units(sm);
  Unit u, following;
  bool running = false;
#pragma unroll 1
  while (true) {
    // the next unit's queries go in while this one's last products run: all its scores are done
    const bool more = !softmax_any(!units.next(following));
    float next_inverse = 1.0f;
    if (running) {  // each query's weight in this stream, by warp
      float v[NT];
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) v[2 * j] = sum[j].x, v[2 * j + 1] = sum[j].y;
      reduce_columns<NT, 16>(v, lane, 0, [&](int j, float total) { sm.warp_value[stream][warp][j] = total; });
    }
    if (more) next_inverse = load_queries<NT>(p, sm, following, thread);
    if (running) {
      softmax_sync();
      const bool whole = u.begin == 0 && u.end == u.info.steps, both = u.end - u.begin > 2;
      // a part that begins a unit goes to the CTA's second slot, one that continues it to the first
      const int part = 2 * blockIdx.x + (u.begin == 0 ? 1 : 0);
      if (thread < NT) {  // join the streams
        float total[2], top = fmaxf(sm.top[0][thread], sm.top[1][thread]), sum_of_both = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          total[h] = sm.extra[h][thread];
#pragma unroll
          for (int w = 0; w < 4; ++w) total[h] += sm.warp_value[h][w][thread];
          sm.share[h][thread] = ex2(sm.top[h][thread] - top);
          sum_of_both += total[h] * sm.share[h][thread];
        }
        if (whole) {
          const float scale = sum_of_both > 0.0f ? p.value_scale / sum_of_both : 0.0f;
          sm.share[0][thread] *= scale;
          sm.share[1][thread] *= scale;
        } else {
          p.partial_stat[(int64_t)(2 * part) * NT + thread] = top;
          p.partial_stat[(int64_t)(2 * part + 1) * NT + thread] = sum_of_both;
        }
      }
      softmax_sync();
      wait(&sm.o_full, unit & 1, &sm.abort_flag);
      tc::fence_after_sync();
      const int out_first = stream * Sh::kOut;
      const int queries = min(u.info.count * p.ratio - u.tile * NT - out_first, Sh::kOut);
      const int query = u.tile * NT + out_first;
      int out_node = query / p.ratio, out_head = query % p.ratio;
      __nv_bfloat16* out = p.out + u.row * p.out_row + (int64_t)u.head * p.ratio * kHeadDim + t;
      float* partial = p.partial + ((int64_t)part * NT + out_first) * kHeadDim + t;
      const uint32_t first_output = sm.tmem + Sh::kO + ((blocks - (u.end - u.begin + 1) / 2) & 1) * NT + out_first + lanes;
      const uint32_t second_output = sm.tmem + Sh::kO + ((blocks - (u.end - u.begin + 1) / 2 + 1) & 1) * NT + out_first + lanes;
      const float* first_share = sm.share[(blocks - (u.end - u.begin + 1) / 2) & 1] + out_first;
      const float* second_share = sm.share[(blocks - (u.end - u.begin + 1) / 2 + 1) & 1] + out_first;
#pragma unroll 1
      for (int j = 0; j < queries; j += 8) {
        float o[8], o2[8];
        tc::tmem_ld8(first_output + j, o);
        tc::tmem_ld8(second_output + j, o2);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i] *= first_share[j + i];
          if (both) o[i] = fmaf(o2[i], second_share[j + i], o[i]);  // (a stream without blocks holds anything)
          if (j + i < queries) {
            if (whole) out[out_node * p.out_node + out_head * kHeadDim] = __float2bfloat16_rn(o[i]);
            else partial[(j + i) * kHeadDim] = o[i];
          }
          if (++out_head == p.ratio) out_head = 0, ++out_node;
        }
      }
      tc::fence_before_sync();
      softmax_sync();  // the output has been read; what is kept per query is written anew
      if (thread == 0) {
        tc::mbar_arrive(&sm.o_empty);
        if (!whole && u.begin == 0) {
          TreeSplit split;
          split.row = u.row;
          split.head = u.head;
          split.tile = u.tile;
          // this CTA's run ends inside the unit; the runs behind it are as long
          split.last = blockIdx.x + (u.info.steps - u.end + sm.per_cta - 1) / sm.per_cta;
          p.splits[blockIdx.x] = split;
        }
      }
      ++unit;
    }
    if (!more) break;
    running = true;
    u = following;
    q_inverse = next_inverse;

    if (t < NT) {
      sm.top[stream][t] = kNoMax;
      sm.extra[stream][t] = 0.0f;
      if (stream == 0) {  // the draft nodes that this query sees
        uint64_t seen = 0;
#pragma unroll 1
        for (int node = min((u.tile * NT + t) / p.ratio, u.info.count - 1); node >= 0;) {
          seen |= 1ull << node;
          const int parent = sm.parents[node];
          node = parent < node ? parent : -1;
        }
        sm.family[t] = seen;
      }
    }
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) sum[j] = make_float2(0.0f, 0.0f);
    softmax_sync();
    const float page_factor = p.scale_log2 * q_inverse * p.key_scale;
    const int all_blocks = (u.end - u.begin + 1) / 2;
#pragma unroll 1
    for (int k = (stream ^ blocks) & 1; k < all_blocks; k += 2) {
      const int block = blocks + k, block_begin = u.begin + 2 * k;
      const int steps = min(2, u.end - block_begin), set = (block >> 1) & 1;
      const uint32_t parity = (block >> 2) & 1;
      // a block in which every query sees every token, and all of it FP4
      const bool plain = block_begin + steps <= u.info.pages && (block_begin > 0 || u.info.sink == 0);
      const uint32_t scores0 = sm.tmem + Sh::kS + (4 * stream + 2 * set) * NT + lanes;
      auto scores_ready = [&](int i) {
        wait(&sm.s_full[stream][set][i], parity, &sm.abort_flag);
        tc::fence_after_sync();
      };
      // Where 16 bytes of P go: chunk index XORed as the swizzle does.
      uint8_t* const p_rows = sm.p[stream][set][0] + t * Sh::kRow;
      auto p_chunk = [&](int i, int chunk) {
        return reinterpret_cast<uint4*>(p_rows + i * (128 * Sh::kRow) + ((chunk ^ (NT == 32 ? (t >> 1) & 3 : (t >> 2) & 1)) * 16));
      };
      // Any step: scores in log2 units above the maxima (plus kShift) are f * score + base; a token may be seen by
      // no query or, a draft, by some.
      struct Step {
        StepKind kind;
        int node;             // of this thread's token, if a draft
        uint32_t all, alive;  // 1: every query sees the token; 1: some may
        float f;
      };
      auto open = [&](int i) {
        Step k;
        k.kind = step_kind(u.info, block_begin + i);
        bool dead;
        if (k.kind == kStepPage) dead = block_begin + i == 0 && t < u.info.sink;
        else if (k.kind == kStepTail) dead = t >= u.info.residual || (u.info.pages == 0 && t < u.info.sink);
        else dead = t < BDFP4_MAX_SINK ? t >= u.info.sink : t - BDFP4_MAX_SINK >= u.info.count;
        const bool draft = k.kind == kStepDraft && t >= BDFP4_MAX_SINK && !dead;
        k.node = draft ? t - BDFP4_MAX_SINK : 0;
        k.all = draft ? 0 : 1;
        k.alive = dead ? 0 : 1;
        k.f = k.kind == kStepPage ? page_factor : p.scale_log2 * q_inverse * sm.key_factor[(n + 2 * (block - blocks) + i) & 7][t];
        return k;
      };
      auto load8 = [&](const Step& k, int i, int j, float* v) {
        tc::tmem_ld8(scores0 + i * NT + j, v);
        tc::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint32_t seen = (uint32_t)(sm.family[j + c] >> k.node) | k.all;
          if (!(seen & k.alive)) v[c] = -INFINITY;
        }
      };
      float s[NT];  // a plain block's probabilities, both steps' added
      bool high, fresh = k < 2;
      // P of this block goes where the stream's one before the last was
      wait(&sm.p_empty[stream][set], parity ^ 1, &sm.abort_flag);
#pragma unroll 1
      while (true) {
        if (fresh) {  // take the maxima anew; what was summed so far is brought down to them
          float mine = -INFINITY;
#pragma unroll 1
          for (int i = 0; i < steps; ++i) {
            scores_ready(i);
            const Step k = open(i);
#pragma unroll 1
            for (int j = 0; j < NT; j += 8) {
              float v[8];
              load8(k, i, j, v);
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const float m = warp_max(v[c] * k.f);
                if (lane == j + c) mine = fmaxf(mine, m);
              }
            }
          }
          if (lane < NT) sm.warp_value[stream][warp][lane] = mine;
          bar_sync(barrier, 128);
          if (t < NT) {
            const float before = sm.top[stream][t];
            float now = before;
#pragma unroll
            for (int w = 0; w < 4; ++w) now = fmaxf(now, sm.warp_value[stream][w][t]);
            const float factor = ex2(before - now);
            sm.top[stream][t] = now;
            sm.base[stream][t] = kShift - now;
            sm.factor[stream][t] = factor;
            sm.extra[stream][t] *= factor;
          }
          bar_sync(barrier, 128);
          if (k >= 2) {
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
              sum[j].x *= sm.factor[stream][2 * j];
              sum[j].y *= sm.factor[stream][2 * j + 1];
            }
            const int last = block - 2;  // the stream's
            wait(&sm.p_empty[stream][(last >> 1) & 1], (last >> 2) & 1, &sm.abort_flag);
            tc::fence_after_sync();
#pragma unroll 1
            for (int j = 0; j < NT; j += 8) {
              float o[8];
              uint32_t r[8];
              tc::tmem_ld8(output + j, o);
              tc::tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(o[i] * sm.factor[stream][j + i]);
              st8(output + j, r);
            }
            tc::tmem_wait_st();
          }
        }
        high = false;
        if (plain) {
#pragma unroll
          for (int j = 0; j < NT; ++j) s[j] = 0.0f;
          const float2 f2 = make_float2(page_factor, page_factor);
          __half2 most = __floats2half2_rn(0.0f, 0.0f);
#pragma unroll 1
          for (int i = 0; i < steps; ++i) {
            scores_ready(i);
            float x[NT];
#pragma unroll
            for (int j = 0; j < NT; j += 16) tc::tmem_ld16(scores0 + i * NT + j, x + j);
            tc::tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < NT; j += 8) {
              uint32_t w[4];
#pragma unroll
              for (int c = j; c < j + 8; c += 4) {
                const float4 b = *reinterpret_cast<const float4*>(base + c);
                const float2 y0 = __ffma2_rn(make_float2(x[c], x[c + 1]), f2, make_float2(b.x, b.y));
                const float2 y1 = __ffma2_rn(make_float2(x[c + 2], x[c + 3]), f2, make_float2(b.z, b.w));
                x[c] = ex2(y0.x), x[c + 1] = ex2(y0.y), x[c + 2] = ex2(y1.x), x[c + 3] = ex2(y1.y);
              }
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const __half2 pair = __floats2half2_rn(x[j + 2 * c], x[j + 2 * c + 1]);
                most = __hmax2(most, pair);
                w[c] = h2(pair);
              }
              *p_chunk(i, j >> 3) = make_uint4(w[0], w[1], w[2], w[3]);
            }
#pragma unroll
            for (int c = 0; c < NT; c += 2) {
              const float2 two = __fadd2_rn(make_float2(s[c], s[c + 1]), make_float2(x[c], x[c + 1]));
              s[c] = two.x, s[c + 1] = two.y;
            }
          }
          high = __half2float(__hmax(__low2half(most), __high2half(most))) > kHighest;
        } else {
          float* const sums = sm.step_sum[stream][set][warp];
#pragma unroll 1
          for (int i = 0; i < steps; ++i) {
            scores_ready(i);
            const Step k = open(i);
#pragma unroll 1
            for (int j = 0; j < NT; j += 8) {
              float v[8];
              load8(k, i, j, v);
              const bool page = opaque(k.kind) == kStepPage;
              uint32_t w[4];
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                v[c] = ex2(fmaf(v[c], k.f, base[j + c]));
                high |= v[c] > kHighest;
              }
#pragma unroll
              for (int c = 0; c < 4; ++c)
                w[c] = page ? h2(__floats2half2_rn(v[2 * c], v[2 * c + 1]))
                            : pack_bf16x2(v[2 * c] * p.inverse_value_scale, v[2 * c + 1] * p.inverse_value_scale);
              *p_chunk(i, j >> 3) = make_uint4(w[0], w[1], w[2], w[3]);
              // four lanes end up with each column's sum
              reduce_columns<8, 16>(v, lane, j, [&](int column, float total) {
                if ((lane & 3) == 0) sums[column] = opaque(i) > 0 ? sums[column] + total : total;
              });
            }
          }
        }
        tc::fence_before_sync();
        tc::fence_proxy_async_smem();
        // against maxima just taken nothing is high: the vote then only ends the block
        if (!bar_any(barrier, 128, high) || fresh) break;
        fresh = true;
      }
      // the barrier stands behind every thread's scores read and probabilities written
      if (t == 0) {
        tc::mbar_arrive(&sm.p_full[stream][set]);
        tc::mbar_arrive(&sm.s_empty[stream][set]);
      }
      if (plain) {
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) sum[j] = __fadd2_rn(sum[j], make_float2(s[2 * j], s[2 * j + 1]));
      } else if (t < NT) {
        float total = sm.extra[stream][t];
#pragma unroll
        for (int w = 0; w < 4; ++w) total += sm.step_sum[stream][set][w][t];
        sm.extra[stream][t] = total;
      }
    }
    blocks += all_blocks;
    n += u.end - u.begin;
  }
}

template <int NT, int PT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
tree_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const TreeParams p) {
  using Sh = Shape<NT>;
  extern __shared__ uint8_t raw_smem[];
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  dependents_may_launch();

  // all steps of the launch, and where this CTA's run begins
  long long mine = 0;
#pragma unroll 1
  for (int row = thread; row < p.rows; row += Sh::kThreads) {
    const RowInfo r = row_info(p, row, PT);
    mine += (long long)r.steps * r.tiles * p.heads_kv;
  }
#pragma unroll 1
  for (int step = 16; step > 0; step >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, step);
  if (lane == 0) sm.sums[warp] = mine;
  if (thread == 0) {
#pragma unroll 1
    for (int i = 0; i < Sh::kStages; ++i) {
      tc::mbar_init(&sm.full_k[i], 1);
      tc::mbar_init(&sm.full_v[i], 1);
      tc::mbar_init(&sm.empty[i], 5);  // the values' four warps and the score product
      tc::mbar_init(&sm.k_ready[i], 1);
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sm.ka_full[i], 4);
      tc::mbar_init(&sm.ka_empty[i], 1);
      tc::mbar_init(&sm.va_full[i], 4);
      tc::mbar_init(&sm.va_empty[i], 1);
      for (int set = 0; set < 2; ++set) {
        tc::mbar_init(&sm.s_full[i][set][0], 1);
        tc::mbar_init(&sm.s_full[i][set][1], 1);
        tc::mbar_init(&sm.s_empty[i][set], 1);
        tc::mbar_init(&sm.p_full[i][set], 1);
        tc::mbar_init(&sm.p_empty[i][set], 1);
      }
    }
#pragma unroll 1
    for (int i = 0; i < kUnits; ++i) {
      tc::mbar_init(&sm.unit_full[i], 1);
      tc::mbar_init(&sm.unit_empty[i], kUnitReaders);
    }
    tc::mbar_init(&sm.q_full, 1);
    tc::mbar_init(&sm.o_full, 1);
    tc::mbar_init(&sm.o_empty, 1);
    tc::mbar_init(&sm.drained, 2);
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
#pragma unroll 1
    for (int w = 0; w < Sh::kThreads / 32; ++w) all += sm.sums[w];
    const long long per = max((all + gridDim.x - 1) / gridDim.x, 1ll);
    const long long first = per * blockIdx.x, last = min(first + per, all);
    if (lane == 0) {
      sm.per_cta = (int)min(per, (long long)INT32_MAX / 2);  // a unit that straddles is shorter
      sm.first = first;
      sm.last = last;
    }
    long long before = 0;
#pragma unroll 1
    for (int row0 = 0; row0 < p.rows && first < last; row0 += 32) {
      long long steps = 0;
      if (row0 + lane < p.rows) {
        const RowInfo r = row_info(p, row0 + lane, PT);
        steps = (long long)r.steps * r.tiles * p.heads_kv;
      }
      long long upto = steps;
#pragma unroll 1
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
    if (warp < 8) {
      trade_registers<Sh::kLaunchRegs, Sh::kValueRegs>();
      values<NT, PT>(p, sm, thread);
    } else if (warp < 16) {
      trade_registers<Sh::kLaunchRegs, Sh::kSoftmaxRegs>();
      softmax<NT>(p, sm, thread - 256);
    } else {
      trade_registers<Sh::kLaunchRegs, Sh::kControlRegs>();
      if (warp == 16) produce<NT, PT, 0>(p, sm, &k_map, lane);
      if (warp == 17) produce<NT, PT, 1>(p, sm, &v_map, lane);
      if (warp == 18) issue_scores<NT, PT>(sm);
      if (warp == 19) issue_output<NT>(sm);
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
    cudaError_t e = cudaFuncSetAttribute(tree_kernel<NT, PT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (slot >= 0) configured.done[slot] = true;
  }
  tree_kernel<NT, PT><<<kTreeCtas, Shape<NT>::kThreads, smem, stream>>>(k_map, v_map, p);
  return cudaGetLastError();
}

template <int PT>
static cudaError_t launch_tile(const CUtensorMap& k_map, const CUtensorMap& v_map, const TreeParams& p, cudaStream_t stream) {
  switch (p.tile) {
    case 16: return launch<16, PT>(k_map, v_map, p, stream);
    default: return launch<32, PT>(k_map, v_map, p, stream);
  }
}

}  // namespace tree
}  // namespace bdfp4
