// Verification of a drafted tree against the target's probabilities.
//
// The walk itself needs one probability per drafted token: they are gathered up front, all at once. What
// costs bandwidth is a vocabulary row of the node where the walk ends (the next token's draw) and, when a
// drafter's distribution is given, one pass over both rows per refusal, whose sum is the new mass. A pass
// leaves the weight of every warp's slice behind, so the draw after it re-reads one slice only. Sums run in
// FP64: acceptance and the drawn index are decisions next to borders, and at 4 to 8 bytes read per value the
// FP64 adds (64 per clock and SM) stay well under the time of the reads.
//
// Small batches are bound by the launch (8 us on the device); 32 rows x 131072 with a drafter take 28 to 31 us, five to
// six times the reads' time: what counts is the chain of a cluster's passes, one per refusal, each a read, a reduction
// and an exchange.
//
// A row is one cluster of CTAs that share the vocabulary; every CTA does the same walk from the same
// numbers, and the passes' sums are exchanged through distributed shared memory. A CTA may only store into
// another's once that one runs: all arrive on the cluster's barrier as they start, and wait for it before their
// first store, behind the gather, the walk and the first pass.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host.h"

namespace bdfp4 {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCluster = 8;
constexpr int kMaxNodes = BDFP4_MAX_TREE_NODES;

struct VerifyParams {
  int rows, nodes, vocab, span;  // span: vocabulary entries of one warp, a multiple of a warp's 16-byte loads
  const void* target;
  int64_t target_row, target_node;
  const void* draft;
  int64_t draft_row, draft_node;
  const int32_t* tokens;
  int64_t tokens_stride;
  const int32_t* parents;
  int64_t parents_stride;
  const float* uniforms;
  int64_t uniforms_stride;
  const int32_t* counts;
  int32_t* accepted;
  int32_t* accepted_counts;
  int32_t* next_tokens;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Sixteen bytes of a probability row. A row may start at any element (odd vocabularies): `lead` is the
// number of elements between the 16-byte boundary before it and its first one, and granule g holds the
// elements g * E - lead + (0 .. E-1); those outside [0, vocab) read as zero.
template <typename T>
struct RowReader {
  static constexpr int E = 16 / sizeof(T);
  const T* row;
  int lead, vocab;
  __device__ RowReader(const T* r, int n) : row(r), lead((int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T))), vocab(n) {}
  // `first` is the vocabulary index of v[0], with this reader's own lead taken into account by the caller
  __device__ __forceinline__ void load(int first, float* v) const {
    if (first >= 0 && first + E <= vocab && ((first + lead) & (E - 1)) == 0) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + first));
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = to_float(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = (first + i >= 0 && first + i < vocab) ? to_float(row[first + i]) : 0.0f;
    }
  }
};

// What turns a node's distribution into the weights that are left of it.
//
// With a drafter, a refusal makes max(w / W - q, 0) of w and W the sum of that. Scaled by the product of the W so
// far, which changes neither a draw nor a comparison with the (equally scaled) mass, that is max(w - W q, 0), and
// refusals in a row collapse: what is left of p after them is max(p - q (W_0 + W_1 + ...), 0), one FP64 FMA per
// value however many there were. (Step by step with their divisions, 32 rows x 131072 with up to five refusals
// took 110 us.)
struct Refusals {
  int steps;      // drafter given: refusals so far
  double share;   // ... and the sum of the masses before them
  int count;      // no drafter: refused tokens, whose weight is zero
  int token[kMaxNodes];
};

__device__ __forceinline__ double subtracted(double w, double q, double share) { return fmax(fma(-share, q, w), 0.0); }

template <typename T, bool DRAFT>
struct Verifier {
  static constexpr int E = RowReader<T>::E;
  const VerifyParams& p;
  const Refusals& r;
  int lane;

  // The weights of the lane's granule of one 32-granule chunk.
  __device__ __forceinline__ void weights(const RowReader<T>& target, const RowReader<T>& draft, int first, double* w) const {
    float v[E];
    target.load(first, v);
    if (DRAFT && r.steps > 0) {
      float q[E];
      draft.load(first, q);
      const double share = r.share;
#pragma unroll
      for (int i = 0; i < E; ++i) w[i] = subtracted((double)v[i], (double)q[i], share);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) w[i] = (double)v[i];
    }
    if (!DRAFT && r.count > 0) {
      const int chunk = __shfl_sync(0xffffffffu, first, 0);
      const int end = chunk + 32 * E;
      bool hit = false;
      for (int j = lane; j < r.count; j += 32) hit |= r.token[j] >= chunk && r.token[j] < end;
      if (__any_sync(0xffffffffu, hit)) {
        for (int j = 0; j < r.count; ++j) {
          const int at = r.token[j] - first;
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (at == i) w[i] = 0.0;
        }
      }
    }
  }

  // Total weight of warp `g`'s slice of the vocabulary.
  __device__ __forceinline__ double slice_total(const RowReader<T>& target, const RowReader<T>& draft, int g) const {
    const int64_t begin = (int64_t)g * p.span - target.lead;
    const int64_t end = min(begin + p.span, (int64_t)p.vocab);
    double sum = 0.0;
#pragma unroll 2
    for (int64_t chunk = begin; chunk < end; chunk += 32 * E) {
      double w[E];
      weights(target, draft, (int)chunk + lane * E, w);
#pragma unroll
      for (int i = 0; i < E; ++i) sum += w[i];
    }
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, step);
    return sum;
  }

  // The first index of warp `g`'s slice whose cumulative weight (on top of `before`) exceeds `goal`; its last
  // index of positive weight if none does.
  __device__ __forceinline__ int locate(const RowReader<T>& target, const RowReader<T>& draft, int g, double before, double goal) const {
    const int64_t begin = (int64_t)g * p.span - target.lead;
    const int64_t end = min(begin + p.span, (int64_t)p.vocab);
    int last = -1;
    for (int64_t chunk = begin; chunk < end; chunk += 32 * E) {
      double w[E], mine = 0.0;
      const int first = (int)chunk + lane * E;
      weights(target, draft, first, w);
#pragma unroll
      for (int i = 0; i < E; ++i) mine += w[i];
      double upto = mine;
#pragma unroll
      for (int step = 1; step < 32; step <<= 1) {
        const double left = __shfl_up_sync(0xffffffffu, upto, step);
        if (lane >= step) upto += left;
      }
      double running = before + (upto - mine);
      int found = -1, positive = -1;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        running += w[i];
        if (w[i] > 0.0) positive = first + i;
        if (found < 0 && running > goal && w[i] > 0.0) found = first + i;
      }
      const unsigned any = __ballot_sync(0xffffffffu, found >= 0);
      if (any) return __shfl_sync(0xffffffffu, found, __ffs(any) - 1);
      const unsigned some = __ballot_sync(0xffffffffu, positive >= 0);
      if (some) last = __shfl_sync(0xffffffffu, positive, 31 - __clz(some));
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return last;
  }
};

// All threads of every CTA of the cluster, once each; the warps converged.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// (Two CTAs per SM: with one, at 100 registers, 32 rows in clusters of eight were two waves, 35 us instead of 25.)
template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const VerifyParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank();
  const int row = blockIdx.x / parts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ int s_token[kMaxNodes], s_parent[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ float s_p[kMaxNodes], s_q[kMaxNodes];  // the parent's target and draft probability of the node's token
  __shared__ Refusals s_refusals;
  __shared__ double s_totals[2][kVerifyMaxCluster * kVerifyWarps];
  __shared__ int s_here, s_resume, s_pass;  // where the walk stands; whether a pass over the vocabulary is due
  __shared__ double s_mass, s_share_before;

  const int count = p.counts ? min(max(p.counts[row], 0), p.nodes) : p.nodes;
  int32_t* accepted = p.accepted + (int64_t)row * p.nodes;
  if (count == 0) {  // the same in every CTA of the cluster
    if (part == 0) {
      for (int i = threadIdx.x; i < p.nodes; i += kVerifyThreads) accepted[i] = -1;
      if (threadIdx.x == 0) {
        p.accepted_counts[row] = 0;
        p.next_tokens[row] = -1;
      }
    }
    return;
  }
  if (parts > 1) cluster_arrive();
  const T* target = static_cast<const T*>(p.target) + row * p.target_row;
  const T* draft = DRAFT ? static_cast<const T*>(p.draft) + row * p.draft_row : nullptr;
  if ((int)threadIdx.x < count) {
    const int i = threadIdx.x;
    const int token = p.tokens[row * p.tokens_stride + i];
    int parent = p.parents[row * p.parents_stride + i];
    if (parent >= i) parent = -1;
    s_parent[i] = parent;
    s_token[i] = token;
    s_u[i] = p.uniforms[row * p.uniforms_stride + i];
    const bool known = i > 0 && parent >= 0 && token >= 0 && token < p.vocab;
    s_p[i] = known ? to_float(target[parent * p.target_node + token]) : 0.0f;
    s_q[i] = DRAFT && known ? to_float(draft[parent * p.draft_node + token]) : 1.0f;
  }
  if (threadIdx.x == 0) {
    s_here = 0;
    s_resume = 1;
    s_mass = 1.0;
    s_refusals.steps = s_refusals.count = 0;
    s_refusals.share = 0.0;
  }
  __syncthreads();

  int buffer = 0, depth = 1;
  if (part == 0 && threadIdx.x == 0) accepted[0] = 0;
  const int g = part * kVerifyWarps + warp, warps = parts * kVerifyWarps;
  bool summed = false;  // s_totals[buffer] holds the current weights' sums
  bool started = parts == 1;  // every CTA of the cluster is known to run
  double total = 0.0;
  while (true) {
    if (warp == 0) {  // the walk, up to its end or to a refusal that needs a pass
      int here = s_here, i = s_resume;
      double mass = s_mass;
      bool pass = false;
      for (; i < count; ++i) {
        // the next child of `here`, among 64 nodes two per lane
        const unsigned low = __ballot_sync(0xffffffffu, lane >= i && lane < count && lane > 0 && s_parent[lane] == here);
        const unsigned high =
            __ballot_sync(0xffffffffu, lane + 32 >= i && lane + 32 < count && s_parent[lane + 32] == here);
        if (!low && !high) {
          i = count;
          break;
        }
        i = low ? __ffs(low) - 1 : 32 + __ffs(high) - 1;
        double w = s_p[i];
        const double q = s_q[i];
        if (DRAFT) {
          w = subtracted(w, q, s_refusals.share);
        } else {
          bool gone = false;
          for (int j = lane; j < s_refusals.count; j += 32) gone |= s_refusals.token[j] == s_token[i];
          if (__any_sync(0xffffffffu, gone)) w = 0.0;
        }
        if ((double)s_u[i] * q * mass < w) {
          here = i;
          mass = 1.0;
          __syncwarp();
          if (lane == 0) {
            s_refusals.steps = s_refusals.count = 0;
            s_refusals.share = 0.0;
            if (part == 0) accepted[depth] = i;
          }
          ++depth;
          __syncwarp();
        } else if (DRAFT) {
          pass = true;
          __syncwarp();
          if (lane == 0) {
            s_share_before = s_refusals.share;
            s_refusals.share += mass;
            ++s_refusals.steps;
          }
          ++i;
          break;
        } else {
          mass = fmax(mass - w, 0.0);
          __syncwarp();
          if (lane == 0 && s_token[i] >= 0 && s_token[i] < p.vocab) s_refusals.token[s_refusals.count++] = s_token[i];
          __syncwarp();
        }
      }
      if (lane == 0) {
        s_here = here;
        s_resume = i;
        s_mass = mass;
        s_pass = pass;
      }
    }
    __syncthreads();
    const bool more = s_pass;
    const int here = s_here;
    if (!more && summed && s_refusals.steps > 0) break;  // the last refusal's sums are the draw's
    // The walk ends at a node whose weights have not been summed, or a refusal asks for the new mass.
    const RowReader<T> target_row(target + here * p.target_node, p.vocab);
    const RowReader<T> draft_row(DRAFT ? draft + here * p.draft_node : target, p.vocab);
    bool whole = false;
    while (true) {
      const Verifier<T, DRAFT> verifier{p, s_refusals, lane};
      const double mine = verifier.slice_total(target_row, draft_row, g);
      buffer ^= 1;
      if (!started) cluster_wait();
      started = true;
      if (lane < parts) cluster.map_shared_rank(&s_totals[buffer][0], lane)[g] = mine;
      if (parts > 1) cluster.sync();
      else __syncthreads();
      total = 0.0;
      for (int j = lane; j < warps; j += 32) total += s_totals[buffer][j];
#pragma unroll
      for (int step = 16; step > 0; step >>= 1) total += __shfl_xor_sync(0xffffffffu, total, step);
      if (more || total > 0.0 || whole || !(s_refusals.steps > 0 || s_refusals.count > 0)) break;
      // nothing is left of the distribution: it stands as it is
      whole = true;
      __syncthreads();
      if (threadIdx.x == 0) {
        s_refusals.steps = s_refusals.count = 0;
        s_refusals.share = 0.0;
      }
      __syncthreads();
    }
    if (!more) break;
    summed = true;
    __syncthreads();
    if (threadIdx.x == 0) {
      if (total > 0.0) s_mass = total;
      else {  // the drafter covers the rest of the target: the refusal changes nothing
        --s_refusals.steps;
        s_refusals.share = s_share_before;
      }
    }
    if (!(total > 0.0)) summed = false;
    __syncthreads();
  }

  if (part == 0 && warp == 0) {
    for (int i = depth + lane; i < p.nodes; i += 32) accepted[i] = -1;
    if (lane == 0) p.accepted_counts[row] = depth;
  }
  // The warp whose slice the goal falls into finds the token; with a goal at or past the total, the last
  // slice of positive weight.
  const double goal = (double)s_u[0] * total;
  // (Every warp finds its slice by itself: a lane adds up to four of them, then a scan over the lanes.)
  constexpr int kPerLane = kVerifyMaxCluster * kVerifyWarps / 32;
  double slice[kPerLane], mine = 0.0;
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) {
    const int at = lane * kPerLane + j;
    slice[j] = at < warps ? s_totals[buffer][at] : 0.0;
    mine += slice[j];
  }
  double upto = mine;
#pragma unroll
  for (int step = 1; step < 32; step <<= 1) {
    const double left = __shfl_up_sync(0xffffffffu, upto, step);
    if (lane >= step) upto += left;
  }
  double running = upto - mine, found_before = 0.0, last_before = 0.0;
  int found = -1, last = -1;
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) {
    if (slice[j] > 0.0) {
      last = lane * kPerLane + j;
      last_before = running;
      if (found < 0 && running + slice[j] > goal) {
        found = last;
        found_before = running;
      }
    }
    running += slice[j];
  }
  const unsigned any = __ballot_sync(0xffffffffu, found >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
  const int from = any ? __ffs(any) - 1 : some ? 31 - __clz(some) : 0;
  const int owner = __shfl_sync(0xffffffffu, any ? found : last, from);
  const double before = __shfl_sync(0xffffffffu, any ? found_before : last_before, from);
  if (owner < 0) {
    if (g == 0 && lane == 0) p.next_tokens[row] = 0;  // a row without any weight
  } else if (g == owner) {
    const int here = s_here;
    const RowReader<T> target_row(target + here * p.target_node, p.vocab);
    const RowReader<T> draft_row(DRAFT ? draft + here * p.draft_node : target, p.vocab);
    const Verifier<T, DRAFT> verifier{p, s_refusals, lane};
    const int token = verifier.locate(target_row, draft_row, g, before, goal);
    if (lane == 0) p.next_tokens[row] = max(token, 0);
  }
}

template <typename T, bool DRAFT>
static cudaError_t launch_verify(const VerifyParams& params, cudaStream_t stream) {
  VerifyParams p = params;
  constexpr int chunk = 32 * RowReader<T>::E;
  // A row's CTAs: as many as fill the GPU twice over, while a warp still has two chunks (one in flight
  // behind the other) to read.
  int parts = 1;
  while (parts < kVerifyMaxCluster && (int64_t)p.rows * parts * 2 <= 2 * 148 &&
         p.vocab >= (int64_t)parts * 2 * kVerifyWarps * chunk * 2)
    parts *= 2;
  const int64_t per_warp = (p.vocab + RowReader<T>::E - 1 + (int64_t)parts * kVerifyWarps - 1) / (parts * kVerifyWarps);
  p.span = (int)((per_warp + chunk - 1) / chunk * chunk);
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = parts;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(p.rows * parts));
  config.blockDim = dim3(kVerifyThreads);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, verify_kernel<T, DRAFT>, p);
}

}  // namespace bdfp4

using namespace bdfp4;

extern "C" int bdfp4_verify_drafts(const bdfp4_verify_args* a, void* stream_handle) {
  if (!a) return BDFP4_E_ARG;
  if (a->rows < 1 || a->nodes < 1 || a->vocab < 1) return BDFP4_E_ARG;
  if (a->nodes > kMaxNodes || a->rows > (1 << 24) || a->vocab > (1 << 30)) return BDFP4_E_UNSUPPORTED;
  if (!a->target_probs || !a->tokens || !a->parents || !a->uniforms || !a->accepted || !a->accepted_counts ||
      !a->next_tokens)
    return BDFP4_E_ARG;
  const uintptr_t element = a->bf16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(a->target_probs) % element || reinterpret_cast<uintptr_t>(a->draft_probs) % element)
    return BDFP4_E_ARG;
  VerifyParams p{};
  p.rows = a->rows;
  p.nodes = a->nodes;
  p.vocab = a->vocab;
  p.target = a->target_probs;
  p.target_row = a->target_row_stride;
  p.target_node = a->target_node_stride;
  p.draft = a->draft_probs;
  p.draft_row = a->draft_row_stride;
  p.draft_node = a->draft_node_stride;
  p.tokens = a->tokens;
  p.tokens_stride = a->tokens_row_stride;
  p.parents = a->parents;
  p.parents_stride = a->parents_row_stride;
  p.uniforms = a->uniforms;
  p.uniforms_stride = a->uniforms_row_stride;
  p.counts = a->node_counts;
  p.accepted = a->accepted;
  p.accepted_counts = a->accepted_counts;
  p.next_tokens = a->next_tokens;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  cudaError_t e;
  if (a->bf16)
    e = a->draft_probs ? launch_verify<__nv_bfloat16, true>(p, stream) : launch_verify<__nv_bfloat16, false>(p, stream);
  else
    e = a->draft_probs ? launch_verify<float, true>(p, stream) : launch_verify<float, false>(p, stream);
  return bdfp4::cuda_status(e);
}
