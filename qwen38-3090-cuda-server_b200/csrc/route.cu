// Around the products grouped by expert: the router (softmax, top-k, slots sorted by expert) and the weighted combination of a token's
// expert outputs.
#include <climits>
#include <cfloat>

#include "ragged.cuh"

namespace w4a16 {
namespace {

constexpr int kRouteWarps = 32;    // tokens of a block: one warp each, one bit each in the blocks' expert masks
constexpr int kRouteMaxK = 16;
constexpr int kCombineThreads = 128;

struct RouteParams {
  int32_t *ids, *offsets, *slots, *rows, *counts;
  float* weights;
  const void* logits;
  int f32, T, E, k, renormalize, blocks;
};

// fp32 as an unsigned key of the same order; -inf and NaN become 0 (never picked), +inf the largest finite value
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(fminf(v, FLT_MAX));
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// Exclusive prefix sum of one int per expert (in place over totals[0, E)), the sum in totals[E]. Called by one whole warp.
__device__ __forceinline__ void scan_experts(int* totals, int E, int lane) {
  int run = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int mine = e0 + lane < E ? totals[e0 + lane] : 0;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (e0 + lane < E) totals[e0 + lane] = run + upto - mine;
    run += __shfl_sync(0xffffffffu, upto, 31);
  }
  __syncwarp();
  if (lane == 0) totals[E] = run;
}

// Picks of a block of 32 tokens: a warp per token holds its logits in registers, EPL per lane (expert 32 i + lane). k times the
// largest key over the warp, then the lowest index that has it. Within a block the tokens that picked an expert are the bits of a
// word, so that a pick's place among them is a population count: sorted by expert and token without sorting.
// With one block the slots follow at once; otherwise the block's counts go out and k_route_scan and k_route_slots finish.
template <int EPL>
__global__ void __launch_bounds__(kRouteWarps * 32) k_route(const RouteParams p) {
  __shared__ uint32_t masks[kMaxSets];
  __shared__ int offs[kMaxSets + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = blockIdx.x * kRouteWarps + warp;
  for (int e = tid; e < p.E; e += kRouteWarps * 32) masks[e] = 0;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  int my_id = -1;  // lane j: pick j
  if (t < p.T) {
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = 32 * i + lane;
      const size_t at = static_cast<size_t>(t) * p.E + e;
      key[i] = 0;
      if (e < p.E)
        key[i] = order_key(p.f32 ? __ldcg(static_cast<const float*>(p.logits) + at)
                                 : bf16_bits_to_float(__ldcg(static_cast<const uint16_t*>(p.logits) + at)));
    }
    uint32_t my_key = 0, top = 0;
    float all = 0.f;  // sum of exp over every expert
    for (int j = 0; j < p.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      if (best == 0) break;  // nothing left to pick
      if (j == 0) {
        top = best;
        if (!p.renormalize) {
#pragma unroll
          for (int i = 0; i < EPL; ++i)
            if (key[i]) all += expf(key_value(key[i]) - key_value(top));
#pragma unroll
          for (int d = 16; d; d /= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
        }
      }
      int at = INT_MAX;
#pragma unroll
      for (int i = EPL - 1; i >= 0; --i)
        if (key[i] == best) at = 32 * i + lane;
      at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (32 * i + lane == at) key[i] = 0;
      if (lane == j) {
        my_id = at;
        my_key = best;
      }
    }
    float mine = my_id >= 0 ? expf(key_value(my_key) - key_value(top)) : 0.f;
    if (p.renormalize) {
      all = 0.f;
      for (int j = 0; j < p.k; ++j) all += __shfl_sync(0xffffffffu, mine, j);  // in the picks' order
    }
    if (my_id >= 0) {
      mine /= all;
      atomicOr(&masks[my_id], 1u << warp);
    }
    if (lane < p.k) {
      p.ids[static_cast<size_t>(t) * p.k + lane] = my_id;
      p.weights[static_cast<size_t>(t) * p.k + lane] = mine;
      if (my_id < 0) p.slots[static_cast<size_t>(t) * p.k + lane] = -1;
    }
  }
  __syncthreads();
  if (p.blocks > 1) {
    for (int e = tid; e < p.E; e += kRouteWarps * 32) p.counts[static_cast<size_t>(blockIdx.x) * p.E + e] = __popc(masks[e]);
    return;
  }
  for (int e = tid; e < p.E; e += kRouteWarps * 32) offs[e] = __popc(masks[e]);
  __syncthreads();
  if (warp == 0) scan_experts(offs, p.E, lane);
  __syncthreads();
  for (int e = tid; e <= p.E; e += kRouteWarps * 32) p.offsets[e] = offs[e];
  if (my_id >= 0) {
    const int slot = offs[my_id] + __popc(masks[my_id] & ((1u << warp) - 1u));
    p.slots[static_cast<size_t>(t) * p.k + lane] = slot;
    p.rows[slot] = t;
  }
}

// counts[block][e] -> the number in earlier blocks, the totals go to row `blocks`. A warp per 32 experts walks the blocks.
__global__ void __launch_bounds__(32) k_route_scan(const RouteParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int e = blockIdx.x * 32 + threadIdx.x;
  if (e >= p.E) return;
  int run = 0;
  for (int b = 0; b < p.blocks; ++b) {
    int32_t* at = p.counts + static_cast<size_t>(b) * p.E + e;
    const int n = __ldcg(at);
    *at = run;
    run += n;
  }
  p.counts[static_cast<size_t>(p.blocks) * p.E + e] = run;
}

__global__ void __launch_bounds__(kRouteWarps * 32) k_route_slots(const RouteParams p) {
  __shared__ uint32_t masks[kMaxSets];
  __shared__ int offs[kMaxSets + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = blockIdx.x * kRouteWarps + warp;
  for (int e = tid; e < p.E; e += kRouteWarps * 32) masks[e] = 0;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  const int id = t < p.T && lane < p.k ? __ldcg(p.ids + static_cast<size_t>(t) * p.k + lane) : -1;
  if (id >= 0) atomicOr(&masks[id], 1u << warp);
  for (int e = tid; e < p.E; e += kRouteWarps * 32) offs[e] = __ldcg(p.counts + static_cast<size_t>(p.blocks) * p.E + e);
  __syncthreads();
  if (warp == 0) scan_experts(offs, p.E, lane);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= p.E; e += kRouteWarps * 32) p.offsets[e] = offs[e];
  if (id >= 0) {
    const int slot = offs[id] + __ldcg(p.counts + static_cast<size_t>(blockIdx.x) * p.E + id) + __popc(masks[id] & ((1u << warp) - 1u));
    p.slots[static_cast<size_t>(t) * p.k + lane] = slot;
    p.rows[slot] = t;
  }
}

struct CombineParams {
  uint16_t* y;
  const uint16_t *parts, *residual;
  const int32_t* slots;
  const float* weights;
  int parts_rows, k, H;
};

__device__ __forceinline__ void add_row(float (&s)[8], const uint4& v, float w) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[2 * i] = fmaf(w, __uint_as_float(u[i] << 16), s[2 * i]);
    s[2 * i + 1] = fmaf(w, __uint_as_float(u[i] & 0xFFFF0000u), s[2 * i + 1]);
  }
}

// A thread takes eight columns of a token; the loads of a token's rows are in flight together.
__global__ void __launch_bounds__(kCombineThreads) k_combine(const CombineParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int col = (blockIdx.y * kCombineThreads + threadIdx.x) * 8;
  const size_t t = blockIdx.x;
  if (col >= p.H) return;
  float s[8] = {};
  for (int j0 = 0; j0 < p.k; j0 += 8) {
    uint4 v[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = 0.f;
      v[j] = make_uint4(0, 0, 0, 0);
      if (j0 + j < p.k) {
        const int slot = __ldcg(p.slots + t * p.k + j0 + j);
        if (slot >= 0 && slot < p.parts_rows) {
          w[j] = __ldcg(p.weights + t * p.k + j0 + j);
          v[j] = __ldcg(reinterpret_cast<const uint4*>(p.parts + static_cast<size_t>(slot) * p.H + col));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) add_row(s, v[j], w[j]);
  }
  const size_t o = t * p.H + col;
  if (p.residual) add_row(s, *reinterpret_cast<const uint4*>(p.residual + o), 1.f);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = float_to_bf16_bits(s[2 * i]) | (static_cast<uint32_t>(float_to_bf16_bits(s[2 * i + 1])) << 16);
  *reinterpret_cast<uint4*>(p.y + o) = make_uint4(out[0], out[1], out[2], out[3]);
}

template <class Kernel, class Params>
int enqueue(Kernel kernel, dim3 grid, int threads, const Params& p, void* stream, const char* who) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? W4A16_OK : fail(W4A16_ECUDA, "%s: launch: %s", who, cudaGetErrorString(e));
}

int route_blocks(int T) { return (T + kRouteWarps - 1) / kRouteWarps; }

}  // namespace
}  // namespace w4a16

using namespace w4a16;

extern "C" {

size_t w4a16_route_workspace(int max_tokens, int num_experts) {
  if (max_tokens < 0 || num_experts < 1 || num_experts > kMaxSets) return 0;
  return (static_cast<size_t>(route_blocks(max_tokens)) + 1) * num_experts * sizeof(int32_t);
}

int w4a16_route(int32_t* ids, float* weights, int32_t* offsets, int32_t* slots, int32_t* rows, const void* logits, int logits_are_f32,
                int T, int num_experts, int top_k, int renormalize, void* workspace, size_t workspace_bytes, void* stream) {
  W4_REQUIRE(num_experts >= 1 && num_experts <= kMaxSets, "route: %d experts (1..%d)", num_experts, kMaxSets);
  W4_REQUIRE(top_k >= 1 && top_k <= kRouteMaxK && top_k <= num_experts, "route: top_k %d of %d experts (at most %d)", top_k, num_experts, kRouteMaxK);
  W4_REQUIRE(T >= 0 && static_cast<long long>(T) * top_k <= INT_MAX, "route: T = %d", T);
  W4_REQUIRE(offsets != nullptr, "route: null offsets");
  W4_REQUIRE(T == 0 || (ids != nullptr && weights != nullptr && slots != nullptr && rows != nullptr && logits != nullptr), "route: null argument");
  const uintptr_t words = reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(offsets) |
                          reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(workspace);
  W4_REQUIRE((words & 3) == 0 && (reinterpret_cast<uintptr_t>(logits) & (logits_are_f32 ? 3 : 1)) == 0, "route: misaligned argument");
  const int blocks = route_blocks(T);
  if (blocks > 1 && (workspace == nullptr || workspace_bytes < w4a16_route_workspace(T, num_experts)))
    return fail(W4A16_ESCRATCH, "route: workspace of %zu bytes for %d tokens, %zu needed", workspace_bytes, T, w4a16_route_workspace(T, num_experts));
  RouteParams p = {};
  p.ids = ids;
  p.weights = weights;
  p.offsets = offsets;
  p.slots = slots;
  p.rows = rows;
  p.counts = static_cast<int32_t*>(workspace);
  p.logits = logits;
  p.f32 = logits_are_f32 != 0;
  p.T = T;
  p.E = num_experts;
  p.k = top_k;
  p.renormalize = renormalize != 0;
  p.blocks = blocks;
  const dim3 grid(blocks > 0 ? blocks : 1);  // (no tokens: the offsets are still written)
  const int per_lane = (num_experts + 31) / 32;
  int rc;
  if (per_lane <= 2) rc = enqueue(k_route<2>, grid, kRouteWarps * 32, p, stream, "route");
  else if (per_lane <= 4) rc = enqueue(k_route<4>, grid, kRouteWarps * 32, p, stream, "route");
  else if (per_lane <= 8) rc = enqueue(k_route<8>, grid, kRouteWarps * 32, p, stream, "route");
  else rc = enqueue(k_route<16>, grid, kRouteWarps * 32, p, stream, "route");
  if (rc != W4A16_OK || blocks <= 1) return rc;
  rc = enqueue(k_route_scan, dim3((num_experts + 31) / 32), 32, p, stream, "route");
  if (rc != W4A16_OK) return rc;
  return enqueue(k_route_slots, grid, kRouteWarps * 32, p, stream, "route");
}

int w4a16_experts_combine(uint16_t* y, const uint16_t* parts, int parts_rows, const int32_t* slots, const float* weights,
                          const uint16_t* residual, int T, int top_k, int hidden, void* stream) {
  W4_REQUIRE(T >= 0 && parts_rows >= 0, "experts_combine: %d tokens, %d rows", T, parts_rows);
  W4_REQUIRE(top_k >= 1 && top_k <= kRouteMaxK, "experts_combine: top_k %d (1..%d)", top_k, kRouteMaxK);
  W4_REQUIRE(hidden > 0 && hidden % 8 == 0 && hidden <= 8 * kCombineThreads * 65535, "experts_combine: hidden %d not a positive multiple of 8", hidden);
  if (T == 0) return W4A16_OK;
  W4_REQUIRE(y != nullptr && slots != nullptr && weights != nullptr && (parts != nullptr || parts_rows == 0), "experts_combine: null argument");
  W4_REQUIRE(((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(parts) | reinterpret_cast<uintptr_t>(residual)) & 15) == 0,
             "experts_combine: y, parts and residual must be 16-byte aligned");
  W4_REQUIRE(((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(weights)) & 3) == 0, "experts_combine: slots or weights not 4-byte aligned");
  const size_t yb = static_cast<size_t>(T) * hidden * 2;
  W4_REQUIRE(ranges_apart(parts, static_cast<size_t>(parts_rows) * hidden * 2, y, yb), "experts_combine: y overlaps parts");
  W4_REQUIRE(residual == nullptr || residual == y || ranges_apart(residual, yb, y, yb), "experts_combine: residual overlaps y but is not y");
  const CombineParams p = {y, parts, residual, slots, weights, parts_rows, top_k, hidden};
  const dim3 grid(T, (hidden / 8 + kCombineThreads - 1) / kCombineThreads);
  return enqueue(k_combine, grid, kCombineThreads, p, stream, "experts_combine");
}

}  // extern "C"
