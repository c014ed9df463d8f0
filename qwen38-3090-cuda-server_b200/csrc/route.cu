// Around the products grouped by expert: the router (softmax, top-k, slots sorted by expert) and the weighted combination of a token's
// expert outputs.
#include <atomic>
#include <climits>
#include <cfloat>
#include <type_traits>

#include "ragged.cuh"

namespace w4a16 {
namespace {

constexpr int kRouteWarps = 32;    // tokens of a block: one warp each, one bit each in the blocks' expert masks
constexpr int kRouteMaxK = 16;
constexpr int kRouteFewWarps = 8;  // tokens of a block while that spreads them over more SMs
constexpr int kRouteFewRows = 256, kRouteFewWords = 8000;  // blocks, and words of their counts, up to which every block adds them up itself
constexpr int kCombineThreads = 128, kCombineCtas = 8;  // and CTAs per SM at most

struct RouteParams {
  int32_t *ids, *offsets, *slots, *rows, *counts;
  float* weights;
  const void* logits;
  int f32, T, E, k, renormalize;
  int per, blocks;  // tokens of a block of k_route, and its blocks
  int few;          // every block adds up the counts itself
};
// Counts of a block's tokens per expert, if few: bytes (at most 32), four experts a word. Else words.
__device__ __forceinline__ int count_words(int E) { return (E + 3) / 4; }

// fp32 as an unsigned key of the same order; -inf and NaN become 0 (never picked), +inf the largest finite value. Negative numbers are
// negated as integers, not complemented: -0 so gets the key of +0, and the two are a tie.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(fminf(v, FLT_MAX));
  return u & 0x80000000u ? 0u - u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : 0u - k); }

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

// Picks of a block of PER tokens: a warp per token holds its logits in registers, EPL per lane (expert 32 i + lane). k times the
// largest key over the warp, then the lowest index that has it. Within a block the tokens that picked an expert are the bits of a
// word, so that a pick's place among them is a population count: sorted by expert and token without sorting.
// With one block the slots follow at once; otherwise the block's counts go out and k_route_scan and k_route_slots finish.
// Bound by its launches and their dependences: one token of 64 experts 5.8 us as an eager call, nearly all the host's (2.8 in a graph), 4096 tokens of 256
// experts 15.6 us in three launches (15.1 in a graph, 16.9 with the logits in HBM), where the logits take 0.7 at HBM's rate.
template <int EPL, int PER>
__global__ void __launch_bounds__(PER * 32) k_route(const RouteParams p) {
  __shared__ uint32_t masks[kMaxSets];
  __shared__ int offs[kMaxSets + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = blockIdx.x * PER + warp;
  constexpr int threads = PER * 32;
  for (int e = tid; e < 4 * count_words(p.E); e += threads) masks[e] = 0;
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
    // The lane's largest key and the first place that has it. With eight keys also the second largest: a lane that is picked goes on with that, and looks
    // for two more when it is picked again, which few lanes are (256 experts, 4096 tokens 15.9 -> 14.9 us; with two or four keys 3 % slower, with sixteen
    // 22.3 -> 16.0 at 4096 tokens, but 22.3 -> 24.4 at 8192: its registers leave room for one block per SM).
    constexpr bool TWO = EPL == 8;
    uint32_t best = 0, next = 0, gone = 0;  // (TWO: the places picked, where key stays as it is)
    int place = 0, next_place = 0;
    bool have_next = TWO;
    auto largest = [&]() {
      best = next = 0;
      place = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const uint32_t v = TWO && (gone >> i & 1u) ? 0u : key[i];
        if (v > best) {
          if constexpr (TWO) {
            next = best;
            next_place = place;
          }
          best = v;
          place = i;
        } else if (TWO && v > next) {
          next = v;
          next_place = i;
        }
      }
    };
    largest();
    for (int j = 0; j < p.k; ++j) {
      const uint32_t most = __reduce_max_sync(0xffffffffu, best);
      if (most == 0) break;  // nothing left to pick
      if (j == 0) {
        top = most;
        if (!p.renormalize) {
#pragma unroll
          for (int i = 0; i < EPL; ++i)
            if (key[i]) all += expf(key_value(key[i]) - key_value(top));
#pragma unroll
          for (int d = 16; d; d /= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
        }
      }
      const int at = __reduce_min_sync(0xffffffffu, best == most ? 32 * place + lane : INT_MAX);
      if ((at & 31) == lane) {  // only this lane looks for its next largest
        if constexpr (TWO) {
          gone |= 1u << place;
        } else {
#pragma unroll
          for (int i = 0; i < EPL; ++i)
            if (i == place) key[i] = 0;
        }
        if (TWO && have_next) {
          best = next;
          place = next_place;
        } else {
          largest();
        }
        have_next = TWO && !have_next;
      }
      if (lane == j) {
        my_id = at;
        my_key = most;
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
  if (p.few) {
    const int w = tid, words = count_words(p.E);
    if (w < words)
      p.counts[blockIdx.x * words + w] = __popc(masks[4 * w]) | __popc(masks[4 * w + 1]) << 8 | __popc(masks[4 * w + 2]) << 16 | __popc(masks[4 * w + 3]) << 24;
    return;
  }
  if (p.blocks > 1) {
    for (int e = tid; e < p.E; e += threads) p.counts[static_cast<size_t>(blockIdx.x) * p.E + e] = __popc(masks[e]);
    return;
  }
  for (int e = tid; e < p.E; e += threads) offs[e] = __popc(masks[e]);
  __syncthreads();
  if (warp == 0) scan_experts(offs, p.E, lane);
  __syncthreads();
  for (int e = tid; e <= p.E; e += threads) p.offsets[e] = offs[e];
  if (my_id >= 0) {
    const int slot = offs[my_id] + __popc(masks[my_id] & ((1u << warp) - 1u));
    p.slots[static_cast<size_t>(t) * p.k + lane] = slot;
    p.rows[slot] = t;
  }
}

// counts[block][e] -> the number in earlier blocks; the totals go to row `blocks`. A CTA takes 32 experts, a warp a 32nd of the blocks:
// sums of its part, a prefix sum over the warps, the part again.
__global__ void __launch_bounds__(kRouteWarps * 32) k_route_scan(const RouteParams p) {
  __shared__ int part[kRouteWarps][32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const int b0 = static_cast<int>(static_cast<long long>(p.blocks) * warp / kRouteWarps);
  const int b1 = static_cast<int>(static_cast<long long>(p.blocks) * (warp + 1) / kRouteWarps);
  int32_t* column = p.counts + e;
  int sum = 0;
  if (e < p.E)
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += __ldcg(column + static_cast<size_t>(b) * p.E);
  part[warp][lane] = sum;
  __syncthreads();
  if (e >= p.E) return;
  int run = 0;
  for (int w = 0; w < warp; ++w) run += part[w][lane];
  for (int b = b0; b < b1; ++b) {
    int32_t* at = column + static_cast<size_t>(b) * p.E;
    const int n = __ldcg(at);
    *at = run;
    run += n;
  }
  if (warp == kRouteWarps - 1) column[static_cast<size_t>(p.blocks) * p.E] = run;
}

// Slots of a block's picks: first slot of the expert, picks of earlier blocks, earlier tokens of the block. With few blocks it adds up
// their counts itself (whole numbers, in any order): a thread takes a word of four experts of some of the blocks and sums the bytes in
// halves of a word, at most 8192.
__global__ void __launch_bounds__(kRouteWarps * 32) k_route_slots(const RouteParams p) {
  __shared__ uint32_t masks[kMaxSets];
  __shared__ int offs[kMaxSets + 1], before[kMaxSets];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = blockIdx.x * kRouteWarps + warp;
  for (int e = tid; e < p.E; e += kRouteWarps * 32) masks[e] = 0;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  const int id = t < p.T && lane < p.k ? __ldcg(p.ids + static_cast<size_t>(t) * p.k + lane) : -1;
  if (id >= 0) atomicOr(&masks[id], 1u << warp);
  if (p.few) {
    const int mine_end = blockIdx.x * (kRouteWarps / p.per);  // (k_route's blocks may have fewer tokens)
    const int words = count_words(p.E), w = tid % words, step = kRouteWarps * 32 / words, first = tid / words;
    const bool takes = first < step && first < p.blocks;
    uint32_t all[2] = {}, mine[2] = {};
    if (takes)
#pragma unroll 8
      for (int b = first; b < p.blocks; b += step) {
        const uint32_t v = __ldcg(reinterpret_cast<const uint32_t*>(p.counts) + b * words + w), even = v & 0x00FF00FFu, odd = (v >> 8) & 0x00FF00FFu;
        all[0] += even;
        all[1] += odd;
        if (b < mine_end) {
          mine[0] += even;
          mine[1] += odd;
        }
      }
    for (int i = tid; i < 4 * words; i += kRouteWarps * 32) offs[i] = before[i] = 0;
    __syncthreads();
    if (takes)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int shift = i & 2 ? 16 : 0;
        atomicAdd(&offs[4 * w + i], static_cast<int>(all[i & 1] >> shift & 0xFFFFu));
        atomicAdd(&before[4 * w + i], static_cast<int>(mine[i & 1] >> shift & 0xFFFFu));
      }
  } else {
    for (int e = tid; e < p.E; e += kRouteWarps * 32) {
      offs[e] = __ldcg(p.counts + static_cast<size_t>(p.blocks) * p.E + e);
      before[e] = __ldcg(p.counts + static_cast<size_t>(blockIdx.x) * p.E + e);
    }
  }
  __syncthreads();
  if (warp == 0) scan_experts(offs, p.E, lane);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= p.E; e += kRouteWarps * 32) p.offsets[e] = offs[e];
  if (id >= 0) {
    const int slot = offs[id] + before[id] + __popc(masks[id] & ((1u << warp) - 1u));
    p.slots[static_cast<size_t>(t) * p.k + lane] = slot;
    p.rows[slot] = t;
  }
}

// 16 bytes global -> shared by this thread, or zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
struct CombineParams {
  uint16_t* y;
  const uint16_t *parts, *residual;
  const int32_t* slots;
  const float* weights;
  int parts_rows, T, k, H;
  uint32_t strips;  // of 256 columns
};

__device__ __forceinline__ void add_row(float (&s)[8], const uint4& v, float w) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[2 * i] = fmaf(w, __uint_as_float(u[i] << 16), s[2 * i]);
    s[2 * i + 1] = fmaf(w, __uint_as_float(u[i] & 0xFFFF0000u), s[2 * i + 1]);
  }
}

// A warp takes 256 columns of a token at a time, eight per lane: the picks' rows and the residual's by asynchronous copies through a ring
// in shared memory. A lane copies and reads its own 16 bytes of every row only, so that no barrier is needed, and the bytes in
// flight take no registers. Empty picks are filled with zeros. Bound by HBM: 4096 tokens of 8 picks x 5120, a tenth empty, 62.6 us (6.2 TB/s). On the way: rows in
// registers 100; a ring of three items 76; the residual in the ring and two items 65 (its load had been waited for where it is added); items counted
// on instead of four divisions each 66 with two items, 62.6 with four (4 picks x 5120 54.7 -> 39.6, one pick 36.2 -> 24.0).
template <int DEPTH>  // items of a warp in shared memory
__global__ void __launch_bounds__(kCombineThreads) k_combine(const CombineParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.k + (p.residual ? 1 : 0);
  const uint32_t item_bytes = rows * 512 + kRouteMaxK * 4;  // rows, the residual's among them, then the weights
  const uint32_t ring = smem_u32(smem) + warp * DEPTH * item_bytes;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t stride = gridDim.x * (kCombineThreads / 32), first = blockIdx.x * (kCombineThreads / 32) + warp;
  const uint32_t step_t = stride / p.strips, step_s = stride - step_t * p.strips, T = p.T;
  struct Item {
    uint32_t t, strip;
  };
  auto behind = [&](Item i) {
    i.t += step_t;
    i.strip += step_s;
    if (i.strip >= p.strips) {
      i.strip -= p.strips;
      ++i.t;
    }
    return i;
  };
  // lane j's pick j of an item, one step before the item's copies start
  int slot;
  float weight;
  auto pick = [&](const Item& i) {
    slot = -1;
    weight = 0.f;
    if (i.t < T && lane < p.k) {
      const size_t o = static_cast<size_t>(i.t) * p.k + lane;
      slot = __ldcg(p.slots + o);
      weight = __ldcg(p.weights + o);
    }
  };
  auto start = [&](const Item& i, uint32_t to, int row_of, float w) {
    if (i.t < T) {
      const int mine = row_of < p.parts_rows ? row_of : -1;
      const int col = i.strip * 256 + lane * 8;
      const bool inside = col < p.H;
      const uint16_t* src = p.parts + (inside ? col : 0);
      const uint32_t dst = to + lane * 16;
#pragma unroll 4
      for (int j = 0; j < p.k; ++j) {
        const int row = __shfl_sync(0xffffffffu, mine, j);
        cp_async16(dst + j * 512, src + static_cast<size_t>(max(row, 0)) * p.H, row >= 0 && inside);
      }
      if (p.residual) cp_async16(dst + p.k * 512, p.residual + static_cast<size_t>(i.t) * p.H + (inside ? col : 0), inside);
      if (lane < p.k) sts32(to + rows * 512 + lane * 4, __float_as_uint(mine >= 0 ? w : 0.f));
    }
    cp_async_commit();
  };
  Item item = {first / p.strips, first % p.strips}, ahead = item;
  pick(item);
  for (int i = 0; i < DEPTH - 1; ++i) {
    const int row_of = slot;
    const float w = weight;
    const Item now = ahead;
    ahead = behind(ahead);
    pick(ahead);
    start(now, ring + i * item_bytes, row_of, w);
  }
  int st = 0, st_ahead = DEPTH - 1;
  for (; item.t < T; item = behind(item)) {
    const int row_of = slot;
    const float w = weight;
    const Item now = ahead;
    ahead = behind(ahead);
    pick(ahead);
    __syncwarp();  // every lane has read the weights that the place held
    start(now, ring + st_ahead * item_bytes, row_of, w);
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    __syncwarp();
    const uint32_t at = ring + st * item_bytes;
    const int col = item.strip * 256 + lane * 8;
    float s[8] = {};
#pragma unroll 8
    for (int j = 0; j < p.k; ++j) add_row(s, lds128<0>(at + j * 512 + lane * 16), __uint_as_float(lds32(at + rows * 512 + j * 4)));
    if (p.residual) add_row(s, lds128<0>(at + p.k * 512 + lane * 16), 1.f);
    if (col < p.H) {
      uint32_t out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = float_to_bf16_bits(s[2 * i]) | (static_cast<uint32_t>(float_to_bf16_bits(s[2 * i + 1])) << 16);
      *reinterpret_cast<uint4*>(p.y + static_cast<size_t>(item.t) * p.H + col) = make_uint4(out[0], out[1], out[2], out[3]);
    }
    if (++st == DEPTH) st = 0;
    if (++st_ahead == DEPTH) st_ahead = 0;
  }
}

template <class Kernel, class Params>
int enqueue(Kernel kernel, dim3 grid, int threads, const Params& p, void* stream, const char* who, int smem = 0) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? W4A16_OK : fail(W4A16_ECUDA, "%s: launch: %s", who, cudaGetErrorString(e));
}

int route_blocks(int T) { return T / kRouteWarps + (T % kRouteWarps != 0); }

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
  // The second launch takes experts and counts as the first one left them, for indices: no table may lie in another, in the logits or in the workspace.
  const size_t table = static_cast<size_t>(T) * top_k * 4;
  const struct {
    const void* at;
    size_t bytes;
  } written[] = {{ids, table}, {weights, table}, {slots, table}, {rows, table}, {offsets, (num_experts + 1) * sizeof(int32_t)},
                 {blocks > 1 ? workspace : nullptr, blocks > 1 ? w4a16_route_workspace(T, num_experts) : 0}};
  for (int i = 0; T > 0 && i < 6; ++i) {
    W4_REQUIRE(ranges_apart(written[i].at, written[i].bytes, logits, static_cast<size_t>(T) * num_experts * (logits_are_f32 ? 4 : 2)),
               "route: logits overlap a table or the workspace");
    for (int j = 0; j < i; ++j)
      W4_REQUIRE(ranges_apart(written[i].at, written[i].bytes, written[j].at, written[j].bytes), "route: a table overlaps another or the workspace");
  }
  const DeviceInfo* di = device_info();
  if (!di) return W4A16_ECUDA;
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
  // A block of 32 tokens keeps one SM busy for microseconds (512 experts: 8): tokens that would leave SMs idle go eight to a block, as long
  // as their counts fit the workspace. Counts of few blocks are added up by every block of k_route_slots, of more by a kernel in between.
  // us in a graph, blocks of 32 and the kernel in between / this: 64 experts, 33 tokens 7.0 / 4.7, 1000 8.1 / 6.7; 256: 10.2 / 7.1,
  // 12.0 / 11.6; 512: 14.3 / 9.9, 18 / 15.7.
  // Without eight tokens to a block, the kernel in between / adding up: 64 experts, 4000 tokens (2000 words) 11.4 / 10.1; 128, 8000 (8000) 14.4 / 13.6, 8192
  // (8192) 13.1 / 13.7; 256, 2000 (4032) 13.9 / 14.0, 4000 (8000) 15.0 / 15.2, 4096 (8192) 15.1 / 15.3, 8192 (16384) 15.6 / 18.2; 512, 1300 (5248)
  // 17.4 / 20.6, 2048 (8192) 19.7 / 22.1, 4096 (16384) 23.5 / 26.0. Around 8000 words it is even, but for 512 experts, which would want fewer.
  const long long row_words = (num_experts + 3) / 4, narrow = (static_cast<long long>(T) + kRouteFewWarps - 1) / kRouteFewWarps;
  const bool spread = blocks > 1 && T <= kRouteFewWarps * di->sms && narrow * row_words <= kRouteFewWords &&
                      narrow * row_words <= (blocks + 1LL) * num_experts;
  p.per = spread ? kRouteFewWarps : kRouteWarps;
  p.blocks = spread ? static_cast<int>(narrow) : blocks;
  p.few = blocks > 1 && (spread || (blocks <= kRouteFewRows && blocks * row_words <= kRouteFewWords));
  const dim3 grid(p.blocks > 0 ? p.blocks : 1);  // (no tokens: the offsets are still written)
  const int per_lane = (num_experts + 31) / 32;
  auto picks = [&](auto per) {
    constexpr int PER = decltype(per)::value;
    if (per_lane <= 2) return enqueue(k_route<2, PER>, grid, PER * 32, p, stream, "route");
    if (per_lane <= 4) return enqueue(k_route<4, PER>, grid, PER * 32, p, stream, "route");
    if (per_lane <= 8) return enqueue(k_route<8, PER>, grid, PER * 32, p, stream, "route");
    return enqueue(k_route<16, PER>, grid, PER * 32, p, stream, "route");
  };
  int rc = spread ? picks(std::integral_constant<int, kRouteFewWarps>()) : picks(std::integral_constant<int, kRouteWarps>());
  if (rc != W4A16_OK || blocks <= 1) return rc;
  if (!p.few) rc = enqueue(k_route_scan, dim3((num_experts + 31) / 32), kRouteWarps * 32, p, stream, "route");
  if (rc != W4A16_OK) return rc;
  return enqueue(k_route_slots, dim3(blocks), kRouteWarps * 32, p, stream, "route");
}

int w4a16_experts_combine(uint16_t* y, const uint16_t* parts, int parts_rows, const int32_t* slots, const float* weights,
                          const uint16_t* residual, int T, int top_k, int hidden, void* stream) {
  W4_REQUIRE(T >= 0 && parts_rows >= 0, "experts_combine: %d tokens, %d rows", T, parts_rows);
  W4_REQUIRE(top_k >= 1 && top_k <= kRouteMaxK, "experts_combine: top_k %d (1..%d)", top_k, kRouteMaxK);
  W4_REQUIRE(hidden > 0 && hidden % 8 == 0, "experts_combine: hidden %d not a positive multiple of 8", hidden);
  if (T == 0) return W4A16_OK;
  W4_REQUIRE(y != nullptr && slots != nullptr && weights != nullptr && (parts != nullptr || parts_rows == 0), "experts_combine: null argument");
  W4_REQUIRE(((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(parts) | reinterpret_cast<uintptr_t>(residual)) & 15) == 0,
             "experts_combine: y, parts and residual must be 16-byte aligned");
  W4_REQUIRE(((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(weights)) & 3) == 0, "experts_combine: slots or weights not 4-byte aligned");
  const size_t yb = static_cast<size_t>(T) * hidden * 2;
  W4_REQUIRE(ranges_apart(parts, static_cast<size_t>(parts_rows) * hidden * 2, y, yb), "experts_combine: y overlaps parts");
  W4_REQUIRE(residual == nullptr || residual == y || ranges_apart(residual, yb, y, yb), "experts_combine: residual overlaps y but is not y");
  const size_t picks = static_cast<size_t>(T) * top_k * 4;
  W4_REQUIRE(ranges_apart(slots, picks, y, yb) && ranges_apart(weights, picks, y, yb), "experts_combine: y overlaps slots or weights");
  if (parts_rows == 0) parts = y;  // (no row is read, but the copies that fill empty picks with zeros name an address)
  const DeviceInfo* di = device_info();
  if (!di) return W4A16_ECUDA;
  const uint32_t strips = (static_cast<uint32_t>(hidden) + 255) / 256;
  W4_REQUIRE(static_cast<unsigned long long>(T) * strips <= INT_MAX, "experts_combine: %d tokens x %d are too many for one call", T, hidden);
  const CombineParams p = {y, parts, residual, slots, weights, parts_rows, T, top_k, hidden, strips};
  // Two items in the ring leave room for more warps, four keep more bytes in flight: us, two / four: 4096 tokens, 5120 columns of 4 picks 42.8 / 39.6, of 8
  // 66.2 / 62.6, 2048 columns of 16 47.1 / 59.6, 4096 of 2 23.1 / 23.6; where a warp has few items: 300 tokens, 8 picks x 5120 7.2 / 7.9, 1024 x 2048 9.1 / 9.7.
  const uint32_t items = static_cast<uint32_t>(T) * strips;
  const bool four = top_k > 2 && top_k <= 8 && items >= 128u * di->sms;
  const int smem = kCombineThreads / 32 * (four ? 4 : 2) * ((top_k + (residual ? 1 : 0)) * 512 + kRouteMaxK * 4);
  static std::atomic<bool> ready[64];
  if (!ready[di->device & 63].load(std::memory_order_acquire)) {
    W4_CUDA(cudaFuncSetAttribute(k_combine<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, di->smem_optin));
    W4_CUDA(cudaFuncSetAttribute(k_combine<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, di->smem_optin));
    ready[di->device & 63].store(true, std::memory_order_release);
  }
  const int fit = di->smem_per_sm / (smem + di->smem_reserved);
  const uint32_t ctas = (items + kCombineThreads / 32 - 1) / (kCombineThreads / 32);
  const uint32_t most = static_cast<uint32_t>(di->sms) * (fit < kCombineCtas ? fit : kCombineCtas);
  const dim3 grid(ctas < most ? ctas : most);
  return four ? enqueue(k_combine<4>, grid, kCombineThreads, p, stream, "experts_combine", smem)
              : enqueue(k_combine<2>, grid, kCombineThreads, p, stream, "experts_combine", smem);
}

}  // extern "C"
