// Linear layers over ragged sets of tokens with their epilogue: what the decode-side kernel (ragged.cu) and the prefill kernel
// (prefill.cu) share. A dense layer is one set with all tokens.
#pragma once
#include "common.cuh"

namespace w4a16 {

// y[p] = bf16(act(x[row of p] W_e^T + bias_e) + residual[p]) for the slots p in [offsets[e], offsets[e + 1]) of every set e.
struct RaggedCall {
  const uint8_t* stream;     // the sets' weight streams one after another
  size_t set_bytes;          // from one set's stream to the next
  int sets, N, K, G;
  const uint16_t* x;         // [x_tokens][K]
  int x_tokens;
  const int32_t* x_rows;     // row of x of every slot (null: slot p takes row p)
  const int32_t* offsets;    // [sets + 1] on the device (null: one set with all slots)
  int slots;
  const uint16_t* bias;      // [sets][N] in the checkpoint's row order, or null
  int act;
  const uint16_t* residual;  // laid out as y, or null; may be y itself
  uint16_t* y;               // [slots][ny]
  int ny;                    // N, or N / 2 with the gated activation
};

// The prefill kernel on a checked call (prefill.cu).
int launch_prefill_ragged(const RaggedCall& c, cudaStream_t stream);

#ifdef __CUDACC__
// v / (1 + exp(-v)); the gated and the tanh form come back to it: 0.5 v (1 + tanh u) = v / (1 + exp(-2 u)) holds its precision where
// the tanh is near -1. Two special-function instructions a value. From exp(-u) = 2^126 on (u = -87.3, results under 2^-119) the quotient is zero.
__device__ __forceinline__ float logistic_times(float v, float u) { return __fdividef(v, 1.f + __expf(-u)); }

// v / 2 erfc(-v / sqrt 2). With x = |v| / sqrt 2 and t = 1 / (1 + x / 2), erfc(x) = t exp(P(t) - x^2), the form of Numerical Recipes; P is a fit of our
// own, the polynomial through ln(erfc(x) exp(x^2) / t) at Chebyshev nodes of t for x in [0, 13.3] (erfc leaves fp32 at x = 10). Relative error
// of erfc by the polynomial 8e-7; with the steps in fp32 (x^2 counts the rounding of x twice) 2.2e-6 for x < 4, 7.6e-6 at x = 7.7 (v = -10.8), 1.7e-5
// at x = 10, the last emulated with an exact exp, to which __expf adds up to (2 + 1.2 x^2) 2^-23: 2^-15.8 in all where the result is above
// 2^-92, 2^-15 where erfc leaves fp32; rounding to bf16 adds 2^-8. (erfcf, a call of some 60 instructions per value, made 34816 x 5120 at M = 4096 with GELU
// 1437 us instead of 1235.)
__device__ __forceinline__ float gelu_erf(float v) {
  const float x = 0.70710678119f * fabsf(v), t = __fdividef(1.f, 1.f + 0.5f * x);
  float e = -0.19175600f;
  e = fmaf(e, t, 0.76816076f);
  e = fmaf(e, t, -1.0295521f);
  e = fmaf(e, t, 0.37581054f);
  e = fmaf(e, t, -0.053080898f);
  e = fmaf(e, t, 0.39786267f);
  e = fmaf(e, t, 0.99799556f);
  e = fmaf(e, t, -1.2654413f);
  e = 0.5f * t * __expf(fmaf(-x, x, e));
  return v * (v > 0.f ? 1.f - e : e);
}

// An activation that acts on each output by itself, in fp32.
template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == W4A16_ACT_SILU) return logistic_times(v, v);
  if constexpr (ACT == W4A16_ACT_GELU_TANH) return logistic_times(v, 1.5957691216f * (v + 0.044715f * v * v * v));  // 2 sqrt(2 / pi)
  if constexpr (ACT == W4A16_ACT_GELU) return gelu_erf(v);
  return v;
}
__device__ __forceinline__ float activate(float v, int act) {
  if (act == W4A16_ACT_NONE) return v;
  if (act == W4A16_ACT_SILU) return activate<W4A16_ACT_SILU>(v);
  return act == W4A16_ACT_GELU ? activate<W4A16_ACT_GELU>(v) : activate<W4A16_ACT_GELU_TANH>(v);
}
// Index of a container row's bias: with the gated activation rows alternate gate, up, gate, up ...; the bias is [gate | up].
__device__ __forceinline__ int bias_index(int row, int N, int act) {
  return act == W4A16_ACT_SWIGLU ? (row >> 1) + (row & 1) * (N >> 1) : row;
}
// The sets' slots into bounds[0 .. sets), by all THREADS threads of the block: within [0, slots] whatever the offsets hold, and no slot in two
// sets. That keeps the number of units within what the launch was laid out for and no output is written twice. Offsets that descend somewhere
// count as the largest before them; only then one thread goes through the sets again.
template <int THREADS>
__device__ __forceinline__ void load_bounds(int2* bounds, const int32_t* offsets, int sets, int slots, int tid) {
  bool descend = false;
  for (int e = tid; e < sets; e += THREADS) {
    const int lo = min(max(__ldcg(offsets + e), 0), slots), hi = min(max(__ldcg(offsets + e + 1), 0), slots);
    bounds[e] = make_int2(lo, hi);
    descend |= hi < lo;
  }
  if (!__syncthreads_or(descend)) return;
  if (tid == 0)
    for (int e = 0, most = 0; e < sets; ++e) {
      const int lo = max(most, bounds[e].x);
      most = max(lo, bounds[e].y);
      bounds[e] = make_int2(lo, most);
    }
  __syncthreads();
}
// Prefix sums of value(0 .. n - 1) into first[0 .. n], the sum in first[n], by one whole warp: a lane takes neighbours. (32 at a time with a
// carry, 256 experts at one token 12.1 us instead of 11.7.)
template <class F>
__device__ __forceinline__ void prefix_sums(int* first, int n, int lane, F value) {
  const int per = (n + 31) / 32, i0 = min(lane * per, n), i1 = min(i0 + per, n);
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += value(i);
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += v;
  }
  int run = upto - mine;
  for (int i = i0; i < i1; ++i) {
    const int v = value(i);
    first[i] = run;
    run += v;
  }
  if (lane == 31) first[n] = run;
}
// The set of unit u, from set e on: the last whose first unit is not behind u. By halves, since every step waits for
// shared memory and most sets may be empty: one token, 8 of 256 experts of 2048 x 1024, 16.8 -> 9.4 us.
__device__ __forceinline__ int set_of(int u, int e, const int* first, int sets) {
  if (u < first[e + 1]) return e;
  for (int last = sets - 1; e < last;) {
    const int mid = (e + last + 1) >> 1;
    if (first[mid] <= u)
      e = mid;
    else
      last = mid - 1;
  }
  return e;
}
#endif

// CTAs that share a tile's range of k: as many as there are clusters of for every tile at once. That goes by what a B200 of 148 SMs runs (`room`, by the
// cluster's CTAs, as cudaOccupancyMaxActiveClusters answers there), not by what this device's GPCs happen to fit, so that a row has the same bits on
// every GPU; the device's own answer (`runs`) only rules out clusters that it cannot run at all.
inline int splits_at_once(int tiles, int most, const int* room, const int* runs) {
  int splits = 1;
  for (int n = 2; n <= most; ++n)
    if (tiles <= room[n] && runs[n] >= 1) splits = n;
  return splits;
}

inline bool ranges_apart(const void* a, size_t an, const void* b, size_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x + an <= y || y + bn <= x;
}

constexpr int kMaxSets = 512;  // experts of a container: their bounds are kept in shared memory

}  // namespace w4a16
