// Linear layers over ragged sets of few tokens, for sm_100a: y[p] = bf16(act(x[row of p] W_e^T + bias_e) + residual[p]).
// The dense layer with an epilogue (one set) and the products grouped by expert; int4 weights, groups of 128.
//
// Mathematics: W = bf16((q - z) s), the value w4a16_dequant_rows gives, made in registers with packed bf16 arithmetic (every
// step but the last exact) and multiplied by the bf16 activations on the tensor cores with fp32 sums, whatever the number of tokens.
//
// A unit of work is a 128-row tile of a set's weights with up to NT of its tokens (NT = 8 or 16). A CTA takes a unit; where there are
// few units, a cluster of S CTAs shares one, each a range of k groups, and adds up through distributed shared memory in a
// fixed order (bitwise reproducible). In a CTA
//   * one producer warp fills a ring of stages, two k groups each: the two 8576-byte weight blocks by one bulk copy (cp.async.bulk), each
//     token's 256 activations by another, so that rows are gathered in the load;
//   * one warp makes what the expansion needs of every row and group (zero point and scale as bf16 pairs) once per stage;
//   * eight consumer warps take 32 rows x 64 k each: mma.sync m16n8k16 with the weights as the A operand straight from the
//     expansion. The fragments' k order is free as long as both operands share it, so a lane takes 16 consecutive k of
//     its row (8 bytes of codes) and of its token (two 16-byte loads). Two warps share 32 rows and add up their halves of K.
//
// What bounds it: the expansion, and what its warps wait for in between. Two CTAs of an SM take 520 to 580 cycles for a weight block in long rows (and
// 660 where a unit has eight blocks, its end among them), where HBM allows 370. Its 1310 warp instructions at M = 8, of which LOP3, shifts and packed bf16
// arithmetic issue at half a scheduler's rate, take 345 cycles by themselves, 408 with the mma.sync; issue slots 56 to 60 % busy, no pipe above
// 46 %. 34816 x 5120 at M = 8 24.2 us (3.8 TB/s), 64 experts 5120 x 1024 at 4.1 slots each 50.3 (3.5 TB/s), start and end of the launch included.
// Tried beside it, the same or slower: 16 rows x 128 k per warp, three CTAs per SM, loads a step ahead, more accumulators, and A in tensor memory for
// tcgen05.mma with two CTAs per SM (28.5 us at M = 1 against 25).
#include <climits>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "ragged.cuh"

namespace w4a16 {
namespace {

constexpr int kRCons = 8;                        // consumer warps
constexpr int kRThreads = (kRCons + 2) * 32;     // and a producer and a warp that prepares the rows' constants
constexpr int kRMaxDepth = 8;                    // ring stages at most
constexpr int kRMaxSplit = 8;                    // CTAs that share a unit at most: the portable cluster size
constexpr int kRGroups = 2;                      // k groups of a stage
constexpr int kXPitch = kRGroups * 256 + 16;     // bytes of a token's activations in a stage: 16 more than they are, against bank conflicts
constexpr uint32_t kRSpin = 1u << 20;

template <int N>
using Const = std::integral_constant<int, N>;

struct RaggedParams {
  RaggedCall c;
  int row_tiles, splits, depth;
  int* status;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Where unit u of the launch lies: set, first slot, tokens, row tile. The chunks of one row tile are neighbours, so that its
// weights come from HBM once. `e` moves on only (a CTA's units ascend).
struct Unit {
  int e, slot0, n, rt;
};
template <int NT>
__device__ __forceinline__ Unit unit_of(int u, int& e, const int* first, const int2* bounds, int sets) {
  e = set_of(u, e, first, sets);
  const int n = bounds[e].y - bounds[e].x, chunks = (n + NT - 1) / NT, at = u - first[e];
  Unit t;
  t.e = e;
  t.rt = at / chunks;
  const int c = at - t.rt * chunks;
  t.slot0 = bounds[e].x + c * NT;
  t.n = min(NT, n - c * NT);
  return t;
}

// A stage: the groups' weight blocks, the tokens' activations, then what the expansion needs of every row and group (16 bytes
// each) and a word that says whether some scale is large.
template <int NT>
__host__ __device__ constexpr int consts_offset() {
  return kRGroups * kTileGroupBytes + NT * kXPitch;
}
template <int NT>
__host__ __device__ constexpr int large_offset() {
  return consts_offset<NT>() + kRGroups * kTileRows * 16;
}
template <int NT>
__host__ __device__ constexpr int stage_bytes() {
  return large_offset<NT>() + 16;
}
template <int NT>
__host__ __device__ constexpr int sum_bytes() {  // the two k halves' sums, [2][NT tokens][128 rows] floats, or one half's of two units
  return 2 * NT * kTileRows * 4;
}

// bf16((q - z) s) of a word's eight weights, pairs of k, from a row's constants {128 + z, s, -z / 4, 4 s} (bf16 pairs). Nibbles 0 and 4
// become (128 + q) - (128 + z) by one OR and a subtraction, exactly; nibbles 1 and 5 stay where they are: as a bf16 pair
// w & 0x00F000F0 is q 2^-129, so one FMA makes (q - z) / 4 of it, exactly too, and 4 s is exact unless s is 2^126 or more: then
// every nibble is shifted down. The product rounds once in either form.
template <bool LARGE>
__device__ __forceinline__ void expand_word(uint32_t word, const uint4& c, uint32_t (&a)[4]) {
  const uint32_t w8 = word >> 8;
  a[0] = mul_bf16x2(sub_bf16x2(and_or(word, 0x000F000Fu, 0x43004300u), c.x), c.y);
  a[2] = mul_bf16x2(sub_bf16x2(and_or(w8, 0x000F000Fu, 0x43004300u), c.x), c.y);
  if constexpr (LARGE) {
    a[1] = mul_bf16x2(sub_bf16x2(and_or(word >> 4, 0x000F000Fu, 0x43004300u), c.x), c.y);
    a[3] = mul_bf16x2(sub_bf16x2(and_or(w8 >> 4, 0x000F000Fu, 0x43004300u), c.x), c.y);
  } else {
    a[1] = mul_bf16x2(fma_bf16x2(word & 0x00F000F0u, 0x7F007F00u, c.z), c.w);
    a[3] = mul_bf16x2(fma_bf16x2(w8 & 0x00F000F0u, 0x7F007F00u, c.z), c.w);
  }
}

// A warp's 32 rows x 64 k of group I of a stage times the tokens: the lane's rows r0, + 8, + 16, + 24, 16 consecutive k of each.
template <int NT, int I, bool LARGE>
__device__ __forceinline__ void multiply_group(float (&acc)[2][NT / 8][4], uint32_t w_at, uint32_t w_last, uint32_t c_at, uint32_t x_at, int n) {
  constexpr int W = I * kTileGroupBytes, X = I * 256, C = I * kTileRows * 16;
  const uint2 w[4] = {lds64<W>(w_at), lds64<W + 128>(w_at), lds64<W + 256>(w_at), lds64<W>(w_last)};
  const uint4 c[4] = {lds128<C>(c_at), lds128<C + 128>(c_at), lds128<C + 256>(c_at), lds128<C + 384>(c_at)};
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // 8 of the lane's 16 k: one word of codes, one 16-byte load per token
    uint32_t a[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) expand_word<LARGE>(h ? w[i].y : w[i].x, c[i], a[i]);
    auto tokens8 = [&](auto at) {
      constexpr int j = decltype(at)::value;
      const uint4 b = h ? lds128<X + 8 * j * kXPitch + 16>(x_at) : lds128<X + 8 * j * kXPitch>(x_at);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        mma_bf16(acc[m][j], a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b.x, b.y);
        mma_bf16(acc[m][j], a[2 * m][2], a[2 * m + 1][2], a[2 * m][3], a[2 * m + 1][3], b.z, b.w);
      }
    };
    tokens8(Const<0>());
    if constexpr (NT > 8)
      if (n > 8) tokens8(Const<1>());
  }
}
template <int NT, bool LARGE>
__device__ __forceinline__ void multiply_stage(float (&acc)[2][NT / 8][4], uint32_t w_at, uint32_t w_last, uint32_t c_at, uint32_t x_at, int n, bool two) {
  multiply_group<NT, 0, LARGE>(acc, w_at, w_last, c_at, x_at, n);
  if (two) multiply_group<NT, 1, LARGE>(acc, w_at, w_last, c_at, x_at, n);
}

template <int NT>
__global__ void __launch_bounds__(kRThreads, 2) k_ragged(const __grid_constant__ RaggedParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const RaggedCall& c = p.c;
  float* sums = reinterpret_cast<float*>(smem);
  uint8_t* ring = smem + sum_bytes<NT>();
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + p.depth * stage_bytes<NT>());
  int2* bounds = reinterpret_cast<int2*>(bars + 3 * kRMaxDepth);
  int* first = reinterpret_cast<int*>(bounds + c.sets);  // [sets + 1] units in front of each set

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int S = p.splits, split = S > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int cluster = blockIdx.x / S, nclusters = gridDim.x / S;
  const uint32_t ring_a = smem_u32(ring), full_a = smem_u32(bars), empty_a = full_a + kRMaxDepth * 8, ready_a = empty_a + kRMaxDepth * 8;
  if (tid == 0) {
    for (int i = 0; i < p.depth; ++i) {
      mbar_init(full_a + i * 8, 1);
      mbar_init(empty_a + i * 8, kRCons);
      mbar_init(ready_a + i * 8, 1);
    }
    fence_mbar_init();
  }
  pdl_launch_dependents();
  if (c.offsets) pdl_wait();  // offsets, and with them everything else, come from the kernels in front
  // units of every set: ceil(tokens / NT) chunks of each row tile
  if (c.offsets) {
    load_bounds<kRThreads>(bounds, c.offsets, c.sets, c.slots, tid);
    if (warp == 0) prefix_sums(first, c.sets, lane, [&](int e) { return (bounds[e].y - bounds[e].x + NT - 1) / NT * p.row_tiles; });
  } else if (tid == 0) {
    bounds[0] = make_int2(0, c.slots);
    first[0] = 0;
    first[1] = (c.slots + NT - 1) / NT * p.row_tiles;
  }
  __syncthreads();
  const int units = first[c.sets];
  const int g0 = c.G * split / S, g1 = c.G * (split + 1) / S;
  bool dead = false;
  int e = 0, st = 0;

  if (warp == kRCons) {
    // ================================================================ producer
    uint32_t ph = 1;
    int issued = 0;
    for (int u = cluster; !dead && u < units; u += nclusters) {
      const Unit t = unit_of<NT>(u, e, first, bounds, c.sets);
      const uint8_t* src = c.stream + static_cast<size_t>(t.e) * c.set_bytes + (static_cast<size_t>(t.rt) * c.G + g0) * kTileGroupBytes;
      // The ring is empty for the first unit: its first stages' weights are on their way before the tokens' rows are known, and, where
      // they do not depend on the kernel in front (one set), before that has ended.
      int early = 0;
      if (u == cluster) {
        early = min(p.depth, (g1 - g0 + kRGroups - 1) / kRGroups);
        if (lane == 0)
          for (int i = 0; i < early; ++i) {
            const uint32_t ng = min(kRGroups, g1 - g0 - i * kRGroups);
            mbar_expect_tx(full_a + i * 8, ng * (kTileGroupBytes + t.n * kGroup * 2));
            bulk_g2s(ring_a + i * stage_bytes<NT>(), src + i * kRGroups * kTileGroupBytes, ng * kTileGroupBytes, full_a + i * 8);
          }
        __syncwarp();
        if (!c.offsets) pdl_wait();
      }
      int row = t.slot0 + min(lane, t.n - 1);
      if (c.x_rows) row = __ldcg(c.x_rows + row);
      row = min(max(row, 0), c.x_tokens - 1);  // (no read outside x, whatever the rows hold)
      const uint16_t* xr = c.x + static_cast<size_t>(row) * c.K + static_cast<size_t>(g0) * kGroup;
      for (int g = g0; g < g1; g += kRGroups, src += kRGroups * kTileGroupBytes, xr += kRGroups * kGroup) {
        const uint32_t dst = ring_a + st * stage_bytes<NT>(), ng = min(kRGroups, g1 - g);
        if (--early < 0) {
          if (!warp_agrees(mbar_wait_bounded_relaxed(empty_a + st * 8, ph, kRSpin))) {
            dead = true;
            break;
          }
          if (lane == 0) {
            mbar_expect_tx(full_a + st * 8, ng * (kTileGroupBytes + t.n * kGroup * 2));
            bulk_g2s(dst, src, ng * kTileGroupBytes, full_a + st * 8);
          }
          __syncwarp();
        }
        if (lane < t.n) bulk_g2s(dst + kRGroups * kTileGroupBytes + lane * kXPitch, xr, ng * kGroup * 2, full_a + st * 8);
        ++issued;
        if (++st == p.depth) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    if (dead) {  // the copies in flight still have to land
      if (lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
      for (int i = 0; i < p.depth && i < issued; ++i) mbar_wait_bounded_relaxed(full_a + i * 8, i < st ? ph ^ 1u : ph, 1u << 10);
    }
    __syncwarp();
    if (S > 1) {
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  if (warp == kRCons + 1) {
    // ================================================================ the rows' constants
    // All lanes of a row need the same ones: made once, read by one 16-byte load in place of eight small loads and eight permutes per lane
    // and group (170 of 1630 warp instructions per weight block, two chunks of tokens).
    uint32_t ph = 0;
    for (int u = cluster; !dead && u < units; u += nclusters) {
      for (int g = g0; g < g1; g += kRGroups) {
        if (!warp_agrees(mbar_wait_bounded(full_a + st * 8, ph, kRSpin))) {
          dead = true;
          break;
        }
        const uint32_t blk = ring_a + st * stage_bytes<NT>();
        bool large = false;
#pragma unroll
        for (int i = 0; i < kRGroups; ++i) {  // (an odd last group's neighbour is whatever the stage held before)
          const uint32_t at = blk + i * kTileGroupBytes, to = blk + consts_offset<NT>() + i * kTileRows * 16 + lane * 16;
          const uint32_t sc[4] = {lds_u16<kTgScaleOff>(at + lane * 2), lds_u16<kTgScaleOff + 64>(at + lane * 2),
                                  lds_u16<kTgScaleOff + 128>(at + lane * 2), lds_u16<kTgScaleOff + 192>(at + lane * 2)};
          const uint32_t zp[4] = {lds_u8<kTgZpOff>(at + lane), lds_u8<kTgZpOff + 32>(at + lane), lds_u8<kTgZpOff + 64>(at + lane),
                                  lds_u8<kTgZpOff + 96>(at + lane)};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t z = __byte_perm(zp[r], 0x43434343u, 0x4040), s2 = __byte_perm(sc[r], 0, 0x1010);  // (128 + z, 128 + z), (s, s)
            sts128(to + r * 512, z, s2, fma_bf16x2(z, 0xBE80BE80u, 0x42004200u), mul_bf16x2(s2, 0x40804080u));  // -z / 4, 4 s
            large |= (sc[r] & 0x7FFFu) - 0x7E80u < 0x100u;
          }
        }
        large = __any_sync(0xffffffffu, large);
        if (lane == 0) sts32(blk + large_offset<NT>(), large);
        __syncwarp();
        if (lane == 0) mbar_arrive(ready_a + st * 8);
        if (++st == p.depth) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    if (dead && lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
    __syncwarp();
    if (S > 1) {
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  // ================================================================ consumers
  const int half = warp & 1, r0 = (warp >> 1) * 32 + (lane >> 2), t4 = lane & 3;
  const int chunk = 2 * half + (t4 >> 1);
  // Offsets of the lane's codes in a stage: rows r0, + 8, + 16 lie 128 bytes apart, the last may wrap round (weight_slot)
  const uint32_t w_off = chunk * kChunkBytes + (t4 & 1) * 8 + weight_slot(r0, chunk) * 16;
  const uint32_t w_last = chunk * kChunkBytes + (t4 & 1) * 8 + weight_slot(r0 + 24, chunk) * 16;
  const uint32_t c_off = consts_offset<NT>() + r0 * 16;
  const uint32_t x_off = kRGroups * kTileGroupBytes + (lane >> 2) * kXPitch + (half * 64 + t4 * 16) * 2;
  uint32_t ph = 0;
  int parity = 0;
  for (int u = cluster; u < units; u += nclusters) {
    const Unit t = unit_of<NT>(u, e, first, bounds, c.sets);
    float acc[2][NT / 8][4] = {};
    for (int g = g0; g < g1 && !dead; g += kRGroups) {
      if (!warp_agrees(mbar_wait_bounded(ready_a + st * 8, ph, kRSpin))) {  // (behind the weights' and activations' arrival)
        dead = true;
        break;
      }
      const uint32_t blk = ring_a + st * stage_bytes<NT>();
      if (lds32(blk + large_offset<NT>()) == 0)
        multiply_stage<NT, false>(acc, blk + w_off, blk + w_last, blk + c_off, blk + x_off, t.n, g + 1 < g1);
      else
        multiply_stage<NT, true>(acc, blk + w_off, blk + w_last, blk + c_off, blk + x_off, t.n, g + 1 < g1);
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_a + st * 8);
      if (++st == p.depth) {
        st = 0;
        ph ^= 1;
      }
    }
    if (!c.offsets) pdl_wait();  // bias and residual, and y's readers, may be in the kernel in front
    // ---- the halves' (and the splits') sums are added up in one order, and every output is finished by one thread
    const bool gated = c.act == W4A16_ACT_SWIGLU;
    struct Beside {
      float b0, b1, r0, r1;
    };
    auto beside = [&](int tok, int r) {  // bias and residual of rows r and r + 1 of the tile, r even
      const int row = t.rt * kTileRows + r;
      Beside v = {};
      if (row >= c.N || tok >= t.n) return v;
      if (c.bias) {
        const uint16_t* b = c.bias + static_cast<size_t>(t.e) * c.N;
        v.b0 = bf16_bits_to_float(b[bias_index(row, c.N, c.act)]);
        v.b1 = bf16_bits_to_float(b[bias_index(row + 1, c.N, c.act)]);
      }
      if (c.residual) {
        const uint16_t* at = c.residual + static_cast<size_t>(t.slot0 + tok) * c.ny + (gated ? row >> 1 : row);
        const uint32_t r2 = gated ? *at : *reinterpret_cast<const uint32_t*>(at);
        v.r0 = bf16_bits_to_float(static_cast<uint16_t>(r2));
        v.r1 = bf16_bits_to_float(static_cast<uint16_t>(r2 >> 16));
      }
      return v;
    };
    auto finish = [&](int tok, int r, float v0, float v1, const Beside& v) {
      const int row = t.rt * kTileRows + r;
      if (row >= c.N || tok >= t.n) return;
      v0 += v.b0;
      v1 += v.b1;
      uint16_t* at = c.y + static_cast<size_t>(t.slot0 + tok) * c.ny + (gated ? row >> 1 : row);
      if (gated)
        *at = float_to_bf16_bits(logistic_times(v0, v0) * v1 + v.r0);
      else
        *reinterpret_cast<uint32_t*>(at) = float_to_bf16_bits(activate(v0, c.act) + v.r0) |
                                           (static_cast<uint32_t>(float_to_bf16_bits(activate(v1, c.act) + v.r1)) << 16);
    };
    if (S == 1) {
      // Two warps share 32 rows. Each hands the other its fragments of 16 and finishes the other 16, through two buffers in turn, so that a
      // unit needs a single barrier of the two (a buffer is written again behind the next unit's).
      const uint32_t pair_a = smem_u32(sums) + ((parity * (kRCons / 2) + (warp >> 1)) * (NT / 4) * 32 + lane) * 16;
      const uint32_t give = pair_a + half * (NT / 8) * 512, take = pair_a + (half ^ 1) * (NT / 8) * 512;
      parity ^= 1;
#pragma unroll
      for (int j = 0; j < NT / 8; ++j)
        if (j == 0 || 8 * j < t.n)
          sts128(give + j * 512, __float_as_uint(half ? acc[0][j][0] : acc[1][j][0]), __float_as_uint(half ? acc[0][j][1] : acc[1][j][1]),
                 __float_as_uint(half ? acc[0][j][2] : acc[1][j][2]), __float_as_uint(half ? acc[0][j][3] : acc[1][j][3]));
      const int odd = (lane >> 2) & 1, tok0 = 2 * t4 + odd, row0 = r0 - odd + 16 * half;
      const Beside early[2] = {beside(tok0, row0), beside(tok0, row0 + 8)};  // under way while the warps meet
      named_bar_sync(1 + (warp >> 1), 64);
      if (dead) continue;
#pragma unroll
      for (int j = 0; j < NT / 8; ++j)
        if (j == 0 || 8 * j < t.n) {
          const uint4 u = j ? lds128<512>(take) : lds128<0>(take);
          const float v[4] = {(half ? acc[1][j][0] : acc[0][j][0]) + __uint_as_float(u.x), (half ? acc[1][j][1] : acc[0][j][1]) + __uint_as_float(u.y),
                              (half ? acc[1][j][2] : acc[0][j][2]) + __uint_as_float(u.z), (half ? acc[1][j][3] : acc[0][j][3]) + __uint_as_float(u.w)};
          // a lane has one row and two tokens; it takes its neighbour row's sum of one token for its own of the other
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v[2 * h] : v[2 * h + 1], 4);
            finish(8 * j + tok0, row0 + 8 * h, odd ? got : v[2 * h], odd ? v[2 * h + 1] : got, j ? beside(8 * j + tok0, row0 + 8 * h) : early[h]);
          }
        }
      continue;
    }
#pragma unroll
    for (int j = 0; j < NT / 8; ++j)
      if (j == 0 || 8 * j < t.n)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sums[(half * NT + 8 * j + 2 * t4 + (i & 1)) * kTileRows + r0 + 16 * m + 8 * (i >> 1)] = acc[m][j][i];
    const int pairs = t.n * (kTileRows / 2), i0 = tid + split * kRCons * 32;
    Beside next = beside(i0 / (kTileRows / 2), 2 * (i0 % (kTileRows / 2)));  // under way while the splits meet
    cluster_sync();
    for (int i = i0; i < pairs && !dead; i += S * kRCons * 32) {
      const int tok = i / (kTileRows / 2), r = 2 * (i % (kTileRows / 2));
      float2 v[kRMaxSplit][2];  // every split's loads are in flight together
#pragma unroll
      for (int s = 0; s < kRMaxSplit; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (s < S) v[s][h] = ld_cluster_f32x2(map_to_rank(smem_u32(sums + (h * NT + tok) * kTileRows + r), s));
      float v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int s = 0; s < kRMaxSplit; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (s < S) {
            v0 += v[s][h].x;
            v1 += v[s][h].y;
          }
      finish(tok, r, v0, v1, next);
      const int in = i + S * kRCons * 32;
      if (in < pairs) next = beside(in / (kTileRows / 2), 2 * (in % (kTileRows / 2)));
    }
    break;  // (a cluster takes one unit)
  }
  if (dead && lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
  __syncwarp();
  if (S > 1) {
    if (cluster >= units) cluster_sync();
    cluster_sync();  // nobody leaves while its sums may still be read
  }
}

template <int NT>
int fixed_bytes(int sets) {
  return sum_bytes<NT>() + 3 * kRMaxDepth * 8 + sets * 8 + (sets + 1) * 4;
}
// How many clusters of n CTAs the device runs at once, index n; asked for once per device, with the largest shared memory that
// leaves two CTAs per SM. The kernel's shared-memory attribute is set on the way.
template <int NT>
const int* clusters_at_once(const DeviceInfo* di) {
  struct Fit {
    bool ready = false;
    int n[kRMaxSplit + 1] = {};
  };
  static std::mutex mu;
  static Fit all[64];
  std::lock_guard<std::mutex> lk(mu);
  Fit& f = all[di->device & 63];
  if (!f.ready) {
    cudaError_t e = cudaFuncSetAttribute(k_ragged<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, di->smem_optin);
    for (int n = 1; n <= kRMaxSplit && e == cudaSuccess; ++n) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1];
      cfg.gridDim = dim3(n);
      cfg.blockDim = dim3(kRThreads);
      cfg.dynamicSmemBytes = di->smem_per_sm / 2 - di->smem_reserved;
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = n;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&f.n[n], k_ragged<NT>, &cfg);
    }
    if (e != cudaSuccess || f.n[1] < 1) {
      fail(W4A16_ECUDA, "linear: the device runs no CTA of the kernel (%s)", cudaGetErrorString(e));
      return nullptr;
    }
    f.ready = true;
  }
  return f.n;
}

template <int NT>
int launch_ragged(RaggedParams& p, const DeviceInfo* di, int max_units, cudaStream_t st) {
  const int fixed = fixed_bytes<NT>(p.c.sets);
  const int room = (di->smem_per_sm / 2 - di->smem_reserved - fixed) / stage_bytes<NT>();
  p.depth = room < kRMaxDepth ? room : kRMaxDepth;
  const int smem = fixed + p.depth * stage_bytes<NT>();
  // Few units: as many CTAs share one as there are clusters for at once. (One more, and a last cluster starts when a first one ends:
  // 5120 x 6144 at M = 1, 40 units: six 9.2 us, seven - of which 37 fit - 13.7; 5120 x 17408 17.6 and 24.0.)
  constexpr int kRoom[kRMaxSplit + 1] = {0, 296, 148, 93, 71, 56, 45, 37, 33};
  const int* fit = clusters_at_once<NT>(di);
  if (!fit) return W4A16_ECUDA;
  const int slots = fit[1], most = p.c.G / kRGroups < kRMaxSplit ? p.c.G / kRGroups : kRMaxSplit;
  const int S = splits_at_once(max_units, most, kRoom, fit);
  p.splits = S;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3(p.splits > 1 ? p.splits * max_units : (max_units < slots ? max_units : slots));
  cfg.blockDim = dim3(kRThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 0;
  if (p.splits > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.splits;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  // (behind a weight write the launch of one set is fully ordered: its weights are read before the wait)
  const bool behind_write = p.c.offsets == nullptr && take_weight_write(st);
  if (!behind_write && pdl_enabled()) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t err = cudaLaunchKernelEx(&cfg, k_ragged<NT>, p);
  if (err == cudaSuccess) return W4A16_OK;
  if (behind_write) note_weight_write(st);
  return fail(W4A16_ECUDA, "linear: launch: %s", cudaGetErrorString(err));
}

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

// Checks what both entry points share and enqueues the call.
int run_ragged(RaggedCall& c, const char* who, cudaStream_t st) {
  W4_REQUIRE(c.act >= W4A16_ACT_NONE && c.act <= W4A16_ACT_SWIGLU, "%s: unknown activation %d", who, c.act);
  W4_REQUIRE(c.act != W4A16_ACT_SWIGLU || c.N % 32 == 0, "%s: out_f %d must be a multiple of 32 (gate, up interleaved)", who, c.N);
  if (c.slots == 0) return W4A16_OK;
  W4_REQUIRE(c.x != nullptr && c.y != nullptr && c.x_tokens > 0, "%s: null or empty matrix", who);
  W4_REQUIRE(aligned16(c.x) && aligned16(c.y) && aligned16(c.residual), "%s: x, y and residual must be 16-byte aligned", who);
  W4_REQUIRE((reinterpret_cast<uintptr_t>(c.bias) & 1) == 0, "%s: bias not 2-byte aligned", who);
  W4_REQUIRE(((reinterpret_cast<uintptr_t>(c.offsets) | reinterpret_cast<uintptr_t>(c.x_rows)) & 3) == 0,
             "%s: offsets or x_rows not 4-byte aligned", who);
  c.ny = c.act == W4A16_ACT_SWIGLU ? c.N / 2 : c.N;
  const size_t xb = static_cast<size_t>(c.x_tokens) * c.K * 2, yb = static_cast<size_t>(c.slots) * c.ny * 2;
  W4_REQUIRE(ranges_apart(c.x, xb, c.y, yb), "%s: y overlaps x", who);
  W4_REQUIRE(c.residual == nullptr || c.residual == c.y || ranges_apart(c.residual, yb, c.y, yb), "%s: residual overlaps y but is not y", who);
  W4_REQUIRE(c.bias == nullptr || ranges_apart(c.bias, static_cast<size_t>(c.sets) * c.N * 2, c.y, yb), "%s: y overlaps bias", who);
  W4_REQUIRE(ranges_apart(c.offsets, c.offsets ? static_cast<size_t>(c.sets + 1) * 4 : 0, c.y, yb) &&
                 ranges_apart(c.x_rows, c.x_rows ? static_cast<size_t>(c.slots) * 4 : 0, c.y, yb),
             "%s: y overlaps offsets or x_rows", who);
  const DeviceInfo* di = device_info();
  if (!di) return W4A16_ECUDA;
  RaggedParams p = {};
  p.c = c;
  p.row_tiles = (c.N + kTileRows - 1) / kTileRows;
  p.status = di->status;
  // More than a few tokens per set: whole tiles on tcgen05, whose time hardly depends on their number up to 128 (here every eight
  // tokens cost 64 mma.sync per weight block, beside 1040 instructions for its expansion), but which cost more at both ends, so that
  // short rows of weights stay here longer. us, here / there: 34816 x 5120 at M = 8 24.8 / 27.9, at 16 30.0 / 28.3; 16384 x 5120 at 16 20.1 / 16.3; 2048 x 5120 in 64 sets of 4.1 in
  // the mean 87.6 / 97.2, of 5 102 / 97, of 6.5 107 / 99; 2048 x 2048 in 256 of 5.6 145 / 149, of 6.5 152 / 151, of 7.5 163 / 156; 5120 x 1024 in 64
  // of 5 56.5 / 61.1, of 6.5 62.6 / 62.8, of 8.5 66.6 / 63.5.
  if (c.offsets ? 2LL * c.slots > (c.G >= 32 ? 9LL : 13LL) * c.sets : c.slots > 8) return launch_prefill_ragged(c, st);
  // chunks of NT tokens at most: every set with tokens has one more than its whole ones
  const int used = c.slots < c.sets ? c.slots : c.sets;
  const int nt = c.slots <= 4LL * c.sets || !c.offsets ? 8 : 16;
  const long long units = static_cast<long long>(c.offsets ? used + (c.slots - used) / nt : 1) * p.row_tiles;
  W4_REQUIRE(units <= INT_MAX, "%s: %d slots x %d rows are too many for one call", who, c.slots, c.N);
  const int max_units = static_cast<int>(units);
  return nt == 8 ? launch_ragged<8>(p, di, max_units, st) : launch_ragged<16>(p, di, max_units, st);
}

int check_experts(const w4a16_experts_t* w) {
  W4_REQUIRE(w != nullptr && w->qweight != nullptr && aligned16(w->qweight), "experts: null or misaligned weights");
  W4_REQUIRE(w->group_size == kGroup && w->in_f > 0 && w->in_f % kGroup == 0 && w->num_groups == w->in_f / kGroup,
             "experts: in_f %d, group_size %d, %d groups", w->in_f, w->group_size, w->num_groups);
  W4_REQUIRE(w->out_f > 0 && w->out_f % kRowGranule == 0, "experts: out_f %d not a positive multiple of 16", w->out_f);
  W4_REQUIRE(w->num_experts >= 1 && w->num_experts <= kMaxSets, "experts: %d experts (1..%d)", w->num_experts, kMaxSets);
  return W4A16_OK;
}

}  // namespace
}  // namespace w4a16

using namespace w4a16;

extern "C" {

int w4a16_linear_epilogue(uint16_t* y, const w4a16_weights_t* w, const uint16_t* x, int M, const uint16_t* bias, int activation,
                          const uint16_t* residual, void* stream) {
  if (int rc = check_weights(w)) return rc;
  W4_REQUIRE(M >= 0, "linear_epilogue: M = %d", M);
  RaggedCall c = {};
  c.stream = reinterpret_cast<const uint8_t*>(w->qweight);
  c.sets = 1;
  c.N = w->out_f;
  c.K = w->in_f;
  c.G = w->num_groups;
  c.x = x;
  c.x_tokens = M;
  c.slots = M;
  c.bias = bias;
  c.act = activation;
  c.residual = residual;
  c.y = y;
  return run_ragged(c, "linear_epilogue", static_cast<cudaStream_t>(stream));
}

int w4a16_experts_alloc(w4a16_experts_t* w, int num_experts, int out_f, int in_f, int group_size, void* stream) {
  W4_REQUIRE(w != nullptr, "experts_alloc: null struct");
  w4a16_experts_t d = {};
  d.qweight = reinterpret_cast<uint32_t*>(16);  // (for the check; replaced below)
  d.num_experts = num_experts;
  d.out_f = out_f;
  d.in_f = in_f;
  d.group_size = group_size;
  d.num_groups = group_size > 0 ? in_f / group_size : 0;
  memset(w, 0, sizeof *w);
  if (int rc = check_experts(&d)) return rc;
  const size_t bytes = stream_bytes(out_f, d.num_groups) * num_experts;
  void* q = nullptr;
  cudaError_t e = cudaMalloc(&q, bytes);
  if (e == cudaSuccess && out_f % kTileRows != 0) {
    // rows past out_f in every expert's last tile: zero scales (see w4a16_weights_alloc)
    e = cudaMemsetAsync(q, 0, bytes, static_cast<cudaStream_t>(stream));
    note_weight_write(static_cast<cudaStream_t>(stream));
  }
  if (e != cudaSuccess) {
    cudaFree(q);
    return fail(W4A16_ECUDA, "experts_alloc(%d x %d x %d): %s", num_experts, out_f, in_f, cudaGetErrorString(e));
  }
  d.qweight = static_cast<uint32_t*>(q);
  *w = d;
  return W4A16_OK;
}

int w4a16_experts_view(const w4a16_experts_t* w, int expert, w4a16_weights_t* view) {
  if (int rc = check_experts(w)) return rc;
  W4_REQUIRE(view != nullptr, "experts_view: null struct");
  W4_REQUIRE(expert >= 0 && expert < w->num_experts, "experts_view: expert %d of %d", expert, w->num_experts);
  uint8_t* q = reinterpret_cast<uint8_t*>(w->qweight) + stream_bytes(w->out_f, w->num_groups) * expert;
  view->qweight = reinterpret_cast<uint32_t*>(q);
  view->scale = reinterpret_cast<uint16_t*>(q);  // nothing is read through these two; w4a16_weights_free knows a view by them
  view->zp = q;
  view->out_f = w->out_f;
  view->in_f = w->in_f;
  view->group_size = w->group_size;
  view->num_groups = w->num_groups;
  return W4A16_OK;
}

int w4a16_experts_free(w4a16_experts_t* w) {
  W4_REQUIRE(w != nullptr, "experts_free: null struct");
  cudaFree(w->qweight);
  memset(w, 0, sizeof *w);
  return W4A16_OK;
}

int w4a16_experts_linear(uint16_t* y, const w4a16_experts_t* w, const uint16_t* x, int x_tokens, const int32_t* x_rows,
                         const int32_t* offsets, int slots, const uint16_t* bias, int activation, void* stream) {
  if (int rc = check_experts(w)) return rc;
  W4_REQUIRE(slots >= 0 && x_tokens >= 0, "experts_linear: %d slots, %d tokens", slots, x_tokens);
  W4_REQUIRE(offsets != nullptr, "experts_linear: null offsets");
  W4_REQUIRE(x_rows != nullptr || slots <= x_tokens, "experts_linear: %d slots of %d rows, without x_rows", slots, x_tokens);
  RaggedCall c = {};
  c.stream = reinterpret_cast<const uint8_t*>(w->qweight);
  c.set_bytes = stream_bytes(w->out_f, w->num_groups);
  c.sets = w->num_experts;
  c.N = w->out_f;
  c.K = w->in_f;
  c.G = w->num_groups;
  c.x = x;
  c.x_tokens = x_tokens;
  c.x_rows = x_rows;
  c.offsets = offsets;
  c.slots = slots;
  c.bias = bias;
  c.act = activation;
  c.y = y;
  return run_ragged(c, "experts_linear", static_cast<cudaStream_t>(stream));
}

}  // extern "C"
