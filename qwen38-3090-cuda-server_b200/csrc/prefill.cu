// Prefill W4A16 GEMM for sm_100a:  C[M, out_f] = A[M, in_f] @ W^T  (bf16 in/out, fp32 accumulate)
// with the dequantisation fused into the tensor-core pipeline.
//
// Replaces gemm_w4a16 of the reference (src/kernels/gemm_w4a16.cu:63-88), which expands a
// weight tile to bf16 in a 256 MB workspace (k_dequant_rows) and calls cublasGemmEx. Here no
// bf16 copy of the weights ever touches global or shared memory:
//   * a pair of CTAs (cta_group::2) computes a tile of 256 output rows x TN tokens: each CTA holds the weights
//     and the fp32 accumulator of its own 128 rows in tensor memory and HALF of the tile's tokens in shared
//     memory. A CTA alone (128 rows x 256 tokens) pulls 72 KB through L2 per k group and 1024 tensor
//     cycles; a pair's CTA pulls 41 KB for the same math, which leaves room for four
//     group stages of activations instead of two;
//   * a producer thread per CTA streams the packed int4 blocks of its row tile through a ring of
//     shared-memory stages with 1-D bulk async copies (cp.async.bulk + mbarrier);
//   * sixteen dequant warps per CTA (one output row per thread; four teams take the k groups in
//     turn) turn 64 bytes of nibbles into bf16 weights in registers - (128+q) by LOP3,
//     minus (128+zp) and times the group scale with packed bf16 arithmetic, which is exactly
//     bf16(float(q-zp)*float(s)), the value w4a16_dequant_rows produces - and store them as the A operand
//     into tensor memory (tcgen05.st);
//   * a second producer thread per CTA brings its half of the activation tile in with tiled TMA loads
//     (cp.async.bulk.tensor, 128-byte swizzle), which is the K-major B operand as is; both CTAs' loads
//     complete on the leader's mbarrier;
//   * one thread of the leader CTA issues tcgen05.mma (256 x N x 16, kind::f16) per 16-k slab for both
//     CTAs, and one commit per group tells both CTAs that the A columns and the stage are free;
//   * eight epilogue warps per CTA read the accumulator back with tcgen05.ld into shared memory, hand it back to the
//     issuer, and store C in 256-byte rows while the next tile's main loop runs;
//   * few tiles (short prompts, narrow layers): a cluster of 2 S CTAs splits K S ways; the splits' fp32 tiles
//     are added through distributed shared memory, always in split order (bitwise reproducible).
//
// The same pipeline carries the layers with an epilogue (kDense: bias, activation and residual while the accumulator is read
// out, in fp32) and the products grouped by expert (kSets: every tile belongs to a set of tokens with weights of its own; rows are
// gathered four at a time by TMA). For few tokens a CTA works alone (PAIR = false: 128 rows x all of the tile's tokens).
//
// What bounds it: long prompts run at the tensor cores' rate under the power cap (256 x 256 x 16 per 128 cycles: 1024
// cycles per k group; tensor pipe 87 % active over a 4096-token launch), short ones by no single role: a CTA and k group takes
// 560 to 640 cycles (5120 x 17408 at M = 77, before rows were stored sixteen registers at a time: issue slots 52 %, ALU pipe 41 % on average and 52 %
// on the busiest SM, tensor pipe 43 % of active cycles), where HBM would allow 386.
// In us, weights cold, against one CTA per tile of 128 x 256 with eight dequant warps (by box and temperature: 2 to 10 %):
//   34816 x 5120, M = 4096: 1264 -> 922 (1583 TFLOP/s); 5120 x 17408, M = 4096: 698 -> 488 (1497)
//   34816 x 5120, M = 777:   300 -> 195;                5120 x 8192, M = 777:   110 -> 49
//   34816 x 5120, M = 77:     73 -> 32;                 5120 x 17408, M = 77:   105 -> 20.5;   8192 x 5120, M = 77: 45 -> 13
// and on the way, 34816 x 5120 at M = 4096 on one device: half groups as the unit of every hand-off 1134 (the first shape; the
// issuing thread is the limit), whole groups 1063, two teams of dequant warps (four since) and C through shared memory 890. A warp's vote on
// its waits took another 9 % off short prompts (34816 x 5120 at M = 77: 40.8 -> 37.1) by keeping the loops warp-uniform.
// Programmatic dependent launch (the next launch sets up, streams and expands its first weights as this one's CTAs leave) took
// the four layers of a block from 104.8 to 96.5 us at M = 77 (5120 -> 8192, 6144 -> 5120, MLP) and from 562.5 to 546.7 at M = 777.
#include <cuda.h>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "ragged.cuh"

namespace w4a16 {
namespace {

constexpr int PW = 16;                      // dequant warps: 4 TMEM lane quarters x 4 groups
constexpr int EW = 8;                       // epilogue warps: two per lane quarter, each half of the tokens
constexpr int kWEpi0 = PW, kWWeights = PW + EW, kWIssue = kWWeights + 1, kWActs = kWIssue + 1;
constexpr int kPWarps = kWActs + 1;
constexpr int kPGather = 3;                 // with sets: warps that gather rows, kWActs and the ones behind it
constexpr int kPMaxTN = 256;                // tokens of a tile: a multiple of 32 (the pair's MMA needs N % 32 == 0)
constexpr int kPMaxSplit = 4;               // 2 S <= 8 CTAs: the portable cluster size
constexpr int kPSteps = 4;                  // activation stages, each one k group of the CTA's TN / 2 tokens
constexpr int kPDone = 8;                   // ring of "group multiplied" barriers: at least kPSteps and the A slots
constexpr int kPMaxWD = 16;                 // weight ring stages (one k group each), at most
constexpr uint32_t kPTmemCols = 512;
constexpr uint32_t kPSpin = 1u << 20;
constexpr uint32_t kMagicP = 0x43004300u, kNibMaskP = 0x000F000Fu;
constexpr int kPTeams = 4;                  // teams of dequant warps
constexpr int kPMaxA = 6;                   // A slots, at most
constexpr int kPBars = 2 * kPMaxWD + kPDone + kPMaxA + kPSteps + 2;
// Tensor memory: the accumulator's TN columns, the rest are slots of the A operand, 64 columns per k group.
__host__ __device__ constexpr int a_slots(int tn) { return tn <= 128 ? 6 : 4; }
constexpr int kPSetsTN = 224, kPSetsNarrow = 128;  // tokens of a tile with sets, and with small ones:
constexpr int kPSetsMean = 64;                     // mean set up to which the narrow tile is taken
constexpr int kPSingleTN = 80;                // tokens of a tile of a CTA alone at most
constexpr int kPSingleMean = 24, kPSingleGathered = 10;  // mean set up to which sets take such tiles
static_assert(kPSingleTN <= kPSetsTN / 2, "lists of rows");
static_assert(128 + 6 * 64 <= 512 && 256 + 4 * 64 <= 512 && kPMaxA <= kPDone && kPSteps <= kPDone, "ring depths");

struct PrefillParams {
  CUtensorMap amap;   // A as [M][K] bf16, box 64 k x TN / 2 tokens, 128-byte swizzle, zero fill
  const uint8_t* stream;
  uint16_t* C;        // [M][ldc] bf16; this launch's rows land in columns [col0, col0 + N)
  int M, N, K, G, row_tiles, pairs;  // pairs: row tiles in twos (an odd last one repeats the last tile and stores nothing)
  int tn, splits, wdepth;            // wdepth is a multiple of four: a stage is always read by the same dequant warps
  int full_tt, tiles;                // token tiles of TN tokens; tiles in all (the ragged token tile's come last)
  long long ldc;
  int wide;                          // C (and every peer's) takes 16-byte stores: base, ldc and col0 are multiples of that
  int col0;
  int* status;
  // column-sharded call: the other ranks' C (peer-mapped) receive the same tile, then the completion flag
  int npeers;
  uint16_t* C_peers[8];
  unsigned* comm_local;
  unsigned* comm_peers[8];
  int comm_n, comm_rank;
  // layers with an epilogue and layers of experts
  RaggedCall call;
};

// What an instance of the kernel does: the plain GEMM, a dense layer with bias, activation and residual in its epilogue, or
// the same per set of tokens with its own weights (experts), rows gathered in the load.
constexpr int kPlain = 0, kDense = 1, kSets = 2;
__host__ __device__ constexpr int prefill_warps(int mode) { return mode == kSets ? kPWarps + kPGather - 1 : kPWarps; }

// ---- CTA pairs and clusters --------------------------------------------------------------
// Arrival on a barrier of any CTA of the cluster (a mapped address). What it hands over is tensor memory, ordered by
// the tcgen05 fences around it, so the barrier needs no cluster-scope release (which costs a memory fence).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>  // the pair leader's barrier (a mapped address), or this CTA's own
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar, std::bool_constant<PAIR>) {
  if constexpr (PAIR)
    mbar_arrive_cluster(bar);
  else
    mbar_arrive(bar);
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t smem_dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D[both CTAs' tmem] (+)= A[both CTAs' tmem] * B[half of the columns from each CTA's shared memory]
__device__ __forceinline__ void umma_bf16_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                  uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same for a CTA alone: 128 rows, all of the columns from its own shared memory
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One arrival on the barrier at this offset in every CTA of `mask` once all MMAs issued so far have completed.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar, uint16_t mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(mask)
      : "memory");
}
// Tiled TMA load of a 64 x TN / 2 box (k, token) into this CTA's shared memory; completion on the pair leader's mbarrier.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Four rows of 64 k, each of its own, into 512 consecutive bytes (with the swizzle of their place in a 1024-byte atom).
template <bool PAIR>
__device__ __forceinline__ void tma_gather(uint32_t dst, const CUtensorMap* map, int x, const int4& rows, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(bar)
        : "memory");
}
// K-major operand descriptor for a 128-byte-swizzled tile ([row][128 B], 8-row groups 1024 B apart)
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// A tile: its row pair, first token, the tokens it multiplies (a multiple of 32; the ragged token tile has fewer) and those of
// them that exist; with sets, its set.
struct PTile {
  int pair, tok0, n, toks, set;
};
// tokens are multiplied in steps of 32 by a pair, of 16 by a CTA alone
template <bool PAIR>
__device__ __forceinline__ int mma_tokens(int n) {
  return PAIR ? (n + 31) & ~31 : (n + 15) & ~15;
}
template <bool PAIR>
__device__ __forceinline__ PTile tile_of(const PrefillParams& p, int tile) {
  const int nfull = p.pairs * p.full_tt;
  PTile t;
  if (tile < nfull) {  // token tiles of one row pair are neighbours: its weights stay in L2
    t.pair = tile / p.full_tt;
    t.tok0 = (tile - t.pair * p.full_tt) * p.tn;
    t.n = p.tn;
  } else {
    t.pair = tile - nfull;
    t.tok0 = p.full_tt * p.tn;
    t.n = mma_tokens<PAIR>(p.M - t.tok0);
  }
  t.toks = min(t.n, p.M - t.tok0);
  t.set = 0;
  return t;
}

// Sets: their slots and the tiles in front of each, in shared memory. A set's tokens are cut into equal tiles (a multiple of 32, for a CTA
// alone of 16, and at most TN), which all expand the set's weights.
struct SetTable {
  const int2* bounds;
  const int* first;  // [sets + 1]
};
// A role's walk over the tiles of its cluster; `set` moves on only.
template <int MODE, bool PAIR>
__device__ __forceinline__ PTile walk_tile(const PrefillParams& p, int tile, int& set, const SetTable& tab) {
  if constexpr (MODE != kSets) return tile_of<PAIR>(p, tile);
  set = set_of(tile, set, tab.first, p.call.sets);
  const int2 b = tab.bounds[set];
  const int n = b.y - b.x, tt = (n + p.tn - 1) / p.tn, per = mma_tokens<PAIR>((n + tt - 1) / tt);
  const int at = tile - tab.first[set];
  PTile t;
  t.set = set;
  t.pair = at / tt;
  const int c = (at - t.pair * tt) * per;
  t.tok0 = b.x + c;
  t.toks = min(per, n - c);
  t.n = mma_tokens<PAIR>(t.toks);
  return t;
}

// An epilogue warp's share of a finished tile: 32 rows (a thread each), every other sixteen of its n tokens, from tensor memory into the
// staging buffer [token][column] with bias, activation and residual (which waits there) in fp32.
template <int ACT, bool RES>
__device__ __forceinline__ void read_out_tokens(uint16_t* cs, uint32_t lane_t, int n, int eh, int q, int lane, float bias) {
#pragma unroll 2
  for (int m = eh * 16; m < n; m += EW / 4 * 16) {
    float v[16];
    tmem_ld<16>(lane_t + m, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += bias;
    if constexpr (ACT == W4A16_ACT_SWIGLU) {
      // gate and up are neighbouring lanes: each finishes eight of the pair's sixteen tokens
      uint16_t* at = cs + (m + (lane & 1) * 8) * (kTileRows / 2) + q * 16 + (lane >> 1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float got = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[i] : v[i + 8], 1);
        const float gate = lane & 1 ? got : v[i], up = lane & 1 ? v[i + 8] : got;
        float o = logistic_times(gate, gate) * up;
        if constexpr (RES) o += bf16_bits_to_float(at[i * (kTileRows / 2)]);
        at[i * (kTileRows / 2)] = float_to_bf16_bits(o);
      }
    } else {
      uint16_t* at = cs + m * kTileRows + q * 32 + lane;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float o = activate<ACT>(v[i]);
        if constexpr (RES) o += bf16_bits_to_float(at[i * kTileRows]);
        at[i * kTileRows] = float_to_bf16_bits(o);
      }
    }
  }
}
template <int MODE, int ACT>
__device__ __forceinline__ void read_out(bool residual, uint16_t* cs, uint32_t lane_t, int n, int eh, int q, int lane, float bias) {
  if (MODE == kDense && residual)  // (sets have none)
    read_out_tokens<ACT, true>(cs, lane_t, n, eh, q, lane, bias);
  else
    read_out_tokens<ACT, false>(cs, lane_t, n, eh, q, lane, bias);
}

// Four rows of a token with their sums complete: bias, activation, residual and the stores (dense layers).
__device__ __forceinline__ void finish_four(const RaggedCall& c, int N, int tok, int r, const float4& acc) {
  float v[4] = {acc.x, acc.y, acc.z, acc.w};
  if (c.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += bf16_bits_to_float(c.bias[bias_index(r + i, N, c.act)]);
  const bool gated = c.act == W4A16_ACT_SWIGLU;
  const size_t o = static_cast<size_t>(tok) * c.ny + (gated ? r >> 1 : r);
  if (gated) {
    v[0] = logistic_times(v[0], v[0]) * v[1];
    v[1] = logistic_times(v[2], v[2]) * v[3];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = activate(v[i], c.act);
  }
  const int n2 = gated ? 1 : 2;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (i < n2) {
      if (c.residual) {
        const uint32_t r2 = *reinterpret_cast<const uint32_t*>(c.residual + o + 2 * i);
        v[2 * i] += bf16_bits_to_float(static_cast<uint16_t>(r2));
        v[2 * i + 1] += bf16_bits_to_float(static_cast<uint16_t>(r2 >> 16));
      }
      *reinterpret_cast<uint32_t*>(c.y + o + 2 * i) =
          float_to_bf16_bits(v[2 * i]) | (static_cast<uint32_t>(float_to_bf16_bits(v[2 * i + 1])) << 16);
    }
}

template <int MODE, bool PAIR>
__global__ void __launch_bounds__(prefill_warps(MODE) * 32, 1) k_prefill(const __grid_constant__ PrefillParams p) {
  constexpr int CG = PAIR ? 2 : 1;  // CTAs of a tile
  constexpr std::bool_constant<PAIR> pair{};

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int xbytes = p.tn / CG * 256;  // one activation stage: two swizzled tiles of this CTA's share of TN tokens x 64 k
  uint8_t* xbuf = smem;          // 128-byte-swizzled TMA tiles start on 1024-byte boundaries
  uint8_t* cbuf = xbuf + kPSteps * xbytes;  // [TN tokens][128 rows] bf16: the finished tile on its way out
  uint8_t* ring = cbuf + p.tn * (kTileRows * 2);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + p.wdepth * kTileGroupBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kPBars);

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t rank = cluster_rank(), leader = PAIR ? rank & ~1u : rank;
  const int half = PAIR ? static_cast<int>(rank & 1u) : 0, split = static_cast<int>(PAIR ? rank >> 1 : rank);
  const int WD = p.wdepth, S = p.splits;
  const int na = a_slots(p.tn);
  const uint32_t ring_a = smem_u32(ring), xbuf_a = smem_u32(xbuf);
  const uint32_t wfull_a = smem_u32(bars);               // [WD] weights of a group landed
  const uint32_t wempty_a = wfull_a + kPMaxWD * 8;       // [WD] read by the 4 dequant warps
  const uint32_t done_a = wempty_a + kPMaxWD * 8;        // [kPDone] group j % 8 multiplied (both CTAs get the commit)
  const uint32_t dfull_a = done_a + kPDone * 8;          // accumulator complete (both CTAs)
  const uint32_t afull_a = dfull_a + 8;                  // [na] leader: a group's A operand written (4 warps of each CTA)
  const uint32_t xfull_a = afull_a + kPMaxA * 8;         // [kPSteps] leader: both CTAs' activations of a group landed
  const uint32_t dempty_a = xfull_a + kPSteps * 8;       // leader: accumulator read out (the epilogue warps of both CTAs)

  if (tid == 0) {
    for (int i = 0; i < kPMaxWD; ++i) {
      mbar_init(wfull_a + i * 8, 1);
      mbar_init(wempty_a + i * 8, 4);
    }
    for (int i = 0; i < kPDone; ++i) mbar_init(done_a + i * 8, 1);
    // activations: one arrival, the leader's, that expects the bytes of both CTAs (gathered rows: of all of the tile's tokens)
    for (int i = 0; i < kPSteps; ++i) mbar_init(xfull_a + i * 8, 1);
    for (int i = 0; i < kPMaxA; ++i) mbar_init(afull_a + i * 8, 4 * CG);
    mbar_init(dfull_a, 1);
    mbar_init(dempty_a, CG * EW);
    fence_mbar_init();
  }
  if (warp == kWIssue) {
    if constexpr (PAIR)
      tmem_alloc_pair(smem_u32(tmem_slot), kPTmemCols);
    else
      tmem_alloc(smem_u32(tmem_slot), kPTmemCols);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTAs' barriers exist from here on
  // The next launch's CTAs may take over each SM as this one's leave it: set-up, first weights and their expansion then run
  // under the rest of this launch. Its activations and everything behind them wait for this launch's end (griddepcontrol.wait).
  pdl_launch_dependents();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_a = tmem + (p.tn <= 128 ? 128 : 256);

  int tiles = p.tiles, set = 0;
  SetTable tab = {};
  if constexpr (MODE == kSets) {
    // the sets' bounds come from the kernel in front, and with them everything else
    int2* bounds = reinterpret_cast<int2*>(bars + kPBars + 2 + kPGather * kPSetsTN / 4);  // (behind the gathering warps' lists of rows)
    int* first = reinterpret_cast<int*>(bounds + p.call.sets);
    tab.bounds = bounds;
    tab.first = first;
    pdl_wait();
    load_bounds<prefill_warps(MODE) * 32>(bounds, p.call.offsets, p.call.sets, p.call.slots, tid);
    if (warp == 0)
      prefix_sums(first, p.call.sets, lane, [&](int e) { return (bounds[e].y - bounds[e].x + p.tn - 1) / p.tn * p.pairs; });
    __syncthreads();
    tiles = first[p.call.sets];
  }
  const int cluster = blockIdx.x / (CG * S), nclusters = gridDim.x / (CG * S);
  const int g0 = p.G * split / S, g1 = p.G * (split + 1) / S;  // this split's k groups (S <= G)
  bool dead = false;

  if (warp == kWWeights) {
    // ================================================================ weight producer
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 1;
      for (int tile = cluster; !dead && tile < tiles; tile += nclusters) {
        const PTile t = walk_tile<MODE, PAIR>(p, tile, set, tab);
        const int rt = min(CG * t.pair + half, p.row_tiles - 1);
        const uint8_t* src = p.stream + (static_cast<size_t>(rt) * p.G + g0) * kTileGroupBytes;
        if constexpr (MODE == kSets) src += p.call.set_bytes * t.set;
        for (int g = g0; g < g1; ++g, src += kTileGroupBytes) {
          if (!mbar_wait_bounded_relaxed(wempty_a + st * 8, ph, kPSpin)) {
            atomicExch(p.status, W4A16_ETIMEOUT);
            dead = true;
            break;
          }
          mbar_expect_tx(wfull_a + st * 8, kTileGroupBytes);
          bulk_g2s(ring_a + st * kTileGroupBytes, src, kTileGroupBytes, wfull_a + st * 8);
          if (++st == WD) {
            st = 0;
            ph ^= 1;
          }
        }
      }
      if (dead) {  // the copies in flight still have to land
        for (int i = 0; i < WD; ++i) mbar_wait_bounded_relaxed(wfull_a + i * 8, i < st ? ph ^ 1u : ph, 1u << 10);
      }
    }
  } else if (warp == kWIssue) {
    // ================================================================ MMA issuer (leader CTA only)
    // The whole warp walks (so that the operands stay in uniform registers), one elected lane issues.
    if (half == 0) {
      const uint16_t both = static_cast<uint16_t>(3u << rank);  // (a pair's two CTAs)
      const uint64_t desc0 = umma_desc_sw128(xbuf_a);
      const uint32_t x16 = static_cast<uint32_t>(xbytes) >> 4;
      uint32_t j = 0, aph = 0, dph = 1;
      int a = 0;
      for (int tile = cluster; !dead && tile < tiles; tile += nclusters, dph ^= 1) {
        const uint32_t idesc = umma_idesc_bf16(CG * kTileRows, walk_tile<MODE, PAIR>(p, tile, set, tab).n);
        if (!warp_agrees(mbar_wait_bounded(dempty_a, dph, kPSpin))) dead = true;  // (passes on the first tile)
        for (int g = g0; !dead && g < g1; ++g, ++j) {
          const uint32_t st = j & (kPSteps - 1);
          if (!warp_waits(xfull_a + st * 8, (j / kPSteps) & 1u, afull_a + a * 8, aph, kPSpin)) {
            dead = true;
            break;
          }
          tc_fence_after();
          // B operand of the group: two swizzled tiles of 128-byte rows, one per token; a 16-k slab is 32 bytes
          // further along them
          const uint64_t b0 = desc0 + st * x16, b1 = b0 + (x16 >> 1);
          const uint32_t at = tmem_a + a * 64;
          if (elect_one()) {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
              if constexpr (PAIR)
                umma_bf16_ts_pair(tmem, at + s * 8, (s < 4 ? b0 : b1) + 2 * (s & 3), idesc, s > 0 || g > g0);
              else
                umma_bf16_ts(tmem, at + s * 8, (s < 4 ? b0 : b1) + 2 * (s & 3), idesc, s > 0 || g > g0);
            }
            if constexpr (PAIR) {
              umma_commit_pair(done_a + (j & (kPDone - 1)) * 8, both);
              if (g == g1 - 1) umma_commit_pair(dfull_a, both);
            } else {
              umma_commit(done_a + (j & (kPDone - 1)) * 8);
              if (g == g1 - 1) umma_commit(dfull_a);
            }
          }
          __syncwarp();
          if (++a == na) {
            a = 0;
            aph ^= 1;
          }
        }
      }
      if (dead && lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
    }
  } else if (warp == kWActs || (MODE == kSets && warp > kWActs)) {
    // ================================================================ activation producer
    // Two tiled TMA loads per k group (64 k each) into this CTA's half of the token tile; rows past M are zero-filled. The
    // leader's barrier expects both CTAs' bytes.
    if (MODE == kSets && p.call.x_rows) {
      // Rows are gathered by TMA, four rows of 64 k a load, half of the tile's tokens in each CTA; places past the tile's tokens repeat
      // the last one. Issuing a load takes a warp some 25 cycles and a group has up to 56 (28 fours of rows, two halves of the group's k), so
      // three warps take the groups in turn, each with its own list of rows. 64 experts 2048 x 5120 of 8 picks, with tiles of 160 tokens (up to 40
      // loads), us at 300 / 1200 / 4096 tokens: one warp (a shuffle per row) 232 / 460 / 1270, two 178 / 319 / 831, with lists 145 / 267 / 675,
      // three 140 / 245 / 623, four the same; rows already in slot order 133 / 216 / 548.
      const uint32_t xfull_l = PAIR ? map_to_rank(xfull_a, leader) : xfull_a;
      int* rows = reinterpret_cast<int*>(bars + kPBars + 2) + (warp - kWActs) * (kPSetsTN / 2);  // (16-byte aligned)
      uint32_t j = 0;
      for (int tile = cluster; !dead && tile < tiles; tile += nclusters) {
        const PTile t = walk_tile<MODE, PAIR>(p, tile, set, tab);
        __syncwarp();
        for (int i = lane; i < t.n / CG; i += 32) {
          const int slot = t.tok0 + min(half * (t.n / CG) + i, t.toks - 1);
          rows[i] = min(max(__ldcg(p.call.x_rows + slot), 0), p.call.x_tokens - 1);  // (no read outside x, whatever the rows hold)
        }
        __syncwarp();
        const int fours = t.n / (4 * CG);
        for (int g = g0; g < g1; ++g, ++j) {
          if (j % kPGather != static_cast<uint32_t>(warp - kWActs)) continue;
          const uint32_t st = j & (kPSteps - 1);
          const uint32_t jd = j - kPSteps;
          if (!warp_agrees(j < kPSteps || mbar_wait_bounded(done_a + (jd & (kPDone - 1)) * 8, (jd / kPDone) & 1u, kPSpin))) {
            dead = true;
            break;
          }
          if (half == 0 && lane == 0) mbar_expect_tx(xfull_a + st * 8, t.n * 256);
          __syncwarp();
          const uint32_t dst = xbuf_a + st * xbytes;
          if (elect_one()) {
#pragma unroll 4
            for (int i = 0; i < fours; ++i) {
              const int4 rr = *reinterpret_cast<const int4*>(rows + 4 * i);
              tma_gather<PAIR>(dst + i * 512, &p.amap, g * kGroup, rr, xfull_l + st * 8);
              tma_gather<PAIR>(dst + i * 512 + (xbytes >> 1), &p.amap, g * kGroup + 64, rr, xfull_l + st * 8);
            }
          }
          __syncwarp();
        }
      }
      if (dead && lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
      if (dead && half == 0) {
        for (uint32_t i = j < kPSteps ? 0 : j - kPSteps; i < j; ++i)
          mbar_wait_bounded_relaxed(xfull_a + (i & (kPSteps - 1)) * 8, (i / kPSteps) & 1u, 1u << 10);
      }
      __syncwarp();
    } else if (warp == kWActs && lane == 0) {
      const uint32_t xfull_l = PAIR ? map_to_rank(xfull_a, leader) : xfull_a;
      pdl_wait();  // the previous kernel produced the activations (the weights never depend on it)
      uint32_t j = 0;
      for (int tile = cluster; !dead && tile < tiles; tile += nclusters) {
        const PTile t = walk_tile<MODE, PAIR>(p, tile, set, tab);
        const int y = t.tok0 + half * (t.n / CG);
        for (int g = g0; g < g1; ++g, ++j) {
          const uint32_t st = j & (kPSteps - 1);
          const uint32_t jd = j - kPSteps;
          if (j >= kPSteps && !mbar_wait_bounded_relaxed(done_a + (jd & (kPDone - 1)) * 8, (jd / kPDone) & 1u, kPSpin)) {
            atomicExch(p.status, W4A16_ETIMEOUT);
            dead = true;
            break;
          }
          if (half == 0) mbar_expect_tx(xfull_a + st * 8, CG * xbytes);
          if constexpr (PAIR) {
            tma_load_pair(xbuf_a + st * xbytes, &p.amap, g * kGroup, y, xfull_l + st * 8);
            tma_load_pair(xbuf_a + st * xbytes + (xbytes >> 1), &p.amap, g * kGroup + 64, y, xfull_l + st * 8);
          } else {
            tma_load(xbuf_a + st * xbytes, &p.amap, g * kGroup, y, xfull_l + st * 8);
            tma_load(xbuf_a + st * xbytes + (xbytes >> 1), &p.amap, g * kGroup + 64, y, xfull_l + st * 8);
          }
        }
      }
      if (dead && half == 0) {
        for (uint32_t i = j < kPSteps ? 0 : j - kPSteps; i < j; ++i)
          mbar_wait_bounded_relaxed(xfull_a + (i & (kPSteps - 1)) * 8, (i / kPSteps) & 1u, 1u << 10);
      }
    }
  } else if (warp < PW) {
    // ================================================================ dequant warps
    // The walk over tiles does not matter here: the groups come in the order of the weight ring.
    // Four teams of four warps (one output row per thread) take the groups in turn: one group's waits, shared-memory loads and
    // tensor-memory stores run beside the others' arithmetic. (The weight ring's depth is a multiple of four and the ring of
    // "group multiplied" barriers has eight, so a barrier's consecutive phases belong to one team; a parity wait could
    // not tell them apart otherwise.)
    // A team of eight warps with half a row each paid every wait, vote and arrival twice: 34816 x 5120 at M = 17 / 77 31.8 / 36.0 us
    // with two teams of eight, 29.6 / 34.7 with four of four (M = 777, four layers of a block: 546 and 533).
    const int q = warp & 3, team = warp >> 2;
    const int row = q * 32 + lane;
    const uint32_t a_t = tmem_a + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t afull_l = PAIR ? map_to_rank(afull_a, leader) : afull_a;
    const int ntiles = cluster < tiles ? (tiles - 1 - cluster) / nclusters + 1 : 0;
    const uint32_t ngroups = static_cast<uint32_t>(ntiles) * static_cast<uint32_t>(g1 - g0);
    const uint32_t off_e = weight_slot(row, 0) * 16, off_o = kChunkBytes + weight_slot(row, 1) * 16;  // even and odd 32-k chunks
    int st = team, a = team;  // weight stage and A slot
    uint32_t wph = 0;
    for (uint32_t j = team; j < ngroups; j += kPTeams) {
      const bool landed = mbar_wait_bounded(wfull_a + st * 8, wph, kPSpin);
      const uint32_t blk = ring_a + st * kTileGroupBytes;
      const uint4 w[4] = {lds128<0>(blk + off_e), lds128<0>(blk + off_o), lds128<2 * kChunkBytes>(blk + off_e),
                          lds128<2 * kChunkBytes>(blk + off_o)};
      const uint32_t zp = lds_u8<kTgZpOff>(blk + row), sc = lds_u16<kTgScaleOff>(blk + 2 * row);
      const uint32_t zpair = __byte_perm(zp, 0x43434343u, 0x4040);  // bf16 pair (128+zp, 128+zp)
      const uint32_t spair = sc | (sc << 16);
      // Nibbles 0 and 4 of a word become (128 + q) - (128 + zp) by one OR and a subtraction. Nibbles 1 and 5 are left where they
      // are: as a bf16 pair w & 0x00F000F0 is q 2^-129 (subnormals, and the first normal binade goes on where they end), so
      // one packed FMA makes (q - zp) / 4 of it, exactly, and 4 s is exact too: the same product, rounded once. The ALU pipe
      // (shifts and LOP3) is the busiest: 80 of its instructions per row and group instead of 112. Four layers of a block at M = 30 /
      // 77: 77.7 / 85.0 us with a shift per nibble position, 76.5 / 83.8 with this (74.1 / 81.7 without the test for large scales).
      const uint32_t zquarter = fma_bf16x2(zpair, 0xBE80BE80u, 0x42004200u);  // -zp / 4 = 32 - (128 + zp) / 4
      const uint32_t s4 = mul_bf16x2(spair, 0x40804080u);
      auto expand = [&](const uint4& c, uint32_t(&v)[16]) {
        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w8 = cw[i] >> 8;
          v[4 * i] = mul_bf16x2(sub_bf16x2(and_or(cw[i], kNibMaskP, kMagicP), zpair), spair);
          v[4 * i + 1] = mul_bf16x2(fma_bf16x2(cw[i] & 0x00F000F0u, 0x7F007F00u, zquarter), s4);
          v[4 * i + 2] = mul_bf16x2(sub_bf16x2(and_or(w8, kNibMaskP, kMagicP), zpair), spair);
          v[4 * i + 3] = mul_bf16x2(fma_bf16x2(w8 & 0x00F000F0u, 0x7F007F00u, zquarter), s4);
        }
      };
      // ... unless 4 s overflows, from 2^126 on
      auto expand_large = [&](const uint4& c, uint32_t(&v)[16]) {
        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int pp = 0; pp < 4; ++pp)
            v[4 * i + pp] = mul_bf16x2(sub_bf16x2(and_or(cw[i] >> (4 * pp), kNibMaskP, kMagicP), zpair), spair);
      };
      const bool fine = warp_agrees(landed && (sc & 0x7FFFu) - 0x7E80u >= 0x100u);
      if (!fine && !warp_agrees(landed)) {
        dead = true;
        break;
      }
      // The row is in registers but used only below: a vote orders no memory accesses, __syncwarp does, so that the next bulk copy
      // into the stage cannot pass another lane's loads.
      __syncwarp();
      if (lane == 0) mbar_arrive(wempty_a + st * 8);
      // the wait for the A slot: the MMAs that read it last, na groups ago, must have completed
      const uint32_t jd = j - na;
      if (!warp_agrees(j < static_cast<uint32_t>(na) ||
                       mbar_wait_bounded(done_a + (jd & (kPDone - 1)) * 8, (jd / kPDone) & 1u, kPSpin))) {
        dead = true;
        break;
      }
      tc_fence_after();
      // Sixteen registers at a time, expanded and stored at once: with half a row expanded in front of the wait the stores' operands had to
      // be moved together. (34816 x 5120 at M = 17 30.2 -> 29.2 us, 64 experts 2048 x 5120 at 300 tokens 124.8 -> 120.6.)
      if (fine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t v[16];
          expand(w[i], v);
          tmem_st16(a_t + a * 64 + 16 * i, v);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t v[16];
          expand_large(w[i], v);
          tmem_st16(a_t + a * 64 + 16 * i, v);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(afull_l + a * 8, pair);
      if ((a += kPTeams) >= na) a -= na;
      if ((st += kPTeams) >= WD) {
        st -= WD;
        wph ^= 1;
      }
    }
    if (dead && lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
  } else if (S == 1) {
    // ================================================================ epilogue warps
    // The next tile's MMAs wait for the accumulator, so it is read out into shared memory (as bf16) and handed back;
    // the stores to C, 256 bytes per token, run beside the next tile's main loop.
    const int q = warp & 3, eh = (warp - kWEpi0) >> 2, et = tid - kWEpi0 * 32;
    const uint32_t lane_t = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t dempty_l = PAIR ? map_to_rank(dempty_a, leader) : dempty_a;
    uint32_t dph = 0;
    // Layers with an epilogue: the sums are finished in registers on their way out, in fp32. The residual's tile waits in the
    // staging buffer by then, brought in beside the main loop.
    auto finish_tile = [&](const PTile& t, uint32_t phase) {
      const RaggedCall& c = p.call;
      const bool gated = c.act == W4A16_ACT_SWIGLU;
      const int w8 = gated ? 3 : 4;                              // log2 of the eights of columns per token
      const int r0 = (CG * t.pair + half) * kTileRows;
      const int cols = min(kTileRows, p.N - r0) >> (gated ? 1 : 0);  // (<= 0: an odd last row tile's second half)
      const int col0 = gated ? r0 >> 1 : r0, cl = (et & ((1 << w8) - 1)) * 8;
      uint16_t* cs = reinterpret_cast<uint16_t*>(cbuf);
      const size_t line0 = static_cast<size_t>(t.tok0) * c.ny + col0 + cl;
      if (c.residual) {
        if (cl < cols)
#pragma unroll 4
          for (int m = et >> w8; m < t.toks; m += EW * 32 >> w8)
            *reinterpret_cast<uint4*>(cs + (m << (w8 + 3)) + cl) = *reinterpret_cast<const uint4*>(c.residual + line0 + static_cast<size_t>(m) * c.ny);
        named_bar_sync(1, EW * 32);
      }
      const int row = r0 + q * 32 + lane;
      const float bias = c.bias && row < p.N
                             ? bf16_bits_to_float(c.bias[static_cast<size_t>(t.set) * p.N + bias_index(row, p.N, c.act)]) : 0.f;
      if (!dead && !warp_agrees(mbar_wait_bounded_relaxed(dfull_a, phase, kPSpin))) {
        dead = true;
        if (lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
      }
      if (!dead) {
        tc_fence_after();
        switch (c.act) {
          case W4A16_ACT_SWIGLU: read_out<MODE, W4A16_ACT_SWIGLU>(c.residual, cs, lane_t, t.n, eh, q, lane, bias); break;
          case W4A16_ACT_SILU: read_out<MODE, W4A16_ACT_SILU>(c.residual, cs, lane_t, t.n, eh, q, lane, bias); break;
          case W4A16_ACT_GELU: read_out<MODE, W4A16_ACT_GELU>(c.residual, cs, lane_t, t.n, eh, q, lane, bias); break;
          case W4A16_ACT_GELU_TANH: read_out<MODE, W4A16_ACT_GELU_TANH>(c.residual, cs, lane_t, t.n, eh, q, lane, bias); break;
          default: read_out<MODE, W4A16_ACT_NONE>(c.residual, cs, lane_t, t.n, eh, q, lane, bias);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(dempty_l, pair);
      }
      named_bar_sync(1, EW * 32);  // every epilogue warp comes here for every tile, dead or not
      if (cl < cols && !dead)
        for (int m = et >> w8; m < t.toks; m += EW * 32 >> w8)
          *reinterpret_cast<uint4*>(c.y + line0 + static_cast<size_t>(m) * c.ny) = *reinterpret_cast<const uint4*>(cs + (m << (w8 + 3)) + cl);
      named_bar_sync(1, EW * 32);  // the next tile overwrites the staged one
    };
    if constexpr (MODE != kPlain) pdl_wait();  // bias and residual may come from the kernel in front
    for (int tile = cluster; tile < tiles; tile += nclusters, dph ^= 1) {
      const PTile t = walk_tile<MODE, PAIR>(p, tile, set, tab);
      uint16_t* cs = reinterpret_cast<uint16_t*>(cbuf);
      if constexpr (MODE != kPlain) {
        finish_tile(t, dph);
        continue;
      }
      if (!dead && !warp_agrees(mbar_wait_bounded_relaxed(dfull_a, dph, kPSpin))) {
        dead = true;
        if (lane == 0) atomicExch(p.status, W4A16_ETIMEOUT);
      }
      if (!dead) {
        tc_fence_after();
#pragma unroll 2
        for (int c = eh * 16; c < t.n; c += EW / 4 * 16) {
          float v[16];
          tmem_ld<16>(lane_t + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) cs[(c + i) * kTileRows + q * 32 + lane] = float_to_bf16_bits(v[i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(dempty_l, pair);
      }
      named_bar_sync(1, EW * 32);  // every epilogue warp comes here for every tile, dead or not
      const int r0 = (CG * t.pair + half) * kTileRows;
      const int rows = min(kTileRows, p.N - r0);                     // (<= 0: an odd last row tile's second half)
      const int toks = dead ? 0 : min(t.n, p.M - t.tok0);
      if (p.wide) {
        const int rl = (et & 15) * 8;  // eight rows of one token per thread
        if (rl < rows) {
          for (int c = et >> 4; c < toks; c += EW * 2) {
            const uint4 v = *reinterpret_cast<const uint4*>(cs + c * kTileRows + rl);
            const size_t o = static_cast<size_t>(t.tok0 + c) * p.ldc + p.col0 + r0 + rl;
            *reinterpret_cast<uint4*>(p.C + o) = v;
            for (int pq = 0; pq < p.npeers; ++pq) *reinterpret_cast<uint4*>(p.C_peers[pq] + o) = v;  // fused all-gather over NVLink
          }
        }
      } else {
        for (int i = et; i < toks * kTileRows; i += EW * 32) {
          const int rl = i & (kTileRows - 1);
          if (rl < rows) {
            const size_t o = static_cast<size_t>(t.tok0 + i / kTileRows) * p.ldc + p.col0 + r0 + rl;
            p.C[o] = cs[i];
            for (int pq = 0; pq < p.npeers; ++pq) p.C_peers[pq][o] = cs[i];
          }
        }
      }
      named_bar_sync(1, EW * 32);  // the next tile overwrites the staged one
    }
  }

  if (MODE != kSets && S > 1) {
    // ================================================================ split K: one tile per cluster
    // Every split's fp32 tile goes to its own shared memory (the activation stages: all MMAs have read them, and
    // [TN tokens][128 rows] floats are exactly their size), then split s adds up and stores the s-th share
    // of the tokens, reading the others' tiles through the cluster.
    const PTile t = tile_of<PAIR>(p, cluster);
    if (warp >= kWEpi0 && warp < kWEpi0 + EW) {
      const int q = warp & 3;
      const uint32_t lane_t = tmem + (static_cast<uint32_t>(q * 32) << 16);
      if (warp_agrees(mbar_wait_bounded(dfull_a, 0, kPSpin))) {
        tc_fence_after();
        float* tile_s = reinterpret_cast<float*>(xbuf) + q * 32 + lane;
#pragma unroll 1
        for (int c = ((warp - kWEpi0) >> 2) * 16; c < t.n; c += EW / 4 * 16) {
          float v[16];
          tmem_ld<16>(lane_t + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) tile_s[(c + i) * kTileRows] = v[i];
        }
      } else if (lane == 0) {
        atomicExch(p.status, W4A16_ETIMEOUT);
      }
    }
    __syncwarp();
    cluster_sync();
    if constexpr (MODE != kPlain) pdl_wait();  // bias and residual may come from the kernel in front
    if (warp < PW + EW) {
      // Four rows of a token per thread: 16-byte loads from every split's tile, 256 contiguous bytes of C per warp. (One row per
      // thread, 4-byte loads and 64-byte runs of C took 1.6 us of a 5120 x 6144 launch at M = 77. The four layers of a block at M = 77,
      // three of which split: 85.1 -> 83.8 us, at M = 40 80.7 -> 79.9.)
      const int c0 = t.n * split / S, n4 = (t.n * (split + 1) / S - c0) * (kTileRows / 4);
      const int r0 = (CG * t.pair + half) * kTileRows;
      uint32_t src[kPMaxSplit];
#pragma unroll
      for (int s = 0; s < kPMaxSplit; ++s)
        src[s] = map_to_rank(xbuf_a, static_cast<uint32_t>(CG * min(s, S - 1) + half)) + c0 * (kTileRows * 4);
#pragma unroll 2
      for (int i = tid; i < n4; i += (PW + EW) * 32) {
        const int r = r0 + 4 * (i & (kTileRows / 4 - 1)), tok = t.tok0 + c0 + i / (kTileRows / 4);
        float4 part[kPMaxSplit];
#pragma unroll
        for (int s = 0; s < kPMaxSplit; ++s)
          if (s < S) part[s] = ld_cluster_f32x4(src[s] + i * 16);
        float4 acc = part[0];
#pragma unroll
        for (int s = 1; s < kPMaxSplit; ++s)
          if (s < S) {
            acc.x += part[s].x;
            acc.y += part[s].y;
            acc.z += part[s].z;
            acc.w += part[s].w;
          }
        if constexpr (MODE != kPlain) {
          if (r < p.N && tok < p.M) finish_four(p.call, p.N, tok, r, acc);
          continue;
        }
        if (r < p.N && tok < p.M) {  // (N is a multiple of 16)
          const size_t o = static_cast<size_t>(tok) * p.ldc + p.col0 + r;
          const uint2 v = make_uint2(float_to_bf16_bits(acc.x) | (static_cast<uint32_t>(float_to_bf16_bits(acc.y)) << 16),
                                     float_to_bf16_bits(acc.z) | (static_cast<uint32_t>(float_to_bf16_bits(acc.w)) << 16));
          auto store = [&](uint16_t* c) {
            if (p.wide) {
              *reinterpret_cast<uint2*>(c) = v;
            } else {
              c[0] = static_cast<uint16_t>(v.x);
              c[1] = static_cast<uint16_t>(v.x >> 16);
              c[2] = static_cast<uint16_t>(v.y);
              c[3] = static_cast<uint16_t>(v.y >> 16);
            }
          };
          store(p.C + o);
          for (int pq = 0; pq < p.npeers; ++pq) store(p.C_peers[pq] + o);
        }
      }
    }
  }

  // Nobody leaves while the other CTAs of the cluster may still reach its barriers, shared or tensor memory.
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  if (warp == kWIssue) {
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem, kPTmemCols);
    else
      tmem_dealloc(tmem, kPTmemCols);
  }
  // every store of this CTA was issued before the barrier above: its share of the launch's completion signal
  if (p.comm_local && tid == 0) signal_cta_done(p.comm_local, p.comm_peers, p.comm_n, p.comm_rank);
}

// ------------------------------------------------------------------ the plan of a launch
struct PrefillPlan {
  bool pair = true;
  int tn = 0, splits = 1, full_tt = 0, tiles = 0, clusters = 0, wdepth = 0, smem = 0;
};

int prefill_smem(bool pair, int tn, int wdepth) {
  return 1024 + kPSteps * tn * (pair ? 128 : 256) + tn * kTileRows * 2 + wdepth * kTileGroupBytes + kPBars * 8 + 16;
}

// Tokens per tile and K splits. A cluster's time for a tile is its k groups times the slower of the tensor cores
// (4 TN cycles per group for a pair) and the expansion of the weights (kExpand cycles per group), plus
// what is paid once per tile (pipeline fill, read-out of the accumulator, the exchange of split K). Tiles go to
// the clusters in turn, dearest first, so cluster 0 has the longest list: its total is what is minimised.
// The constants rank the shapes, they do not predict times: a group of a short prompt takes about one and a half times kExpand (see
// above). Against every other (TN, S), on 22 shapes of 1024..34816 rows, 4096..17408 columns and 17..1500 tokens: the choice was the
// fastest on 17. 5120 x 17408 at M = 24: 32 tokens and three splits 20.1 us, two 25.7, one 45.0; 6144 x 5120 at M = 100: two
// splits 13.2, one 15.7; 34816 x 5120 at M = 520: 192 tokens 141, 224 149, 160 161, 128 182. Where kExpand misleads it, tiles
// come out too narrow: 12288 x 4096 at M = 200 96 tokens 30.7 us, 224 23.2; 8192 x 5120 at M = 777 96 tokens 69.1, 224 55.1; 34816 x 5120
// at M = 1024 128 tokens 285, 256 271; 1024 x 4096 at M = 64 32 tokens in four splits 6.6, 64 tokens 5.8. Too wide: 34816 x 5120 at M = 777
// 224 tokens 208, 160 203.
// `only` > 0 asks for that number of splits. The choice goes by what a B200 of 148 SMs runs (index S: clusters of 2 S CTAs
// at once, as cudaOccupancyMaxActiveClusters answers on two of them), not by what this device's GPCs happen to fit, so that a
// row has the same bits on every GPU; the device only rules out clusters it cannot run at all and sizes the grid.
PrefillPlan plan_prefill(int M, int pairs, int G, const int* device_clusters, int smem_optin, int only) {
  constexpr int kClusters[kPMaxSplit + 1] = {0, 74, 33, 22, 15};
  constexpr int kExpand = 420, kFill = 2500, kReduce = 4000;
  PrefillPlan best;
  long long best_cost = -1;
  for (int S = 1; S <= kPMaxSplit && S <= G; ++S) {
    const int slots = kClusters[S];
    if (device_clusters[S] < 1 || (only > 0 && S != only)) continue;
    for (int tn = 32; tn <= kPMaxTN; tn += 32) {
      const int full = M / tn, rest = M - full * tn;
      if (full == 0 && tn - 32 >= rest) break;  // one token tile: the smallest that holds M
      const long long nfull = static_cast<long long>(pairs) * full, tiles = nfull + (rest ? pairs : 0);
      if (S > 1 && tiles > slots) continue;     // split clusters take one tile each
      const int groups = (G + S - 1) / S;
      auto cost = [&](int n) {
        const long long loop = static_cast<long long>(groups) * (4 * n > kExpand ? 4 * n : kExpand);
        return loop + (S > 1 ? kFill + kReduce : kFill / 2);
      };
      const long long cf = cost(tn), cr = cost((rest + 31) & ~31);
      const long long wf = (nfull + slots - 1) / slots, wa = (tiles + slots - 1) / slots;
      const long long total = wf * cf + (wa - wf) * cr;
      if (best_cost < 0 || total < best_cost) {
        best_cost = total;
        best.tn = tn;
        best.splits = S;
        best.full_tt = full;
        best.tiles = static_cast<int>(tiles);
        best.clusters = static_cast<int>(S > 1 || tiles < device_clusters[S] ? tiles : device_clusters[S]);
      }
    }
  }
  // A multiple of the teams: tiles of 224 tokens keep four stages of the six that would fit, of 128 twelve of fourteen. Two teams and six
  // (fourteen) stages -> four teams and four (twelve), in us: 34816 x 5120 at M = 200 55.8 -> 55.4, 16384 x 5120 at M = 210 28.48 -> 28.43, 5120 x
  // 17408 at M = 209 35.3 -> 34.8; at 128 tokens 16384 x 5120 at M = 112 20.0 -> 19.1, 34816 x 5120 at M = 128 39.4 -> 37.7.
  best.wdepth = kPMaxWD;
  while (best.wdepth > kPTeams && prefill_smem(best.pair, best.tn, best.wdepth) > smem_optin) best.wdepth -= kPTeams;
  best.smem = prefill_smem(best.pair, best.tn, best.wdepth);
  return best;
}

// The plan of a dense layer with an epilogue whose tokens fit one tile of a CTA alone: as many K splits as find clusters at
// once. (row tiles of 128; clusters of S CTAs, as many at once as a B200 of 148 SMs runs)
PrefillPlan plan_single(int M, int row_tiles, int G, const int* device_clusters, int smem_optin) {
  constexpr int kClusters[kPMaxSplit + 1] = {0, 148, 74, 45, 33};
  PrefillPlan plan;
  plan.pair = false;
  plan.tn = (M + 15) & ~15;
  plan.splits = splits_at_once(row_tiles, G < kPMaxSplit ? G : kPMaxSplit, kClusters, device_clusters);
  plan.full_tt = M / plan.tn;
  plan.tiles = row_tiles;
  plan.clusters = plan.splits > 1 || row_tiles < device_clusters[1] ? row_tiles : device_clusters[1];
  plan.wdepth = kPMaxWD;
  while (plan.wdepth > kPTeams && prefill_smem(false, plan.tn, plan.wdepth) > smem_optin) plan.wdepth -= kPTeams;
  plan.smem = prefill_smem(false, plan.tn, plan.wdepth);
  return plan;
}

int table_bytes(int sets) { return kPGather * (kPSetsTN / 2) * 4 + sets * 12 + 16; }

}  // namespace
}  // namespace w4a16

using namespace w4a16;

extern "C" {

int w4a16_workspace_alloc(w4a16_workspace_t* ws, size_t bytes) {
  W4_REQUIRE(ws != nullptr, "workspace_alloc: null struct");
  memset(ws, 0, sizeof *ws);
  // The fused kernel needs no dequantised tile; keep a small valid allocation because the
  // reference's callers free `wbuf` themselves (src/model/model.cu:440-441).
  (void)bytes;
  void* p = nullptr;
  W4_CUDA(cudaMalloc(&p, 4096));
  ws->wbuf = static_cast<uint16_t*>(p);
  ws->bytes = 4096;
  return W4A16_OK;
}

int w4a16_workspace_free(w4a16_workspace_t* ws) {
  W4_REQUIRE(ws != nullptr, "workspace_free: null struct");
  cudaFree(ws->wbuf);
  memset(ws, 0, sizeof *ws);
  return W4A16_OK;
}

}  // extern "C"

namespace w4a16 {
namespace {
void cluster_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* at, int warps, int size, int clusters, int smem) {
  cfg.gridDim = dim3(size * clusters);
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = smem;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
}

// How many clusters of S tiles' CTAs (one CTA per SM) the device runs at once, index S; asked for once per device.
// The kernel's shared-memory attribute is set on the way. Returns nullptr (and sets the error) on failure.
template <int MODE, bool PAIR>
const int* cluster_slots(int dev, const DeviceInfo* di) {
  struct Slots {
    bool ready = false;
    int n[kPMaxSplit + 1] = {};
  };
  static std::mutex mu;
  static Slots all[64];
  std::lock_guard<std::mutex> lk(mu);
  Slots& s = all[dev & 63];
  if (!s.ready) {
    cudaError_t e = cudaFuncSetAttribute(k_prefill<MODE, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, di->smem_optin);
    for (int S = 1; S <= kPMaxSplit && e == cudaSuccess; ++S) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1];
      cluster_config(cfg, at, prefill_warps(MODE), PAIR ? 2 * S : S, 1, prefill_smem(true, kPMaxTN, kPTeams));
      e = cudaOccupancyMaxActiveClusters(&s.n[S], k_prefill<MODE, PAIR>, &cfg);
    }
    if (e != cudaSuccess || s.n[1] < 1) {
      fail(W4A16_ECUDA, "gemm_prefill: the device runs no CTA pair of the kernel (%s)", cudaGetErrorString(e));
      return nullptr;
    }
    s.ready = true;
  }
  return s.n;
}

// The current device's plan for M tokens through `row_tiles` row tiles and G k groups of a layer of `layer_tiles` row
// tiles. A shard is split as the whole layer would be, so that a row has the same bits sharded and unsharded; as its
// tiles are fewer, they always fit the clusters that the layer's would. (What the shard's own choice would save is left.)
template <int MODE>
int current_plan(PrefillPlan& plan, int M, int row_tiles, int layer_tiles, int G) {
  const DeviceInfo* di = device_info();
  if (!di) return W4A16_ECUDA;
  const int* slots = cluster_slots<MODE, true>(di->device, di);
  if (!slots) return W4A16_ECUDA;
  plan = plan_prefill(M, (layer_tiles + 1) / 2, G, slots, di->smem_optin, 0);
  if (row_tiles < layer_tiles && plan.tn > 0)
    plan = plan_prefill(M, (row_tiles + 1) / 2, G, slots, di->smem_optin, plan.splits);
  W4_REQUIRE(plan.tn > 0, "gemm_prefill: no launch shape for M = %d, %d row tiles x %d k groups", M, row_tiles, G);
  return W4A16_OK;
}

// The tensor map of activations [tokens][K]: boxes of 64 k x `rows` tokens, 128-byte swizzle, zeros past the last token.
int encode_acts(CUtensorMap* map, const uint16_t* A, int K, int tokens, int rows) {
  // driver entry point for the tensor-map encoder (no link-time dependency on libcuda)
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    W4_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres));
    W4_REQUIRE(fn != nullptr && qres == cudaDriverEntryPointSuccess, "gemm_prefill: cuTensorMapEncodeTiled unavailable");
    encode = reinterpret_cast<EncodeFn>(fn);
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(K) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult cr = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t*>(A), dims, strides,
                             box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return cr == CUDA_SUCCESS ? W4A16_OK : fail(W4A16_ECUDA, "gemm_prefill: cuTensorMapEncodeTiled failed (%d)", int(cr));
}

// The launch, programmatic unless a weight write is in front of a kernel that reads weights before its wait.
template <int MODE, bool PAIR>
int enqueue_prefill(const PrefillParams& p, const PrefillPlan& plan, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cluster_config(cfg, at, prefill_warps(MODE), PAIR ? 2 * plan.splits : plan.splits, plan.clusters, plan.smem);
  const bool behind_write = MODE != kSets && take_weight_write(stream);
  if (!behind_write && pdl_enabled()) {
    // (behind a weight write the launch is fully ordered: the weights are read before the wait)
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  cfg.stream = stream;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_prefill<MODE, PAIR>, p);
  if (e == cudaSuccess) return W4A16_OK;
  if (behind_write) note_weight_write(stream);
  return fail(W4A16_ECUDA, "gemm_prefill: launch: %s", cudaGetErrorString(e));
}

int launch_prefill(PrefillParams& p, uint16_t* C, const w4a16_weights_t* w, const uint16_t* A, int M, w4a16_workspace_t* ws,
                   void* stream) {
  if (int rc = check_weights(w)) return rc;
  W4_REQUIRE(C != nullptr && A != nullptr, "gemm_prefill: null matrix");
  W4_REQUIRE((reinterpret_cast<uintptr_t>(A) & 15) == 0, "gemm_prefill: A not 16-byte aligned");
  W4_REQUIRE(M >= 1, "gemm_prefill: M = %d", M);
  W4_REQUIRE(ws != nullptr, "gemm_prefill: null workspace");
  const DeviceInfo* di = device_info();
  if (!di) return W4A16_ECUDA;
  p.stream = reinterpret_cast<const uint8_t*>(w->qweight);
  p.C = C;
  p.M = M;
  p.N = w->out_f;
  p.K = w->in_f;
  p.G = w->num_groups;
  p.row_tiles = (w->out_f + kTileRows - 1) / kTileRows;
  p.pairs = (p.row_tiles + 1) / 2;
  PrefillPlan plan;
  const int layer_tiles = static_cast<int>((p.ldc + kTileRows - 1) / kTileRows);
  if (int rc = current_plan<kPlain>(plan, M, p.row_tiles, layer_tiles, p.G)) return rc;
  p.tn = plan.tn;
  p.splits = plan.splits;
  p.wdepth = plan.wdepth;
  p.full_tt = plan.full_tt;
  p.tiles = plan.tiles;
  p.status = di->status;
  p.wide = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && p.ldc % 8 == 0 && p.col0 % 8 == 0;
  for (int q = 0; q < p.npeers; ++q)
    if (reinterpret_cast<uintptr_t>(p.C_peers[q]) & 15) p.wide = 0;
  if (int rc = encode_acts(&p.amap, A, w->in_f, M, plan.tn / 2)) return rc;
  return enqueue_prefill<kPlain, true>(p, plan, static_cast<cudaStream_t>(stream));
}
}  // namespace

int launch_prefill_ragged(const RaggedCall& c, cudaStream_t stream) {
  const DeviceInfo* di = device_info();
  if (!di) return W4A16_ECUDA;
  PrefillParams p = {};
  p.call = c;
  p.stream = c.stream;
  p.M = c.slots;
  p.N = c.N;
  p.K = c.K;
  p.G = c.G;
  p.row_tiles = (c.N + kTileRows - 1) / kTileRows;
  p.pairs = (p.row_tiles + 1) / 2;
  p.status = di->status;
  PrefillPlan plan;
  const bool sets = c.offsets != nullptr;
  // Few tokens: a CTA alone per tile. It has no hand-over to another CTA, and twice as many tiles to share out; for it every CTA brings in all
  // of the tile's tokens, in the sets' gathered loads sooner than pays. us, pair / alone: 34816 x 5120 at M = 9 29.6 / 27.9, at 64 32.5 / 31.6, at 77
  // 33.5 / 32.8; 2048 x 2048 at M = 9 6.4 / 4.0; 64 experts of 8 picks, 2048 x 5120 gathered, at 64 / 128 / 200 tokens 101 / 103 / 112 and 99 / 108 / 120,
  // 5120 x 1024 in slot order 67 / 70 / 71 and 63 / 67 / 69, at 300 73.8 and 74.8.
  const bool single = sets ? c.slots <= static_cast<long long>(c.x_rows ? kPSingleGathered : kPSingleMean) * c.sets : c.slots <= kPSingleTN;
  if (!sets && single) {
    const int* slots = cluster_slots<kDense, false>(di->device, di);
    if (!slots) return W4A16_ECUDA;
    plan = plan_single(c.slots, p.row_tiles, c.G, slots, di->smem_optin);
  } else if (!sets) {
    if (int rc = current_plan<kDense>(plan, c.slots, p.row_tiles, p.row_tiles, c.G)) return rc;
  } else {
    const int* slots = single ? cluster_slots<kSets, false>(di->device, di) : cluster_slots<kSets, true>(di->device, di);
    if (!slots) return W4A16_ECUDA;
    // A set is cut into equal tiles of up to 224 tokens, the most whose stages fit: every tile expands the set's weights anew, which costs
    // time up to some 160 tokens (4 TN cycles of MMA against some 650) and power, the limit of a long launch, beyond. Sets that mostly
    // fit 128 take that, which leaves room for six slots of the A operand and three times the weight stages. us in loops of half a second, 160 / 192 / 224: 64
    // experts of 8 picks, 2048 x 5120 gathered, at 300 tokens 128.0 / 127.9 / 128.5, 600 169.7 / 174.1 / 166.6, 800 199 / 195 / 195, 1400 281 / 270 / 262, 3000
    // 514 / 504 / 482, 8192 1295 / 1250 / 1194; 5120 x 1024 in slot order 79.0 / 79.6 / 81.0, 95.7 / 95.9 / 97.2, 111 / 110 / 109, 158 / 152 / 150, 283 / 277 /
    // 273, 713 / 689 / 682. In short runs, 160 / 128: 300 tokens 119.5 / 117.9 and 71.9 / 71.1, 450 134.0 / 132.6 and 76.6 / 76.7, 600 149.3 / 148.7 and 81.6 / 84.1.
    // (Two accumulators of 128 columns, so that a tile is read out under the next one's main loop, gave 1 % at most.)
    plan.pair = !single;
    plan.tn = single ? kPSingleTN : c.slots <= static_cast<long long>(kPSetsMean) * c.sets ? kPSetsNarrow : kPSetsTN;
    plan.clusters = slots[1];
    plan.wdepth = kPMaxWD;
    while (plan.wdepth > kPTeams && prefill_smem(plan.pair, plan.tn, plan.wdepth) + table_bytes(c.sets) > di->smem_optin) plan.wdepth -= kPTeams;
    plan.smem = prefill_smem(plan.pair, plan.tn, plan.wdepth) + table_bytes(c.sets);
    W4_REQUIRE(plan.smem <= di->smem_optin, "experts_linear: %d bytes of shared memory", plan.smem);
  }
  if (single) p.pairs = p.row_tiles;
  p.tn = plan.tn;
  p.splits = plan.splits;
  p.wdepth = plan.wdepth;
  p.full_tt = plan.full_tt;
  p.tiles = plan.tiles;
  if (int rc = encode_acts(&p.amap, c.x, c.K, c.x_tokens, c.x_rows ? 1 : single ? plan.tn : plan.tn / 2)) return rc;
  if (single) return sets ? enqueue_prefill<kSets, false>(p, plan, stream) : enqueue_prefill<kDense, false>(p, plan, stream);
  return sets ? enqueue_prefill<kSets, true>(p, plan, stream) : enqueue_prefill<kDense, true>(p, plan, stream);
}
}  // namespace w4a16

extern "C" {

int w4a16_gemm_prefill(uint16_t* C, const w4a16_weights_t* w, const uint16_t* A, int M, w4a16_workspace_t* ws,
                       void* stream) {
  PrefillParams p = {};
  p.ldc = w ? w->out_f : 0;
  return launch_prefill(p, C, w, A, M, ws, stream);
}

int w4a16_prefill_plan(int M, int out_f, int in_f, int* tokens_per_tile, int* k_splits) {
  W4_REQUIRE(tokens_per_tile != nullptr && k_splits != nullptr, "prefill_plan: null output");
  W4_REQUIRE(M >= 1 && out_f > 0 && out_f % kRowGranule == 0 && in_f > 0 && in_f % kGroup == 0,
             "prefill_plan: M = %d, %d x %d", M, out_f, in_f);
  PrefillPlan plan;
  const int row_tiles = (out_f + kTileRows - 1) / kTileRows;
  if (int rc = current_plan<kPlain>(plan, M, row_tiles, row_tiles, in_f / kGroup)) return rc;
  *tokens_per_tile = plan.tn;
  *k_splits = plan.splits;
  return W4A16_OK;
}

int w4a16_gemm_prefill_sharded(uint16_t* const* C_peers, const w4a16_comm_t* comm, int out_f_total, int row_begin,
                               const w4a16_weights_t* w_shard, const uint16_t* A, int M, w4a16_workspace_t* ws,
                               void* stream) {
  W4_REQUIRE(C_peers != nullptr && comm != nullptr && w_shard != nullptr, "gemm_prefill_sharded: null argument");
  if (comm->nranks < 1 || comm->nranks > 8 || comm->rank < 0 || comm->rank >= comm->nranks)
    return fail(W4A16_ECOMM, "gemm_prefill_sharded: rank %d of %d (1..8 ranks)", comm->rank, comm->nranks);
  if (row_begin < 0 || row_begin % kRowGranule != 0 || row_begin + w_shard->out_f > out_f_total)
    return fail(W4A16_ECOMM, "gemm_prefill_sharded: rows [%d,%d) outside [0,%d)", row_begin, row_begin + w_shard->out_f,
                out_f_total);
  PrefillParams p = {};
  p.ldc = out_f_total;
  p.col0 = row_begin;
  for (int r = 0; r < comm->nranks; ++r) {
    if (C_peers[r] == nullptr || comm->blocks[r] == nullptr)
      return fail(W4A16_ECOMM, "gemm_prefill_sharded: null output or flag block of rank %d", r);
    p.comm_peers[r] = comm->blocks[r];
    if (r != comm->rank) p.C_peers[p.npeers++] = C_peers[r];
  }
  p.comm_local = comm->blocks[comm->rank];
  p.comm_n = comm->nranks;
  p.comm_rank = comm->rank;
  return launch_prefill(p, C_peers[comm->rank], w_shard, A, M, ws, stream);
}

}  // extern "C"
