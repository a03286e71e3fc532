// Products in 8-bit integers with a scale for each token and each channel, and the gated
// feed-forward block made of two of them:
//   out[t, n] = round( ((float) sum_k x[t, k] w[n, k]) * xs[t] * ws[n] + bias[n] )
//   h[t, i]   = silu(gate) * up  of the products with rows i and I + i of w13, in fp32
// The sums are exact 32-bit integers (at most 2^17 - 1 products of at most 2^14), so they do
// not depend on how the depth is split or in which order the parts are added; what follows is
// fp32 and one rounding to the output's type.
//
// tcgen05 kind::i8, operands by TMA as 128-byte-swizzled K-major boxes of 128 bytes of depth.
// Two forms:
//  * int8_stream_kernel (few tokens; bound by the weights' stream). 128 weight rows are the
//    MMA's M side and up to 128 tokens its N side, so one token costs one column and the
//    tokens' padding costs no memory traffic. Few tiles do not fill the GPU: the CTAs of a
//    cluster share a tile's depth and exchange their integer parts through distributed shared
//    memory, each adding and finishing its share of the tokens. No workspace, no atomics, no counters.
//  * int8_tile_kernel (many tokens; bound by the tensor pipe). A CTA pair owns 256 tokens x
//    256 weight rows (cta_group::2: each CTA stages half of either operand, half the shared
//    memory traffic of two single tiles), persistent, with two accumulators in TMEM so that
//    the epilogue of one tile runs under the products of the next.
// A gated tile takes gate rows and the up rows of the same features together: 64 and 64 as the
// 128 rows of the stream form (they meet in shared memory, where its parts are added anyway),
// 128 and 128 as the two halves of the tile form's columns (one TMEM lane then holds both).
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "megamoe.h"
#include "mm_dense.cuh"
#include "mm_kernels.cuh"
#include "mm_ptx.cuh"

namespace mm {
namespace {

constexpr int kBlockK = 128;          // depth of a stage, bytes
constexpr int kRowsM = 128;           // the MMA's rows of a CTA: weight rows, or a pair's half of tokens
constexpr int kBoxBytes = kRowsM * kBlockK;

// Up to this many tokens the stream form always, beyond it what the estimates say (us).
constexpr int kTileTokens = 128;
constexpr double kTileUs = 4.0, kTileColumnUs = 0.346 / 448;  // a launch; a column of a block of depth
constexpr double kStreamUs = 7.5, kStreamBlockUs = 0.45;      // a round of 128-token CTAs; a block

// In place of a part that a CTA could not compute: parts are sums of at most 2^17 - 1 products
// of at most 2^14 in magnitude.
constexpr int kNoPart = INT32_MIN;

// Error word of this file's launches: bounded waits that ran out (mm_int8_check).
__device__ uint32_t g_int8_error;

struct alignas(64) Int8Args {
  CUtensorMap w_map;    // {depth, rows, planes}: plane 1 holds the up rows of w13
  CUtensorMap x_map;    // {depth, tokens}
  CUtensorMap out_map;  // {features, tokens}, where stage_out
  const float *x_scale, *w_scale, *bias;
  void *out;
  int64_t ld_out;
  int tokens, features, blocks_k;
  int out_type;
  int stage_out;        // output rows start and end on 16-byte boundaries: TMA stores (a store
                        // that ends inside a 16-byte unit also writes the rest of the unit)
  int has_clamp;
  float clamp;
  int token_tiles, feature_tiles, tile_n;  // of the tile form
  int w_early;          // the launch's predecessors do not write the weights: load before waiting
  int split;            // CTAs of a cluster that share a tile's depth (stream form), a power of two
  int withhold;         // mm_int8_withhold: this rank's CTAs leave out a load; -1: none
  uint64_t wait_ns;     // budget of every bounded wait (mm_int8_set_wait_budget)
};

// A bounded wait for the phase of `bar` with this parity (CLUSTER: other CTAs arrive on it too).
// One that runs out sets the error word, for the host alone, and `failed`, this CTA's own, at which
// the CTA's other waits give up; no other launch's waits do.
template <bool CLUSTER>
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile uint32_t *failed, uint32_t code, uint64_t budget_ns) {
  auto there = [&] { return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (there()) return true;
  const uint64_t t0 = globaltimer();
#pragma unroll 1
  for (uint32_t i = 0;; ++i) {
    if (there()) return true;
    if ((i & 63u) == 0u) {
      if (*failed) return false;
      if (globaltimer() - t0 > budget_ns) {
        error_raise(&g_int8_error, code);
        *failed = 1u;
        __threadfence_block();
        return false;
      }
    }
  }
}

// A whole warp waits, one elected lane issues: the lanes go on together, or give up together.
__device__ __forceinline__ bool warp_agrees(bool ok) { return __all_sync(0xffffffffu, ok); }

__device__ __forceinline__ float gate_up(const Int8Args &p, float g, float u) {
  if (p.has_clamp) {
    // NaN stays NaN: comparisons instead of fminf / fmaxf
    g = g > p.clamp ? p.clamp : g;
    u = u > p.clamp ? p.clamp : u;
    u = u < -p.clamp ? -p.clamp : u;
  }
  return __fmul_rn(u, __fdiv_rn(g, __fadd_rn(1.0f, expf(-g))));
}

// PER (two or four) consecutive features of one token, `left` of them inside the row.
template <int PER>
__device__ __forceinline__ void store_some(const Int8Args &p, int64_t at, int left, const float (&v)[PER], bool wide) {
  if (p.out_type == MM_DTYPE_FP32) {
    float *o = static_cast<float *>(p.out) + at;
    if (wide && left >= PER) {
      if constexpr (PER == 4) *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<float2 *>(o) = make_float2(v[0], v[1]);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < left) o[i] = v[i];
    }
  } else {
    uint16_t h[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      h[i] = p.out_type == MM_DTYPE_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[i]))
                                         : __half_as_ushort(__float2half_rn(v[i]));
    uint16_t *o = static_cast<uint16_t *>(p.out) + at;
    if (wide && left >= PER) {
      const uint32_t lo = h[0] | static_cast<uint32_t>(h[1]) << 16;
      if constexpr (PER == 4) *reinterpret_cast<uint2 *>(o) = make_uint2(lo, h[2] | static_cast<uint32_t>(h[3]) << 16);
      else *reinterpret_cast<uint32_t *>(o) = lo;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < left) o[i] = h[i];
    }
  }
}

// ---------------------------------------------------------------------------------------
// The stream form. Two CTAs share an SM (at most 113 KB each), so that one's start, its
// accumulator read and its reduction run under the other's loads.
template <int BN, bool GATED>
struct Stream {
  static constexpr int kFeatures = GATED ? kRowsM / 2 : kRowsM;  // of a tile
  static constexpr int kStageBytes = kBoxBytes + BN * kBlockK;
  static constexpr int kRing = 108 * 1024;
  static constexpr int kStages = kRing / kStageBytes;
  static constexpr int kCols = BN < 32 ? 32 : BN;  // TMEM columns, a power of two
  static constexpr int kSmem = kStages * kStageBytes + 1024 + 256;
  // Parts are sent where they are few and read where they are many (us, sent against read: 1 x
  // 4096 x 7168 7.3 and 7.7, 16 x 7168 x 7168 10.6 and 11.0, 64 x 7168 x 7168 12.9 and 12.4, 128 x
  // 7168 x 7168 16.5 and 15.0): a send moves 4 bytes a lane, a read 16.
  static constexpr bool kPush = BN <= 32;
  // Warp 0 loads, warp 1 issues the products, kGroups of four warps read the sums, all of them add
  // the parts. More warps start later and finish more tokens at once (us with 6, 8 and 10: 1 x 7168
  // x 2048 4.6, 4.8, 4.9; 64 x 2048 x 7168 7.95, 7.6, 7.6; 80 x 2048 x 7168 8.8, 9.1, 8.7; 128 x 18432 x 7168
  // 26.9, 26.0, 25.8).
  static constexpr int kWarps = BN <= 32 ? 6 : BN == 64 ? 8 : 10;
  static constexpr int kGroups = (kWarps - 2) / 4;
  static_assert(kStages >= 2 && kCols <= 256, "two CTAs an SM share 512 columns");
  static_assert(BN * kRowsM * 4 <= kStages * kStageBytes, "the parts take the ring's place");
};

template <int BN, bool GATED>
__global__ void __launch_bounds__(Stream<BN, GATED>::kWarps * 32) int8_stream_kernel(const __grid_constant__ Int8Args p) {
  using S = Stream<BN, GATED>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  uint8_t *ring_ptr = smem_raw + (ring - raw);
  const uint32_t bars = ring + S::kStages * S::kStageBytes;
  const uint32_t full = bars, empty = bars + 8 * S::kStages, acc = bars + 16 * S::kStages, recv = acc + 8, slot = recv + 8;
  __shared__ float x_scale[BN];
  uint32_t *slot_ptr = reinterpret_cast<uint32_t *>(ring_ptr + (slot - ring));
  volatile uint32_t *failed = slot_ptr + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int f0 = (blockIdx.x / split) * S::kFeatures;
  const int t0 = blockIdx.y * BN, live = min(BN, p.tokens - t0);
  const int kb0 = p.blocks_k * rank / split, kb1 = p.blocks_k * (rank + 1) / split;
  const int n = kb1 - kb0;

  if (warp == 0 && lane == 0) {
    // the weights do not depend on the launch before this one: bring the first stages into L2
    tma_prefetch_desc(&p.w_map);
    tma_prefetch_desc(&p.x_map);
#pragma unroll 1
    for (int i = 0; i < n && i < S::kStages; ++i)
#pragma unroll
      for (int a = 0; a < kRowsM / S::kFeatures; ++a) tma_prefetch_3d(&p.w_map, (kb0 + i) * kBlockK, f0, a);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(acc, 1);
    mbar_init(recv, 1);
    *failed = 0u;
    fence_barrier_init();
    // a part of each token that this CTA finishes, from every CTA
    const int mine = (live - rank + split - 1) / split;
    if (S::kPush && split > 1 && mine > 0) mbar_expect_tx(recv, mine * split * kRowsM * 4);
  }
  if (warp == 1) {
    tmem_alloc(slot, S::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot_ptr;
  // Dependents start only now. After the allocation: a dependent's CTA that started sooner
  // could take the TMEM columns that a CTA of this launch on the same SM still waits for, and
  // then wait for this launch to end. After the wait: whatever ran before this launch's
  // predecessor has ended by then, so that a launch two further on, whose own predecessor is
  // known not to write its weights, may load them at once (w_early).
  if (warp != 0) {
    pdl_wait();
    pdl_launch_dependents();
  }

  if (warp == 0) {
    const uint64_t stream_once = policy_evict_first(), keep = policy_evict_last();
    auto load_w = [&](int i) {
      const uint32_t stage = ring + (i % S::kStages) * S::kStageBytes, bar = full + 8 * (i % S::kStages);
      mbar_expect_tx(bar, S::kStageBytes);
#pragma unroll
      for (int a = 0; a < kRowsM / S::kFeatures; ++a)
        tma_load_3d(stage + a * S::kFeatures * kBlockK, &p.w_map, (kb0 + i) * kBlockK, f0, a, bar, gridDim.y > 1 ? keep : stream_once);
    };
    const int loads = n - (p.withhold == rank ? 1 : 0);
    const int early = p.w_early ? min(loads, S::kStages) : 0;
    if (elect_one())
      for (int i = 0; i < early; ++i) load_w(i);
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    int i = 0;
    for (; i < loads; ++i) {
      const int s = i % S::kStages;
      if (i >= S::kStages &&
          !warp_agrees(wait_for<false>(empty + 8 * s, ((i / S::kStages) - 1) & 1, failed, kErrTimeoutEmpty, p.wait_ns)))
        break;
      if (elect_one()) {
        if (i >= early) load_w(i);
        tma_load_2d(ring + s * S::kStageBytes + kBoxBytes, &p.x_map, (kb0 + i) * kBlockK, t0, full + 8 * s, keep);
      }
      __syncwarp();
    }
    // leave no copy in flight, whatever ended the loop
    for (int j = max(0, i - S::kStages); j < i; ++j) mbar_wait_drain(full + 8 * (j % S::kStages), (j / S::kStages) & 1);
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_i8(kRowsM, BN);
    for (int i = 0; i < n; ++i) {
      const int s = i % S::kStages;
      if (!warp_agrees(wait_for<false>(full + 8 * s, (i / S::kStages) & 1, failed, kErrTimeoutFull, p.wait_ns))) break;
      tc_fence_after();
      const uint32_t stage = ring + s * S::kStageBytes;
      const uint64_t w = smem_desc(stage, 16, 1024, kLayoutSw128);
      const uint64_t b = smem_desc(stage + kBoxBytes, 16, 1024, kLayoutSw128);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kBlockK / 32; ++k)  // 32 bytes of depth an instruction
          tc_mma_i8(tmem, w + 2 * k, b + 2 * k, idesc, i > 0 || k > 0);
        tc_commit(empty + 8 * s);
      }
      __syncwarp();
    }
    if (elect_one()) tc_commit(acc);
    __syncwarp();
    mbar_wait_drain(acc, 0);
    __syncwarp();
  }

  // a lane finishes PER neighbouring features of a token
  constexpr int PER = S::kFeatures / 32;
  const int es = p.out_type == MM_DTYPE_FP32 ? 4 : 2;
  const bool wide = reinterpret_cast<uintptr_t>(p.out) % (PER * es) == 0 && p.ld_out % PER == 0;
  const int f = f0 + PER * lane;
  const int left = p.features - f;
  float ws[PER], second[PER];  // second: the bias, or the up rows' scales
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    ws[i] = i < left ? p.w_scale[f + i] : 0.0f;
    second[i] = i >= left ? 0.0f : GATED ? p.w_scale[static_cast<int64_t>(p.features) + f + i] : p.bias ? p.bias[f + i] : 0.0f;
  }
  if (warp >= 2 && threadIdx.x - 64 < live) x_scale[threadIdx.x - 64] = p.x_scale[t0 + threadIdx.x - 64];
  const bool ok = warp_agrees(wait_for<false>(acc, 0, failed, kErrTimeoutAcc, p.wait_ns) && *failed == 0u);
  if (!ok) pause_drain();  // copies still in flight land before this CTA's marks below, not over them
  tc_fence_after();
  // Every CTA of the cluster finishes the tokens rank, rank + split, ... Groups of four warps read the
  // sums (warp w: TMEM lanes 32 (w % 4) and on, weight rows; a column a token), 16 tokens in turn.
  const int q = warp & 3, group = warp < 2 ? -1 : (warp - 2) >> 2;
  const uint32_t sums = tmem + (static_cast<uint32_t>(q * 32) << 16);
  auto finish = [&](int j, int4 sum, int least) {
    const float xs = least != kNoPart ? x_scale[j] : __uint_as_float(0x7fc00000u);  // NaN where a part is missing
    const float a[4] = {__fmul_rn(static_cast<float>(sum.x), xs), __fmul_rn(static_cast<float>(sum.y), xs),
                        __fmul_rn(static_cast<float>(sum.z), xs), __fmul_rn(static_cast<float>(sum.w), xs)};
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if constexpr (GATED) v[i] = gate_up(p, __fmul_rn(a[i], ws[i]), __fmul_rn(a[PER + i], second[i]));
      else v[i] = __fmaf_rn(a[i], ws[i], second[i]);
    }
    if (left > 0) store_some<PER>(p, (t0 + j) * p.ld_out + f, left, v, wide);
  };
  // The four sums of a lane: four features, or two features' gate and up. A CTA that gave up leaves
  // kNoPart, which no part can be, where its sums are missing; neighbours among the four come from
  // one of its warps, and are missing together.
  int least;
  auto add = [&](int4 &sum, const int4 &v) {
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    least = min(least, GATED ? min(v.x, v.z) : v.x);
  };
  auto parts = [&](int j, uint32_t (&r)[16]) {
    tc_ld_32x32b_x16(sums + j, r);
    tc_wait_ld();
    if (!ok) {
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = static_cast<uint32_t>(kNoPart);
    }
  };
  if (S::kPush && split > 1) {
    // The parts go into the ring of the CTA that finishes their token, once every CTA of the
    // cluster is past its products: [token's turn][part][weight row].
    cluster_arrive();
    if (group >= 0 && group < S::kGroups) {
      const int turns = __ffs(split) - 1;  // split is a power of two
      const uint32_t at = ring + (rank * kRowsM + q * 32 + lane) * 4;
#pragma unroll 1
      for (int j = 16 * group; j < live; j += 16 * S::kGroups) {
        uint32_t r[16];
        parts(j, r);
        if (j == 16 * group) cluster_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int owner = (j + i) & (split - 1), turn = (j + i) >> turns;
          if (j + i < live)
            cluster_store_async(cluster_map(at + turn * split * kRowsM * 4, owner), r[i], cluster_map(recv, owner));
        }
      }
    } else {
      cluster_wait();
    }
    tc_fence_before();
    __syncthreads();  // x's scales, and the TMEM reads
    if (warp == 1) tmem_dealloc(tmem, S::kCols);
    if (rank >= live) return;
    const bool came = warp_agrees(wait_for<true>(recv, 0, failed, kErrTimeoutAcc, p.wait_ns));
#pragma unroll 1
    for (int j = rank + split * warp; j < live; j += split * S::kWarps) {
      const int *part = reinterpret_cast<const int *>(ring_ptr) + (j & ~(split - 1)) * kRowsM + PER * lane;
      int4 sum = make_int4(0, 0, 0, 0);
      least = came ? 0 : kNoPart;
#pragma unroll 8
      for (int r = 0; r < split; ++r, part += kRowsM) {
        if constexpr (GATED) {
          const int2 g = *reinterpret_cast<const int2 *>(part), u = *reinterpret_cast<const int2 *>(part + S::kFeatures);
          add(sum, make_int4(g.x, g.y, u.x, u.y));
        } else {
          add(sum, *reinterpret_cast<const int4 *>(part));
        }
      }
      finish(j, sum, least);
    }
    if (!came) cluster_sync();  // parts may still come: stay until their senders are gone
    return;
  }
  // Each CTA leaves its parts in its own ring, [token][weight row], and reads the others' there, from
  // its neighbour on (all from the first CTA's at once: 48 x 2048 x 7168 7.45 us instead of 7.1).
  if (group >= 0 && group < S::kGroups) {
#pragma unroll 1
    for (int j = 16 * group; j < live; j += 16 * S::kGroups) {
      uint32_t r[16];
      parts(j, r);
      uint32_t *to = reinterpret_cast<uint32_t *>(ring_ptr) + j * kRowsM + q * 32 + lane;
#pragma unroll
      for (int i = 0; i < 16; ++i) to[i * kRowsM] = r[i];
    }
  }
  tc_fence_before();
  cluster_sync();
  if (warp == 1) tmem_dealloc(tmem, S::kCols);
#pragma unroll 1
  for (int j = rank + split * warp; j < live; j += split * S::kWarps) {
    const uint32_t at = ring + (j * kRowsM + PER * lane) * 4;
    int4 sum = make_int4(0, 0, 0, 0);
    least = 0;
#pragma unroll 2
    for (int r = 0; r < split; ++r) {
      const uint32_t from = cluster_map(at, (rank + r) & (split - 1));
      if constexpr (GATED) {
        const int2 g = cluster_load_v2(from), u = cluster_load_v2(from + 4 * S::kFeatures);
        add(sum, make_int4(g.x, g.y, u.x, u.y));
      } else {
        add(sum, cluster_load_v4(from));
      }
    }
    finish(j, sum, least);
  }
  cluster_sync();  // the parts are read: the CTA may end
}

// ---------------------------------------------------------------------------------------
// The tile form. Per CTA: warp 0 loads, warp 1 (of the pair's leader) issues the products,
// warps 2..9 are the epilogue; every warp of both CTAs walks the same tiles.
constexpr int kTileM = 256;                        // tokens of a pair
constexpr int kTileN = 256;                        // weight rows of a pair at most
// A stage is two blocks of depth, 64 KB of this CTA's halves of both operands: a hand-over
// (full barrier, commit, empty barrier) costs about 225 ns whatever it hands over, a block's
// products 266 ns at 256 columns and 66 at 64. One block a stage: 128 columns 439 us against
// 324 at 8192 x 7168 x 7168, 256 columns the same.
constexpr int kTileBlocks = 2;
constexpr int kTileStages = 3;
constexpr int kTileStageBytes = kTileBlocks * 2 * kBoxBytes;
// Eight epilogue warps: two a quarter of the TMEM lanes take turns by chunks of columns (with
// four, 4096 x 7008 x 512 was bound by them: 34 us).
constexpr int kEpilogueWarps = 8;
constexpr int kTileThreads = 64 + 32 * kEpilogueWarps;
constexpr int kOutBytes = 32 * 64;                 // a staged chunk: 32 rows of 64 bytes
constexpr int kScaleFloats = 2 * (kTileN / 2);     // a warp's columns' scales, and bias or up scales
constexpr int kTileSmem = 1024 + kTileStages * kTileStageBytes + kEpilogueWarps * (kOutBytes + kScaleFloats * 4) + 256;

// The tile of a step: token tiles in groups of 16 (their codes stay in L2 while the weights
// pass by once a group), fastest inside a group.
__device__ __forceinline__ void tile_at(const Int8Args &p, int i, int &tt, int &ft) {
  const int per = 16 * p.feature_tiles;
  const int g = i / per, r = i - g * per;
  const int rows = min(16, p.token_tiles - 16 * g);
  ft = r / rows;
  tt = 16 * g + r - ft * rows;
}

template <typename Out, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTileThreads, 1) int8_tile_kernel(const __grid_constant__ Int8Args p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  uint8_t *base = smem_raw + (ring - raw);
  const uint32_t out_stage = ring + kTileStages * kTileStageBytes;
  float *scales = reinterpret_cast<float *>(base + kTileStages * kTileStageBytes + kEpilogueWarps * kOutBytes);
  const uint32_t bars = out_stage + kEpilogueWarps * (kOutBytes + kScaleFloats * 4);
  const uint32_t full = bars, empty = full + 8 * kTileStages, acc_full = empty + 8 * kTileStages,
                 acc_empty = acc_full + 16, drained = acc_empty + 16, slot = drained + 8;
  uint32_t *slot_ptr = reinterpret_cast<uint32_t *>(base + (slot - ring));
  volatile uint32_t *failed = slot_ptr + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.token_tiles * p.feature_tiles;
  const int half_n = p.tile_n / 2;                 // weight rows that this CTA stages
  const int tile_f = GATED ? half_n : p.tile_n;    // features of a tile

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.w_map);
    tma_prefetch_desc(&p.x_map);
    if (p.stage_out) tma_prefetch_desc(&p.out_map);
    for (int s = 0; s < kTileStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + 8 * b, 1);
      mbar_init(acc_empty + 8 * b, 2 * kEpilogueWarps);  // of both CTAs
    }
    mbar_init(drained, 1);
    *failed = 0u;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_pair_alloc(slot, 512);
    tmem_pair_relinquish();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *slot_ptr;
  // after the allocation and the wait, as in the stream form; the bounded waits below count from here
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    const uint32_t block_tx = 2 * (kBoxBytes + half_n * kBlockK);  // both CTAs' bytes
    int it = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      int tt, ft;
      tile_at(p, tile, tt, ft);
      const int t0 = tt * kTileM + rank * kRowsM;
      const int row = GATED ? ft * tile_f : ft * tile_f + rank * half_n, plane = GATED ? rank : 0;
      for (int kb = 0; kb < p.blocks_k; kb += kTileBlocks, ++it) {
        if (p.withhold == rank && kb + kTileBlocks >= p.blocks_k) {  // of the first tile
          ok = false;
          break;
        }
        const int s = it % kTileStages;
        if (it >= kTileStages &&
            !warp_agrees(wait_for<true>(empty + 8 * s, ((it / kTileStages) - 1) & 1, failed, kErrTimeoutEmpty, p.wait_ns))) {
          ok = false;
          break;
        }
        const uint32_t stage = ring + s * kTileStageBytes;
        // the leader's barrier counts the bytes of both CTAs: this CTA's copies may land
        // there before the leader expects them, the phase still ends with its arrival
        const uint32_t bar = cluster_map(full + 8 * s, 0);
        const int blocks = min(kTileBlocks, p.blocks_k - kb);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(full + 8 * s, blocks * block_tx);
          for (int j = 0; j < blocks; ++j) {
            tma_pair_load_2d(stage + 2 * j * kBoxBytes, &p.x_map, (kb + j) * kBlockK, t0, bar);
            tma_pair_load_3d(stage + (2 * j + 1) * kBoxBytes, &p.w_map, (kb + j) * kBlockK, row, plane, bar);
          }
        }
        __syncwarp();
      }
    }
    // leave no copy in flight: the last stages' barriers complete with both CTAs' copies
    if (rank == 0)
      for (int j = max(0, it - kTileStages); j < it; ++j)
        mbar_wait_drain(full + 8 * (j % kTileStages), (j / kTileStages) & 1);
    // where either CTA stopped early, the other's later copies are on no barrier that completes
    if (!ok) pause_drain();
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = idesc_i8(kTileM, p.tile_n);
      int it = 0, n = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs, ++n) {
        const int b = n & 1;
        if (n >= 2 && !warp_agrees(wait_for<true>(acc_empty + 8 * b, ((n >> 1) - 1) & 1, failed, kErrTimeoutAcc, p.wait_ns))) break;
        tc_fence_after();
        for (int kb = 0; kb < p.blocks_k; kb += kTileBlocks, ++it) {
          const int s = it % kTileStages;
          if (!warp_agrees(wait_for<true>(full + 8 * s, (it / kTileStages) & 1, failed, kErrTimeoutFull, p.wait_ns))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t stage = ring + s * kTileStageBytes;
          const int blocks = min(kTileBlocks, p.blocks_k - kb);
          if (elect_one()) {
            for (int j = 0; j < blocks; ++j) {
              const uint64_t x = smem_desc(stage + 2 * j * kBoxBytes, 16, 1024, kLayoutSw128);
              const uint64_t w = smem_desc(stage + (2 * j + 1) * kBoxBytes, 16, 1024, kLayoutSw128);
#pragma unroll
              for (int k = 0; k < kBlockK / 32; ++k)
                tc_pair_mma_i8(tmem + b * kTileN, x + 2 * k, w + 2 * k, idesc, kb > 0 || j > 0 || k > 0);
            }
            tc_pair_commit(empty + 8 * s);
          }
          __syncwarp();
        }
        if (ok && elect_one()) tc_pair_commit(acc_full + 8 * b);
        __syncwarp();
      }
      if (elect_one()) tc_pair_commit(drained);
      __syncwarp();
      mbar_wait_drain(drained, 0);
    }
    __syncwarp();
  } else {
    constexpr int CH = 64 / sizeof(Out);           // columns of a chunk
    const int q = warp & 3, e = warp - 2;          // TMEM lanes 32 q and on: token rows
    const int half = e >> 2;                       // this warp's chunks: half, half + 2, ...
    float *ws = scales + e * kScaleFloats, *second = ws + kScaleFloats / 2;  // second: the bias, or the up rows' scales
    const uint32_t mine = out_stage + e * kOutBytes;
    // a tile's scales: this lane's share, fetched while the tile before it is finished
    constexpr int PER_LANE = kScaleFloats / 2 / 32;
    float next_w[PER_LANE], next_s[PER_LANE], next_x = 0.0f;
    auto fetch = [&](int tile) {
      int tt, ft;
      tile_at(p, tile, tt, ft);
      const int t = tt * kTileM + rank * kRowsM + q * 32 + lane, f0 = ft * tile_f, end = min(p.features, f0 + tile_f);
      next_x = t < p.tokens ? p.x_scale[t] : 0.0f;
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k) {
        const int i = k * 32 + lane, f = f0 + (2 * (i / CH) + half) * CH + i % CH;  // its place among this warp's chunks
        next_w[k] = f < end ? p.w_scale[f] : 0.0f;
        next_s[k] = f >= end ? 0.0f : GATED ? p.w_scale[p.features + f] : p.bias ? p.bias[f] : 0.0f;
      }
    };
    if (pair < tiles) fetch(pair);
    int n = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles; tile += pairs, ++n) {
      const int b = n & 1;
      int tt, ft;
      tile_at(p, tile, tt, ft);
      const int t0 = tt * kTileM + rank * kRowsM + q * 32, f0 = ft * tile_f;
      float xs = next_x;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k) {
        ws[k * 32 + lane] = next_w[k];
        second[k * 32 + lane] = next_s[k];
      }
      __syncwarp();
      if (tile + pairs < tiles) fetch(tile + pairs);
      // after a wait that ran out, this and the tiles that follow are NaN, not the memory's old values
      ok = ok && warp_agrees(wait_for<true>(acc_full + 8 * b, (n >> 1) & 1, failed, kErrTimeoutAcc, p.wait_ns));
      if (!ok) xs = __uint_as_float(0x7fc00000u);
      tc_fence_after();
      const uint32_t from = tmem + (static_cast<uint32_t>(q * 32) << 16) + b * kTileN;
      for (int c = half * CH, i0 = 0; c < tile_f; c += 2 * CH, i0 += CH) {
        uint32_t r[CH], u[GATED ? CH : 1];
        if constexpr (CH == 32) tc_ld_32x32b_x32(from + c, r);
        else tc_ld_32x32b_x16(from + c, r);
        if constexpr (GATED) tc_ld_32x32b_x16(from + half_n + c, u);
        tc_wait_ld();
        if (c + 2 * CH >= tile_f) {
          // this warp's columns are in registers: the pair's next but one tile may overwrite them
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_map(acc_empty + 8 * b, 0));
        }
        float v[CH];
#pragma unroll
        for (int j = 0; j < CH; j += 4) {
          const float4 w4 = *reinterpret_cast<const float4 *>(ws + i0 + j), s4 = *reinterpret_cast<const float4 *>(second + i0 + j);
          const float w[4] = {w4.x, w4.y, w4.z, w4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = __fmul_rn(static_cast<float>(static_cast<int>(r[j + i])), xs);
            if constexpr (GATED)
              v[j + i] = gate_up(p, __fmul_rn(a, w[i]), __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(u[j + i])), xs), s[i]));
            else
              v[j + i] = __fmaf_rn(a, w[i], s[i]);
          }
        }
        uint32_t word[16];  // the row's 64 bytes
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (sizeof(Out) == 4) {
            word[i] = __float_as_uint(v[i]);
          } else {
            union { uint32_t w; Out h[2]; } pk;
            pk.h[0] = Out(v[2 * i]);
            pk.h[1] = Out(v[2 * i + 1]);
            word[i] = pk.w;
          }
        }
        uint8_t *buf = base + (mine - ring);
        if (p.stage_out) {
          // this warp's 32 rows, swizzled as the map says (16-byte units XORed with the row, so
          // that eight lanes' stores meet no bank twice), then one store
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4 *>(buf + lane * 64 + ((i ^ ((lane >> 1) & 3)) * 16)) =
                make_uint4(word[4 * i], word[4 * i + 1], word[4 * i + 2], word[4 * i + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && t0 < p.tokens && f0 + c < p.features) {
            tma_store_2d(&p.out_map, mine, f0 + c, t0);
            bulk_commit_group();
          }
        } else {
          // rows that TMA cannot store: turned in shared memory (words XORed with the row), then
          // whole rows an instruction, one of 16-bit columns or two of fp32
          uint32_t *turn = reinterpret_cast<uint32_t *>(buf);
#pragma unroll
          for (int i = 0; i < 16; ++i) turn[lane * 16 + (i ^ (lane & 15))] = word[i];
          __syncwarp();
          constexpr int AT_ONCE = 32 / CH;
          const int col = lane & (CH - 1), rows = min(32, p.tokens - t0);
          if (f0 + c + col < p.features) {
            Out *o = static_cast<Out *>(p.out) + static_cast<int64_t>(t0) * p.ld_out + f0 + c + col;
#pragma unroll 8
            for (int j = lane / CH; j < rows; j += AT_ONCE) {
              const Out *at = reinterpret_cast<const Out *>(turn + j * 16 + ((col * static_cast<int>(sizeof(Out)) / 4) ^ (j & 15)));
              o[j * p.ld_out] = at[sizeof(Out) == 4 ? 0 : col & 1];
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();
  if (warp == 1) tmem_pair_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------------------
// Host side
typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                             const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encoder(EncodeFn *fn) {
  static EncodeFn cached = nullptr;
  if (cached == nullptr) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess || p == nullptr || q != cudaDriverEntryPointSuccess)
      return set_error(MM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cached = reinterpret_cast<EncodeFn>(p);
  }
  *fn = cached;
  return MM_OK;
}

// Boxes of 128 (or 64) bytes by `box_rows` rows with the swizzle of that width; out-of-range
// elements read as zero and are not written, so odd depths, tokens and features need no padding.
int encode(CUtensorMap *map, CUtensorMapDataType type, int es, const void *base, int64_t cols, int64_t rows_total,
           int64_t planes, int64_t ld, int box_rows, int box_bytes = 128) {
  EncodeFn fn;
  if (const int rc = encoder(&fn)) return rc;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows_total), static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * es), static_cast<cuuint64_t>(ld * es * rows_total)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_bytes / es), static_cast<cuuint32_t>(box_rows), 1u};
  const cuuint32_t step[3] = {1u, 1u, 1u};
  const CUresult r = fn(map, type, planes ? 3 : 2, const_cast<void *>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(MM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return MM_OK;
}

template <typename K>
cudaError_t raise_smem(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

template <typename K>
cudaError_t launch_cluster(K kernel, dim3 grid, int threads, int smem, int cluster, void *stream, const Int8Args &a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// The budget of the bounded waits, and what mm_int8_withhold asked for: of this process's launches.
std::atomic<int64_t> g_wait_ns{static_cast<int64_t>(kWaitBudgetNs)};
std::atomic<int> g_withhold_rank{0}, g_withhold_launches{0};

int withheld() {
  for (int n = g_withhold_launches.load(); n > 0;)
    if (g_withhold_launches.compare_exchange_weak(n, n - 1)) return g_withhold_rank.load();
  return -1;
}

// CTAs of a cluster that share a tile's depth: enough CTAs for most SMs, each with at least two
// blocks of depth.
int stream_split(int64_t tiles, int blocks_k) {
  int split = 1;
  while (split < 8 && tiles * split < 148 && 4 * split <= blocks_k) split *= 2;
  return split;
}

template <int BN, bool GATED>
cudaError_t launch_stream(Int8Args &a, void *stream) {
  using S = Stream<BN, GATED>;
  static bool done[64] = {};
  const cudaError_t e = raise_smem(int8_stream_kernel<BN, GATED>, S::kSmem, done);
  if (e != cudaSuccess) return e;
  const int tiles = (a.features + S::kFeatures - 1) / S::kFeatures, token_tiles = (a.tokens + BN - 1) / BN;
  a.split = stream_split(tiles * token_tiles, a.blocks_k);
  return launch_cluster(int8_stream_kernel<BN, GATED>, dim3(tiles * a.split, token_tiles), S::kWarps * 32, S::kSmem, a.split, stream, a);
}

// CTA pairs that the current device runs at once (of the tile form: one CTA an SM, all its
// forms alike), the persistent grid's size. 0: not known.
int sm_pairs() {
  static int cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!cached[dev]) {
    static bool done[64] = {};
    if (raise_smem(int8_tile_kernel<float, true>, kTileSmem, done) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(256);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = kTileSmem;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, int8_tile_kernel<float, true>, &cfg) != cudaSuccess) return 0;
    cached[dev] = clusters;
  }
  return cached[dev];
}

template <typename Out, bool GATED>
cudaError_t launch_tile(Int8Args &a, int pairs, void *stream) {
  static bool done[64] = {};
  const cudaError_t e = raise_smem(int8_tile_kernel<Out, GATED>, kTileSmem, done);
  if (e != cudaSuccess) return e;
  const int tiles = a.token_tiles * a.feature_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(tiles, pairs));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = kTileSmem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int8_tile_kernel<Out, GATED>, a);
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

struct Product {
  const int8_t *x;
  int64_t ld_x;
  const float *x_scale;
  const int8_t *w;
  int64_t ld_w;
  const float *w_scale, *bias;
  void *out;
  int64_t ld_out;
  int out_type, tokens, features, depth;  // gated: features of h, w holds twice as many rows
  bool gated;
  float clamp;
  bool out_pad;         // the columns from features to ld_out may be written
  bool w_early;         // see Int8Args
};

int check(const char *what, const Product &q) {
  if (q.tokens < 0 || q.features < 1 || q.depth < 1)
    return set_error(MM_ERR_INVALID, "%s: %d tokens, %d features, depth %d", what, q.tokens, q.features, q.depth);
  if (q.features > 1 << 30) return set_error(MM_ERR_UNSUPPORTED, "%s: %d features: at most 2^30", what, q.features);
  if (q.tokens >= 1 << 23) return set_error(MM_ERR_UNSUPPORTED, "%s: %d tokens: fewer than 2^23 a call", what, q.tokens);
  if (q.depth >= 1 << 17)
    return set_error(MM_ERR_UNSUPPORTED, "%s: depth %d: 32-bit sums hold fewer than 131072 products", what, q.depth);
  if (q.out_type != MM_DTYPE_BF16 && q.out_type != MM_DTYPE_FP16 && q.out_type != MM_DTYPE_FP32)
    return set_error(MM_ERR_INVALID, "%s: unknown output type %d", what, q.out_type);
  if (q.tokens == 0) return MM_OK;
  if (!q.x || !q.x_scale || !q.w || !q.w_scale || !q.out) return set_error(MM_ERR_INVALID, "%s: null pointer", what);
  if (q.ld_x < q.depth || q.ld_w < q.depth || q.ld_out < q.features)
    return set_error(MM_ERR_INVALID, "%s: a row stride below the row's length", what);
  if (!aligned(q.x, 16) || !aligned(q.w, 16) || q.ld_x % 16 || q.ld_w % 16)
    return set_error(MM_ERR_INVALID, "%s: int8 rows must start on 16-byte boundaries", what);
  if (!aligned(q.x_scale, 4) || !aligned(q.w_scale, 4) || !aligned(q.bias, 4) || !aligned(q.out, q.out_type == MM_DTYPE_FP32 ? 4 : 2))
    return set_error(MM_ERR_INVALID, "%s: a misaligned pointer", what);
  const int es = q.out_type == MM_DTYPE_FP32 ? 4 : 2;
  const int64_t w_rows = q.gated ? 2 * static_cast<int64_t>(q.features) : q.features;
  auto written = [&](const Bytes &b) { return overlap(row_bytes(q.out, q.tokens, q.features, q.ld_out, es), b); };
  if (written(row_bytes(q.x, q.tokens, q.depth, q.ld_x, 1)) || written(row_bytes(q.w, w_rows, q.depth, q.ld_w, 1)) ||
      written(flat_bytes(q.x_scale, q.tokens * 4ll)) || written(flat_bytes(q.w_scale, w_rows * 4)) ||
      written(flat_bytes(q.bias, q.features * 4ll)))
    return set_error(MM_ERR_INVALID, "%s: the output overlaps an input", what);
  return MM_OK;
}

int run(const char *what, const Product &q, void *stream) {
  Int8Args a = {};
  a.x_scale = q.x_scale;
  a.w_scale = q.w_scale;
  a.bias = q.bias;
  a.out = q.out;
  a.ld_out = q.ld_out;
  a.tokens = q.tokens;
  a.features = q.features;
  a.blocks_k = (q.depth + kBlockK - 1) / kBlockK;
  a.out_type = q.out_type;
  a.has_clamp = q.clamp > 0.0f;
  a.clamp = q.clamp;
  a.w_early = q.w_early;
  a.wait_ns = static_cast<uint64_t>(g_wait_ns.load());
  a.withhold = withheld();
  auto w_map = [&](int rows) { return encode(&a.w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w, q.depth, q.features, q.gated ? 2 : 1, q.ld_w, rows); };
  int rc;
  auto x_map = [&](int rows) { return encode(&a.x_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.x, q.depth, q.tokens, 0, q.ld_x, rows); };
  cudaError_t e;
  const int pairs = sm_pairs();
  if (pairs < 1) return set_error(MM_ERR_CUDA, "%s: CTA pairs do not fit this device", what);
  // Which form, and the tile form's width, by the time that they take. A tile's time grows with
  // the depth and as its width plus 192 columns (8192 x 7168 x 7168, a tile's share of the whole:
  // 19.4 us at 256 columns, 13.0 at 128, 11.1 at 64). 2048 tokens: 224 columns 72 us, 256 columns
  // 74, 128 columns 87; 1024 x 2048 x 7168: 128 columns 16.1 us, 256 columns 23.1.
  double tile_us = 1e30;
  a.token_tiles = (q.tokens + kTileM - 1) / kTileM;
  for (int n = kTileN; n >= 64; n -= q.gated ? 64 : 32) {
    const int f = q.gated ? n / 2 : n;
    const int64_t tiles = static_cast<int64_t>(a.token_tiles) * ((q.features + f - 1) / f);
    const double us = kTileUs + static_cast<double>((tiles + pairs - 1) / pairs) * a.blocks_k * (n + 192) * kTileColumnUs;
    if (us < tile_us) tile_us = us, a.tile_n = n, a.feature_tiles = (q.features + f - 1) / f;
  }
  const int64_t stream_tiles = (static_cast<int64_t>(q.features) * (q.gated ? 2 : 1) + kRowsM - 1) / kRowsM * ((q.tokens + 127) / 128);
  const int split = stream_split(stream_tiles, a.blocks_k);
  const double stream_us = static_cast<double>((stream_tiles * split + 295) / 296) * (kStreamUs + (a.blocks_k + split - 1) / split * kStreamBlockUs);
  if (q.tokens > kTileTokens && (tile_us <= stream_us || q.tokens > 65535 * 128)) {
    const int es = q.out_type == MM_DTYPE_FP32 ? 4 : 2;
    a.stage_out = aligned(q.out, 16) && q.ld_out * es % 16 == 0 && (q.out_pad || static_cast<int64_t>(q.features) * es % 16 == 0);
    if ((rc = x_map(kRowsM)) || (rc = w_map(a.tile_n / 2))) return rc;
    if (a.stage_out &&
        (rc = encode(&a.out_map, q.out_type == MM_DTYPE_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : q.out_type == MM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                     es, q.out, q.features, q.tokens, 0, q.ld_out, 32, 64)))
      return rc;
    if (q.gated) e = launch_tile<float, true>(a, pairs, stream);
    else if (q.out_type == MM_DTYPE_FP32) e = launch_tile<float, false>(a, pairs, stream);
    else if (q.out_type == MM_DTYPE_BF16) e = launch_tile<__nv_bfloat16, false>(a, pairs, stream);
    else e = launch_tile<__half, false>(a, pairs, stream);
    if (e != cudaSuccess) return set_error(MM_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    return MM_OK;
  }
  if ((rc = w_map(q.gated ? kRowsM / 2 : kRowsM))) return rc;
  int bn = 16;
  while (bn < q.tokens && bn < 128) bn *= 2;
  if ((rc = x_map(bn))) return rc;
  switch (q.gated ? -bn : bn) {
    case 16: e = launch_stream<16, false>(a, stream); break;
    case 32: e = launch_stream<32, false>(a, stream); break;
    case 64: e = launch_stream<64, false>(a, stream); break;
    case 128: e = launch_stream<128, false>(a, stream); break;
    case -16: e = launch_stream<16, true>(a, stream); break;
    case -32: e = launch_stream<32, true>(a, stream); break;
    case -64: e = launch_stream<64, true>(a, stream); break;
    default: e = launch_stream<128, true>(a, stream); break;
  }
  if (e != cudaSuccess) return set_error(MM_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return MM_OK;
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace
}  // namespace mm

using namespace mm;

extern "C" {

int mm_int8_linear(const int8_t *x, int64_t ld_x, const float *x_scale, const int8_t *w, int64_t ld_w,
                   const float *w_scale, const float *bias, void *out, int64_t ld_out, int32_t out_dtype,
                   int32_t tokens, int32_t features, int32_t depth, void *stream) {
  const Product q = {x, ld_x, x_scale, w, ld_w, w_scale, bias, out, ld_out, out_dtype, tokens, features, depth, false, 0.0f, false, false};
  const int rc = check("mm_int8_linear", q);
  if (rc || tokens == 0) return rc;
  return run("mm_int8_linear", q, stream);
}

int64_t mm_int8_ffn_workspace(int32_t tokens, int32_t inter) {
  if (tokens < 1 || inter < 1) return 0;
  return up(tokens * up(inter, 4) * 4, 256) + up(tokens * up(inter, 16), 256) + static_cast<int64_t>(tokens) * 4;
}

int mm_int8_ffn(const mm_int8_ffn_args *f, void *stream) {
  if (!f) return set_error(MM_ERR_INVALID, "mm_int8_ffn: null pointer");
  if (f->clamp < 0.0f || !(f->clamp < INFINITY)) return set_error(MM_ERR_INVALID, "mm_int8_ffn: clamp %g", f->clamp);
  if (f->tokens < 0 || f->inter < 1 || f->inter >= 1 << 30)
    return set_error(MM_ERR_INVALID, "mm_int8_ffn: %d tokens, inter %d", f->tokens, f->inter);
  uint8_t *ws = static_cast<uint8_t *>(f->workspace);
  if (f->tokens > 0 && (!ws || !aligned(ws, 256) || f->workspace_bytes < mm_int8_ffn_workspace(f->tokens, f->inter)))
    return set_error(MM_ERR_INVALID, "mm_int8_ffn: the workspace needs %lld bytes on a 256-byte boundary",
                     static_cast<long long>(mm_int8_ffn_workspace(f->tokens, f->inter)));
  // h in fp32 (its rounding to int8 is the only one), rows on 16-byte boundaries; its codes; scales
  const int64_t ld_h = up(f->inter, 4), ld_q = up(f->inter, 16);
  float *h = reinterpret_cast<float *>(ws);
  int8_t *hq = ws ? reinterpret_cast<int8_t *>(ws + up(f->tokens * ld_h * 4, 256)) : nullptr;
  float *hs = ws ? reinterpret_cast<float *>(hq + up(f->tokens * ld_q, 256)) : nullptr;
  const Product up_q = {f->x, f->ld_x, f->x_scale, f->w13, f->ld_w13, f->w13_scale, nullptr, h, ld_h, MM_DTYPE_FP32,
                        f->tokens, f->inter, f->hidden, true, f->clamp, true, false};
  // the down product's predecessors, the row kernel and the gated product, do not write w2
  const Product down_q = {hq, ld_q, hs, f->w2, f->ld_w2, f->w2_scale, nullptr, f->out, f->ld_out, f->out_dtype,
                          f->tokens, f->hidden, f->inter, false, 0.0f, false, true};
  int rc = check("mm_int8_ffn", up_q);
  if (!rc) rc = check("mm_int8_ffn", down_q);
  if (rc || f->tokens == 0) return rc;
  const Bytes first[] = {row_bytes(f->x, f->tokens, f->hidden, f->ld_x, 1), row_bytes(f->w13, 2ll * f->inter, f->hidden, f->ld_w13, 1),
                         flat_bytes(f->x_scale, f->tokens * 4ll), flat_bytes(f->w13_scale, f->inter * 8ll)};
  const Bytes second[] = {row_bytes(f->w2, f->hidden, f->inter, f->ld_w2, 1), flat_bytes(f->w2_scale, f->hidden * 4ll)};
  const Bytes out = row_bytes(f->out, f->tokens, f->hidden, f->ld_out, f->out_dtype == MM_DTYPE_FP32 ? 4 : 2);
  const Bytes space = flat_bytes(ws, mm_int8_ffn_workspace(f->tokens, f->inter));
  auto in_workspace = [&](const Bytes &b) { return overlap(space, b); };
  for (const Bytes &b : first)  // the down product's own check covers second
    if (overlap(out, b)) return set_error(MM_ERR_INVALID, "mm_int8_ffn: the output overlaps an input");
  if (std::any_of(first, first + 4, in_workspace) || std::any_of(second, second + 2, in_workspace) || in_workspace(out))
    return set_error(MM_ERR_INVALID, "mm_int8_ffn: the workspace overlaps a buffer");
  if ((rc = run("mm_int8_ffn", up_q, stream))) return rc;
  if ((rc = quantize_rows("mm_int8_ffn", h, ld_h, MM_DTYPE_FP32, hq, ld_q, hs, f->tokens, f->inter, stream))) return rc;
  return run("mm_int8_ffn", down_q, stream);
}

int mm_int8_set_wait_budget(int64_t microseconds) {
  if (microseconds < 1 || microseconds > 60000000)
    return set_error(MM_ERR_INVALID, "mm_int8_set_wait_budget: %lld us outside 1..60000000", static_cast<long long>(microseconds));
  g_wait_ns.store(microseconds * 1000);
  return MM_OK;
}

int mm_int8_withhold(int32_t rank, int32_t launches) {
  if (rank < 0 || rank > 7 || launches < 0) return set_error(MM_ERR_INVALID, "mm_int8_withhold: rank %d, %d launches", rank, launches);
  g_withhold_rank.store(rank);
  g_withhold_launches.store(launches);
  return MM_OK;
}

int mm_int8_check(void) {
  cudaError_t e = cudaDeviceSynchronize();
  uint32_t word = 0;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&word, g_int8_error, sizeof(word));
  if (e == cudaSuccess && word) {
    const uint32_t zero = 0;
    e = cudaMemcpyToSymbol(g_int8_error, &zero, sizeof(zero));
  }
  if (e != cudaSuccess) return set_error(MM_ERR_CUDA, "mm_int8_check: %s", cudaGetErrorString(e));
  if (word) return set_error(MM_ERR_DEVICE_TIMEOUT, "device wait timed out (error word 0x%x)", word);
  return MM_OK;
}

}  // extern "C"
