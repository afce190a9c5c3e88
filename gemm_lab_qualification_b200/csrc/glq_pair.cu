// glq_pair.cu -- the large matrix product of the feed-forward operators, one
// tile per CTA pair, with the operator's epilogue fused in.
//
//   out[m, n] = epilogue(sum_k A[m, k] B[n, k])
//
// What it computes (see Product in glq_ffn.h): the linear layer with bias,
// activation and residual; the gated pair h = act(A Bg^T + bg) * (A Bu^T + bu)
// from one pass over A; and the backward products: dA = dz B, of the gated
// layer over the concatenated contraction of both projections, and dB = dz^T A
// for both projections in one launch.
//
// Bound: the tensor cores, from a few hundred tokens on.  Hence:
//   * Two CTAs (cta_group::2) compute a 256 x BN tile: each loads its own 128
//     rows of A and BN / 2 rows of B, so a stage of 64 K moves 64 KB for 256 x
//     256 x 64 products where two separate CTAs would move 96 KB.
//   * Gated pair: CTA 0's half of B is Bg's rows, CTA 1's is Bu's, so columns
//     [0, BN / 2) of every accumulator row are gate and [BN / 2, BN) are up,
//     in the same TMEM lane: the product needs no exchange.
//   * Persistent grid; warp 0 feeds a TMA ring, warp 1 of the leader issues
//     tcgen05.mma, warps 4-11 run the epilogue of one tile from tensor memory
//     while the next tile accumulates in the other half of it.  Two epilogue
//     warps per SM sub-partition: with one, nothing hid the latency of a chain
//     of tensor-memory load, conversion and store, and a 128 x 256 tile took
//     4.8 us, longer than the main loop of K = 1000.
//   * Few tiles (a wave that would leave SMs idle): the K range of a tile is
//     split over the pairs of one larger cluster (SPLIT).  Each CTA leaves its
//     FP32 partial tile in its drained ring; after a cluster barrier the pairs
//     share out the tile's column chunks, read the partials through
//     distributed shared memory and add them in split order.
//   * Operands are K-major or MN-major (the transposed operands of the
//     backward products), both read by TMA as they lie in memory: no
//     transposition pass.
//   * The epilogue works on units of 32 rows x 32 accumulator columns per warp
//     in FP32, rounds once to the 16-bit output, stages the unit in swizzled
//     shared memory and lets the TMA store it (clipped at the edges), or, where
//     the output's pitch or base is off 16 bytes, copies it out element by
//     element.
//
// Every wait is bounded; an expired one raises a bit in the device error word
// and the kernel returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "glq_act.cuh"
#include "glq_ffn.h"
#include "glq_internal.h"
#include "glq_ptx_pair.cuh"

namespace glq {
namespace {

constexpr int kBK = 64;         // K elements per stage: one 128-byte swizzle row
constexpr int kThreads = 384;
constexpr int kTileM = 256;     // rows per pair
constexpr int kEpiWarps = 8;    // warps 4..11, two per 32 TMEM lanes
constexpr int kSlots = 4;       // staging buffers per epilogue warp
constexpr uint32_t kSlotBytes = 32 * 64;  // a unit: 32 rows x 32 16-bit columns
constexpr uint32_t kMnBox = 64 * kBK * 2;  // MN-major box: 64 elements x 64 K rows
constexpr uint32_t kSmemMax = 232448;
constexpr int kMaxPairs = 4;  // K ranges of a split tile: clusters of up to 8 CTAs

template <int BN>
struct PairConfig {
  static_assert(BN == 128 || BN == 256, "pair tiles are 128 or 256 columns");
  static constexpr int kStages = BN == 256 ? 5 : 6;
  static constexpr uint32_t kABytes = 128 * kBK * 2;
  static constexpr uint32_t kBBytes = (BN / 2) * kBK * 2;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kRing = kStages * kStageBytes;
  static constexpr uint32_t kStaging = kEpiWarps * kSlots * kSlotBytes;
  static constexpr uint32_t kBias = kEpiWarps * 64 * 2;  // a unit's columns of both biases
  // full, empty, accumulator full (2) and empty (2); TMEM slot, abort flag.
  static constexpr int kBars = 2 * kStages + 4;
  static constexpr uint32_t kSmem = 1024 + kRing + kStaging + kBias + kBars * 8 + 16;
  static constexpr uint32_t kTmemCols = 2 * BN;  // two accumulators
  static_assert(128 * BN * 4 <= kRing, "a split tile's partials reuse the ring");
  static_assert(kSmem <= kSmemMax, "shared memory");
};

struct alignas(64) PairMaps {
  CUtensorMap a[2], b[2], out[2], pre[2];
};

struct PairArgs {
  int m, n;              // of one output
  int tiles_m, tiles_n;  // of one output
  int outputs;           // 2: Parts::kTwo
  int kb_part, kb_total; // K blocks of the first contraction range, of all
  int group_m;           // tile rows that share a column of tiles in launch order
  int split;             // K ranges per tile (SPLIT kernels), pairs per cluster
  int act;
  const void* bias[2];
  const void* residual;
  long long ld_residual;
  int residual_vec;      // residual rows are 16-byte aligned
  void* out[2];
  long long ld_out;
  int out_tma;
  void* pre[2];
  long long ld_pre;
  int pre_tma;
  unsigned int* err;
};

struct Tile {
  int part, m0, n0;
};

// Tile t: outputs one after the other; in each, groups of group_m tile rows,
// rows fastest, so the tiles in flight share B columns and A rows in L2.
template <int TILE_N>
__device__ __forceinline__ Tile tile_at(const PairArgs& args, int t) {
  const int per = args.tiles_m * args.tiles_n;
  Tile c;
  c.part = t / per;
  int r = t - c.part * per;
  const int group = r / (args.group_m * args.tiles_n);
  r -= group * args.group_m * args.tiles_n;
  const int first = group * args.group_m;
  const int rows = min(args.group_m, args.tiles_m - first);
  const int col = r / rows;
  c.m0 = (first + r - col * rows) * kTileM;
  c.n0 = col * TILE_N;
  return c;
}

template <typename T, bool A_MN, bool B_MN, int BN, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairArgs args) {
  using Cfg = PairConfig<BN>;
  using E = Elem16<T>;
  constexpr int kStages = Cfg::kStages;
  constexpr int kTileN = GATED ? BN / 2 : BN;  // output columns of a tile

  extern __shared__ uint8_t smem_dyn[];
  const uint32_t raw = ptx::smem_addr(smem_dyn);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  uint8_t* smem = smem_dyn + pad;
  const uint32_t sbase = raw + pad;
  uint8_t* staging = smem + Cfg::kRing;
  T* bias_smem = reinterpret_cast<T*>(staging + Cfg::kStaging);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(bias_smem) + Cfg::kBias);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  auto bar = [&](int i) { return ptx::smem_addr(&bars[i]); };
  auto full_bar = [&](int i) { return bar(i); };
  auto empty_bar = [&](int i) { return bar(kStages + i); };
  auto acc_full = [&](int i) { return bar(2 * kStages + i); };
  auto acc_empty = [&](int i) { return bar(2 * kStages + 2 + i); };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cluster_rank = ptx::cluster_ctarank();
  const uint32_t rank = cluster_rank & 1u;                // half of the pair
  const uint32_t leader = cluster_rank & ~1u;             // the pair's CTA that issues the MMAs
  const int range = static_cast<int>(cluster_rank >> 1);  // K range of this pair (SPLIT)
  const int num_tiles = args.outputs * args.tiles_m * args.tiles_n;
  const int split = SPLIT ? args.split : 1;
  const int first_tile = static_cast<int>(blockIdx.x >> 1) / split;
  // A SPLIT cluster computes one tile.
  const int tile_step = SPLIT ? num_tiles : static_cast<int>(gridDim.x >> 1);
  const int kb_begin = SPLIT ? static_cast<int>(static_cast<long long>(range) * args.kb_total / split) : 0;
  const int kb_end = SPLIT ? static_cast<int>(static_cast<long long>(range + 1) * args.kb_total / split) : args.kb_total;
  auto raise = [&](unsigned int bit) {
    atomicOr(args.err, bit);
    *abort_flag = 1;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full_bar(i), 1);   // leader: its producer's expect; both CTAs' bytes
      ptx::mbar_init(empty_bar(i), 1);  // the leader's commit
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(acc_full(i), 1);               // the leader's commit
      ptx::mbar_init(acc_empty(i), 2 * kEpiWarps);  // leader: both CTAs' epilogue warps
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
    for (int i = 0; i < 2; ++i) {
      ptx::prefetch_tensormap(&maps.a[i]);
      ptx::prefetch_tensormap(&maps.b[i]);
    }
  }
  if (warp == 2) {
    ptx::tmem_alloc_pair(ptx::smem_addr(tmem_slot), Cfg::kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync();  // both CTAs' barriers are initialised
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  if (warp == 0 && lane == 0) {
    // ---- TMA producer: this CTA's halves, counted on the leader's barriers.
    int it = 0;
    for (int t = first_tile; t < num_tiles && *abort_flag == 0; t += tile_step) {
      const Tile tile = tile_at<kTileN>(args, t);
      const int a_row = tile.m0 + static_cast<int>(rank) * 128;
      const int b_row = GATED ? tile.n0 : tile.n0 + static_cast<int>(rank) * (BN / 2);
      for (int kb = kb_begin; kb < kb_end; ++kb, ++it) {
        const int stage = it % kStages;
        const int round = it / kStages;
        if (round > 0 &&
            !ptx::mbar_wait_bounded(empty_bar(stage), (round - 1) & 1, abort_flag, kWaitBudgetNs)) {
          raise(kErrTimeoutProducer);
          break;
        }
        const int half = kb >= args.kb_part ? 1 : 0;
        const int k0 = (kb - half * args.kb_part) * kBK;
        const CUtensorMap* map_a = &maps.a[tile.part + half];
        const CUtensorMap* map_b = &maps.b[GATED ? static_cast<int>(rank) : tile.part + half];
        const uint32_t a_dst = sbase + stage * Cfg::kStageBytes;
        const uint32_t b_dst = a_dst + Cfg::kABytes;
        if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * Cfg::kStageBytes);
        const uint32_t signal = ptx::map_to_rank(full_bar(stage), leader);
        if constexpr (A_MN) {
          ptx::tma_load_2d_pair(a_dst, map_a, a_row, k0, signal);
          ptx::tma_load_2d_pair(a_dst + kMnBox, map_a, a_row + 64, k0, signal);
        } else {
          ptx::tma_load_2d_pair(a_dst, map_a, k0, a_row, signal);
        }
        if constexpr (B_MN) {
#pragma unroll
          for (int j = 0; j < BN / 128; ++j) {
            ptx::tma_load_2d_pair(b_dst + j * kMnBox, map_b, b_row + 64 * j, k0, signal);
          }
        } else {
          ptx::tma_load_2d_pair(b_dst, map_b, k0, b_row, signal);
        }
      }
    }
    if (*abort_flag != 0) {
      // Give the copies in flight time to land before shared memory goes.
      const uint64_t t0 = ptx::globaltimer_ns();
      for (uint32_t i = 0; i < (1u << 20) && ptx::globaltimer_ns() - t0 < 2000000ull; ++i) {
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- MMA issuer (leader CTA).
    constexpr uint32_t idesc = ptx::umma_idesc_f16_ab(kTileM, BN, E::kFormat, A_MN ? 1 : 0, B_MN ? 1 : 0);
    // Descriptor steps (16-byte units) per K = 16: 32 bytes along a swizzled
    // K-major row, or 16 K rows of 128 bytes.
    constexpr uint32_t kAStep = A_MN ? 128 : 2;
    constexpr uint32_t kBStep = B_MN ? 128 : 2;
    const uint16_t pair_mask = static_cast<uint16_t>(3u << leader);
    int it = 0, local = 0;
    for (int t = first_tile; t < num_tiles && *abort_flag == 0; t += tile_step, ++local) {
      const int acc = local & 1;
      if (local >= 2 &&
          !ptx::mbar_wait_bounded_cluster(acc_empty(acc), ((local >> 1) - 1) & 1, abort_flag, kWaitBudgetNs)) {
        raise(kErrTimeoutMma);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t d = tmem + acc * BN;
      bool ok = true;
      for (int kb = kb_begin; kb < kb_end; ++kb, ++it) {
        const int stage = it % kStages;
        if (!ptx::mbar_wait_bounded(full_bar(stage), (it / kStages) & 1, abort_flag, kWaitBudgetNs)) {
          raise(kErrTimeoutMma);
          ok = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t a_src = sbase + stage * Cfg::kStageBytes;
        const uint64_t da = A_MN ? ptx::umma_desc_mn_sw128(a_src) : ptx::umma_desc_k_sw128(a_src);
        const uint32_t b_src = a_src + Cfg::kABytes;
        const uint64_t db = B_MN ? ptx::umma_desc_mn_sw128(b_src) : ptx::umma_desc_k_sw128(b_src);
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
          ptx::tc_mma_f16_pair(d, da + kAStep * kk, db + kBStep * kk, idesc, kb > kb_begin || kk > 0 ? 1u : 0u);
        }
        ptx::tc_commit_pair(empty_bar(stage), pair_mask);
      }
      if (!ok) break;
      ptx::tc_commit_pair(acc_full(acc), pair_mask);
    }
  } else if (warp >= 4) {
    // ---- Epilogue: warp 4 + 4 h + w holds tile rows 32 w .. + 31, lane = row,
    // and every other unit of 32 columns.
    const int w = warp & 3;
    const int half = (warp >> 2) - 1;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(w * 32) << 16);
    uint8_t* slots = staging + (warp - 4) * kSlots * kSlotBytes;
    T* sbias = bias_smem + (warp - 4) * 64;
    const bool keep = args.pre[0] != nullptr;
    const bool biased = args.bias[0] != nullptr || args.bias[1] != nullptr;
    const T* res = static_cast<const T*>(args.residual);
    // Staging buffers a unit fills: the output and what is kept.
    const int per_unit = 1 + (keep ? (GATED ? 2 : 1) : 0);
    // This warp's units of a tile; a split tile's are shared by its pairs.
    const int first_col = SPLIT ? 32 * (2 * range + half) : 32 * half;
    const int col_step = SPLIT ? 64 * split : 64;
    int slot = 0, local = 0;
    bool joined = false;
    for (int t = first_tile; t < num_tiles; t += tile_step, ++local) {
      const int acc = local & 1;
      const Tile tile = tile_at<kTileN>(args, t);
      const int row0 = tile.m0 + static_cast<int>(rank) * 128 + w * 32;
      const int row = row0 + lane;
      // The residual of a unit is requested one unit ahead, the tile's first
      // before its accumulator is waited for.
      uint4 ahead[4] = {};
      [[maybe_unused]] auto request = [&](int c) {
        const int u0 = tile.n0 + c;
        if (!GATED && res != nullptr && args.residual_vec && c < kTileN && row < args.m && u0 + 32 <= args.n) {
          const uint4* rp = reinterpret_cast<const uint4*>(res + static_cast<long long>(row) * args.ld_residual + u0);
#pragma unroll
          for (int q = 0; q < 4; ++q) ahead[q] = rp[q];
        }
      };
      request(first_col);
      const bool ready =
          ptx::mbar_wait_bounded(acc_full(acc), (local >> 1) & 1, abort_flag, kWaitBudgetNs);
      if (!__all_sync(0xffffffffu, ready)) {  // the warp leaves together
        if (lane == 0) raise(kErrTimeoutEpilogue);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t src = lane_base + acc * BN;
      if constexpr (SPLIT) {
        // FP32 partials into the drained ring: [group of 4 columns][tile row].
        float4* part = reinterpret_cast<float4*>(smem) + w * 32 + lane;
#pragma unroll 1
        for (int c = 32 * half; c < BN; c += 64) {
          uint32_t r[32];
          ptx::tmem_ld_32x32b_x32(src + c, r);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            part[(c / 4 + q) * 128] = make_float4(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]),
                                                  __uint_as_float(r[4 * q + 2]), __uint_as_float(r[4 * q + 3]));
          }
        }
        joined = true;
        ptx::cluster_arrive_release();
        ptx::cluster_wait();
      }
      // 32 accumulator columns from `at`: from tensor memory, or the sums of
      // the cluster's partials in split order.
      auto load32 = [&](int at, uint32_t(&r)[32]) {
        if constexpr (SPLIT) {
          const uint32_t local_at = sbase + static_cast<uint32_t>((at / 4 * 128 + w * 32 + lane) * 16);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float4 x[kMaxPairs];
#pragma unroll
            for (int p = 0; p < kMaxPairs; ++p) {
              if (p < split) x[p] = ptx::ld_dsmem_v4(ptx::map_to_rank(local_at + q * 128 * 16, 2 * p + rank));
            }
#pragma unroll
            for (int p = 1; p < kMaxPairs; ++p) {
              if (p < split) {
                x[0].x += x[p].x;
                x[0].y += x[p].y;
                x[0].z += x[p].z;
                x[0].w += x[p].w;
              }
            }
            r[4 * q] = __float_as_uint(x[0].x);
            r[4 * q + 1] = __float_as_uint(x[0].y);
            r[4 * q + 2] = __float_as_uint(x[0].z);
            r[4 * q + 3] = __float_as_uint(x[0].w);
          }
        } else {
          ptx::tmem_ld_32x32b_x32(src + at, r);
        }
      };
#pragma unroll 1
      for (int c = first_col; c < kTileN; c += col_step) {
        const int u0 = tile.n0 + c;  // first output column of the unit
        uint32_t r[32];
        load32(c, r);
        [[maybe_unused]] uint32_t r2[32];
        if constexpr (GATED) load32(BN / 2 + c, r2);
        // The buffers about to be filled must have been read by their stores.
        if (lane == 0) {
          if (per_unit == 1) {
            ptx::bulk_wait_read<kSlots - 1>();
          } else if (per_unit == 2) {
            ptx::bulk_wait_read<kSlots - 2>();
          } else {
            ptx::bulk_wait_read<kSlots - 3>();
          }
        }
        __syncwarp();
        if (biased) {
          const bool in = u0 + lane < args.n;
          const T* b0 = static_cast<const T*>(args.bias[0]);
          sbias[lane] = b0 != nullptr && in ? b0[u0 + lane] : E::from_f(0.0f);
          if constexpr (GATED) {
            const T* b1 = static_cast<const T*>(args.bias[1]);
            sbias[32 + lane] = b1 != nullptr && in ? b1[u0 + lane] : E::from_f(0.0f);
          }
          __syncwarp();
        }
        uint8_t* buf[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) buf[i] = slots + ((slot + i) % kSlots) * kSlotBytes;
        if constexpr (!SPLIT) {
          ptx::tmem_ld_wait();
          if (c + 64 >= kTileN) {
            // This warp's share of the accumulator is in registers.
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_rank(acc_empty(acc), leader));
          }
        }
        auto with_bias = [&](const uint32_t(&from)[32], const T* bias, float(&to)[32]) {
#pragma unroll
          for (int j = 0; j < 32; ++j) to[j] = __uint_as_float(from[j]);
          if (biased) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              const uint4 x = *reinterpret_cast<const uint4*>(bias + j);
              const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = E::to_f2(xs[e]);
                to[j + 2 * e] += f.x;
                to[j + 2 * e + 1] += f.y;
              }
            }
          }
        };
        // The unit's row of this lane into a staging buffer: 64-byte swizzle.
        auto put = [&](uint8_t* to, const float(&x)[32]) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 p;
            p.x = E::from_f2(x[8 * q], x[8 * q + 1]);
            p.y = E::from_f2(x[8 * q + 2], x[8 * q + 3]);
            p.z = E::from_f2(x[8 * q + 4], x[8 * q + 5]);
            p.w = E::from_f2(x[8 * q + 6], x[8 * q + 7]);
            *reinterpret_cast<uint4*>(to + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = p;
          }
        };
        float v[32];
        with_bias(r, sbias, v);
        if (keep) put(buf[1], v);
        if constexpr (GATED) {
          float v2[32];
          with_bias(r2, sbias + 32, v2);
          if (keep) put(buf[2], v2);
          with_act(args.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_f<decltype(act)::value>(v[j]) * v2[j];
          });
        } else {
          with_act(args.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_f<decltype(act)::value>(v[j]);
          });
          if (res != nullptr && row < args.m) {
            if (args.residual_vec && u0 + 32 <= args.n) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint32_t xs[4] = {ahead[q].x, ahead[q].y, ahead[q].z, ahead[q].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = E::to_f2(xs[e]);
                  v[8 * q + 2 * e] += f.x;
                  v[8 * q + 2 * e + 1] += f.y;
                }
              }
            } else {
              const T* rp = res + static_cast<long long>(row) * args.ld_residual + u0;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (u0 + j < args.n) v[j] += E::to_f(rp[j]);
              }
            }
          }
          request(c + col_step);
        }
        put(buf[0], v);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        // Output first, then what is kept, each its own bulk group.
        auto leave = [&](int i, const CUtensorMap* map, void* base, long long ld, bool tma) {
          if (tma) {
            if (lane == 0) {
              if (row0 < args.m && u0 < args.n) ptx::tma_store_2d(map, ptx::smem_addr(buf[i]), u0, row0);
              ptx::bulk_commit();
            }
          } else {
            T* y = static_cast<T*>(base) + u0 + lane;
            if (u0 + lane < args.n) {
              for (int rr = 0; rr < 32 && row0 + rr < args.m; ++rr) {
                y[static_cast<long long>(row0 + rr) * ld] = *reinterpret_cast<const T*>(
                    buf[i] + rr * 64 + (((lane >> 3) ^ ((rr >> 1) & 3)) << 4) + (lane & 7) * 2);
              }
            }
            __syncwarp();
            if (lane == 0) ptx::bulk_commit();  // keeps the group count uniform
          }
        };
        leave(0, &maps.out[tile.part], args.out[tile.part], args.ld_out, args.out_tma != 0);
        if (keep) {
          leave(1, &maps.pre[0], args.pre[0], args.ld_pre, args.pre_tma != 0);
          if constexpr (GATED) leave(2, &maps.pre[1], args.pre[1], args.ld_pre, args.pre_tma != 0);
        }
        slot = (slot + per_unit) % kSlots;
      }
    }
    // The staging buffers have been read; the grid's end completes the writes.
    if (lane == 0) ptx::bulk_wait_read<0>();
    // An aborted epilogue still takes its part in the join's barrier.
    if (SPLIT && !joined) {
      ptx::cluster_arrive_release();
      ptx::cluster_wait();
    }
  }
  __syncwarp();
  if (SPLIT && warp < 4) {
    ptx::cluster_arrive_release();
    ptx::cluster_wait();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync();  // the peer's MMA operands and barriers are no longer needed
  if (warp == 2) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem, Cfg::kTmemCols);
  }
}

bool aligned_rows(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * 2) % 16 == 0;
}

// The map of an operand with `rows` output rows and contraction `k`: boxes of
// box_rows rows x 64 K, or 64 rows x 64 K when MN-major.
bool operand_map(CUtensorMap* map, int dtype, const Operand& o, int64_t rows, int64_t k, uint32_t box_rows) {
  return o.k_major ? encode_tile_map(map, dtype, o.base, rows, k, o.pitch, box_rows)
                   : encode_tile_map(map, dtype, o.base, k, rows, o.pitch, kBK);
}

// How a product is cut up: columns per tile and K ranges per tile.
struct Cut {
  int bn;
  int split;
};

template <typename T, bool A_MN, bool B_MN, int BN, bool GATED, bool SPLIT>
cudaError_t launch_typed(const Product& p, int split, int sm_count, unsigned int* err, cudaStream_t s) {
  using Cfg = PairConfig<BN>;
  constexpr int kTileN = GATED ? BN / 2 : BN;
  const bool concat = p.parts == Parts::kConcatK, two = p.parts == Parts::kTwo;
  PairMaps maps;
  PairArgs args = {};
  bool ok = true;
  for (int i = 0; i < 2; ++i) {
    const Operand& a = concat || two ? p.a[i] : p.a[0];
    const Operand& b = concat || two || GATED ? p.b[i] : p.b[0];
    ok = ok && operand_map(&maps.a[i], p.dtype, a, p.m, p.k, 128);
    ok = ok && operand_map(&maps.b[i], p.dtype, b, p.n, p.k, BN / 2);
  }
  args.out_tma = aligned_rows(p.out[0], p.ld_out) && (!two || aligned_rows(p.out[1], p.ld_out)) ? 1 : 0;
  args.pre_tma = p.pre[0] != nullptr && aligned_rows(p.pre[0], p.ld_pre) &&
                         (!GATED || aligned_rows(p.pre[1], p.ld_pre))
                     ? 1
                     : 0;
  for (int i = 0; i < 2; ++i) {
    args.out[i] = p.out[two ? i : 0];
    args.pre[i] = p.pre[i];
    args.bias[i] = p.bias[i];
    // A map that no store uses repeats an operand's.
    maps.out[i] = maps.a[0];
    maps.pre[i] = maps.a[0];
    if (args.out_tma) ok = ok && encode_tile_map(&maps.out[i], p.dtype, args.out[i], p.m, p.n, p.ld_out, 32, 32);
    if (args.pre_tma && args.pre[i] != nullptr) {
      ok = ok && encode_tile_map(&maps.pre[i], p.dtype, args.pre[i], p.m, p.n, p.ld_pre, 32, 32);
    }
  }
  if (!ok) return cudaErrorInvalidValue;
  args.m = static_cast<int>(p.m);
  args.n = static_cast<int>(p.n);
  args.tiles_m = static_cast<int>((p.m + kTileM - 1) / kTileM);
  args.tiles_n = static_cast<int>((p.n + kTileN - 1) / kTileN);
  args.outputs = two ? 2 : 1;
  args.kb_part = static_cast<int>((p.k + kBK - 1) / kBK);
  args.kb_total = args.kb_part * (concat ? 2 : 1);
  args.group_m = 16;
  args.split = split;
  args.act = p.act;
  args.residual = p.residual;
  args.ld_residual = p.ld_residual;
  args.residual_vec = aligned_rows(p.residual, p.ld_residual) ? 1 : 0;
  args.ld_out = p.ld_out;
  args.ld_pre = p.ld_pre;
  args.err = err;
  const int64_t tiles = static_cast<int64_t>(args.outputs) * args.tiles_m * args.tiles_n;
  const int64_t pairs = SPLIT ? tiles * split : std::min<int64_t>(tiles, std::max(sm_count / 2, 1));

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLIT ? 2 * split : 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (p.flags & GLQ_FLAG_NO_PDL) ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, pair_kernel<T, A_MN, B_MN, BN, GATED, SPLIT>, maps, args);
}

template <typename T, int BN, bool SPLIT>
cudaError_t launch_order(const Product& p, int split, int sm_count, unsigned int* err, cudaStream_t s) {
  // The operand orders that occur: both K-major or B MN-major (forward and
  // input gradient), both MN-major (weight gradient).
  const bool a_mn = !p.a[0].k_major, b_mn = !p.b[0].k_major;
  if (p.parts == Parts::kGated) {
    if (a_mn) return cudaErrorInvalidValue;
    return b_mn ? launch_typed<T, false, true, BN, true, SPLIT>(p, split, sm_count, err, s)
                : launch_typed<T, false, false, BN, true, SPLIT>(p, split, sm_count, err, s);
  }
  if (a_mn) {
    return b_mn ? launch_typed<T, true, true, BN, false, SPLIT>(p, split, sm_count, err, s) : cudaErrorInvalidValue;
  }
  return b_mn ? launch_typed<T, false, true, BN, false, SPLIT>(p, split, sm_count, err, s)
              : launch_typed<T, false, false, BN, false, SPLIT>(p, split, sm_count, err, s);
}

template <typename T>
cudaError_t launch_cut(const Product& p, Cut cut, int sm_count, unsigned int* err, cudaStream_t s) {
  if (cut.split > 1) {
    return cut.bn == 256 ? launch_order<T, 256, true>(p, cut.split, sm_count, err, s)
                         : launch_order<T, 128, true>(p, cut.split, sm_count, err, s);
  }
  return cut.bn == 256 ? launch_order<T, 256, false>(p, 1, sm_count, err, s)
                       : launch_order<T, 128, false>(p, 1, sm_count, err, s);
}

template <typename T, bool A_MN, bool B_MN, int BN, bool GATED>
cudaError_t set_attr() {
  constexpr cudaFuncAttribute kAttr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  const int bytes = static_cast<int>(PairConfig<BN>::kSmem);
  const cudaError_t e = cudaFuncSetAttribute(pair_kernel<T, A_MN, B_MN, BN, GATED, false>, kAttr, bytes);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(pair_kernel<T, A_MN, B_MN, BN, GATED, true>, kAttr, bytes);
}

template <typename T, int BN>
cudaError_t set_attrs() {
  cudaError_t e = set_attr<T, false, false, BN, true>();
  if (e == cudaSuccess) e = set_attr<T, false, true, BN, true>();
  if (e == cudaSuccess) e = set_attr<T, false, false, BN, false>();
  if (e == cudaSuccess) e = set_attr<T, false, true, BN, false>();
  if (e == cudaSuccess) e = set_attr<T, true, true, BN, false>();
  return e;
}

// Clusters of 2 * split CTAs that run at once on each device (one CTA per SM;
// a cluster stays inside a GPC), asked once per device.
constexpr int kMaxDevices = 64;
int g_resident[kMaxDevices][kMaxPairs + 1];

cudaError_t ask_resident(int device, int sm_count) {
  g_resident[device][1] = sm_count / 2;
  for (int split = 2; split <= kMaxPairs; ++split) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = PairConfig<256>::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(2 * split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(
        &g_resident[device][split], pair_kernel<__half, false, false, 256, false, true>, &cfg);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// The cut with the least estimated time.  A K block of 64 takes a pair 0.27 us
// whatever the tile's width (its loads through L2 bound it: 128 columns move
// 24 KB per CTA, 256 move 32 KB, in 0.29 and 0.27 us), so a narrow tile only
// saves epilogue (1.2 us against 2.4; 1.8 when waves follow one another), and a
// split costs 1.5 us for the join, 3 us when a unit has two accumulators, and
// 1.2 us more for clusters of more than two pairs.  Measured with 131 tokens:
// 4096 x 4096, 25.9 us whole, 17.5 us in 2 ranges, 16.1 us in 3; gated 2736 x
// 1000, 12.2 us, 10.4 us with narrow tiles, 11.2 us in 2 ranges.
Cut choose_cut(const Product& p) {
  const bool gated = p.parts == Parts::kGated;
  const int64_t kb = (p.k + kBK - 1) / kBK * (p.parts == Parts::kConcatK ? 2 : 1);
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return {256, 1};
  Cut best = {256, 1};
  double best_us = 0.0;
  for (int bn = 256; bn >= 128; bn /= 2) {
    const int tile_n = gated ? bn / 2 : bn;
    const int64_t tiles =
        (p.m + kTileM - 1) / kTileM * ((p.n + tile_n - 1) / tile_n) * (p.parts == Parts::kTwo ? 2 : 1);
    const double epilogue_us = bn == 256 ? 2.4 : 1.2;
    for (int split = 1; split <= kMaxPairs && split <= kb; ++split) {
      const int64_t at_once = std::max(g_resident[device][split], 0);
      if (at_once == 0 || (split > 1 && tiles > at_once)) continue;
      const double loop_us = 0.27 * static_cast<double>((kb + split - 1) / split);
      const double waves = static_cast<double>((tiles + at_once - 1) / at_once);
      const double join_us = (gated ? 3.0 : 1.5) + (split > 2 ? 1.2 : 0.0);
      const double us = split > 1 ? loop_us + epilogue_us / split + join_us
                                  : waves * std::max(loop_us, bn == 256 ? 2.4 : 1.8) + epilogue_us;
      if (best_us == 0.0 || us < best_us) {
        best_us = us;
        best = {bn, split};
      }
    }
  }
  return best;
}

}  // namespace

cudaError_t pair_prepare_device() {
  cudaError_t e = set_attrs<__half, 256>();
  if (e == cudaSuccess) e = set_attrs<__half, 128>();
  if (e == cudaSuccess) e = set_attrs<__nv_bfloat16, 256>();
  if (e == cudaSuccess) e = set_attrs<__nv_bfloat16, 128>();
  int device = 0, sm_count = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess && device >= kMaxDevices) e = cudaErrorInvalidDevice;
  return e != cudaSuccess ? e : ask_resident(device, sm_count);
}

cudaError_t launch_pair(const Product& p, int sm_count, unsigned int* err, cudaStream_t s) {
  if (p.m < 1 || p.n < 1 || p.k < 1) return cudaErrorInvalidValue;
  Cut cut = choose_cut(p);
  return p.dtype == GLQ_DTYPE_BF16 ? launch_cut<__nv_bfloat16>(p, cut, sm_count, err, s)
                                   : launch_cut<__half>(p, cut, sm_count, err, s);
}

}  // namespace glq
