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
//   * Few tiles: the K range of a tile is split over the pairs of one larger
//     cluster (SPLIT).  Each CTA leaves its FP32 partial tile in its drained
//     ring; after a cluster barrier the pairs share out the tile's units, read
//     the partials through distributed shared memory and add them in order.
//   * The partial wave that is left after whole waves of tiles, and two
//     products in one launch: the K blocks are dealt to the pairs in equal
//     runs.  A pair whose run starts inside a tile leaves its FP32 partial in
//     the workspace and publishes a flag per warp; the pair that has the tile's
//     first block adds the partials in run order and runs the epilogue.
//     Neither join depends on timing.
//   * Two products may share a launch (the input's and the weights' gradients):
//     together they fill waves that each alone would leave ragged.
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

#include <algorithm>
#include <atomic>
#include <chrono>

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
constexpr int kSlots = 4;       // staging buffers per epilogue warp: a tile's units, or a unit's outputs
constexpr int kMaxPairs = 4;    // K ranges of a split tile: clusters of up to 8 CTAs
constexpr uint32_t kSlotBytes = 32 * 64;  // a unit: 32 rows x 32 16-bit columns
constexpr uint32_t kMnBox = 64 * kBK * 2;  // MN-major box: 64 elements x 64 K rows
constexpr uint32_t kSmemMax = 232448;

constexpr int kTileN = 256;     // accumulator columns per pair
constexpr int kStages = 5;  // (6 with half the staging: no faster)
constexpr uint32_t kOperandBytes = 128 * kBK * 2;  // a CTA's half of either operand
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr uint32_t kRing = kStages * kStageBytes;
constexpr uint32_t kStaging = kEpiWarps * kSlots * kSlotBytes;
constexpr uint32_t kBias = kEpiWarps * 64 * 2;  // a unit's columns of both biases
// full, empty, accumulator full (2) and empty (2); TMEM slot, abort flag.
constexpr int kBars = 2 * kStages + 4;
constexpr uint32_t kSmem = 1024 + kRing + kStaging + kBias + kBars * 8 + 16;
static_assert(kSmem <= kSmemMax, "shared memory");
static_assert(128 * kTileN * 4 <= kRing, "a split tile's partials reuse the ring");
constexpr uint32_t kTmemCols = 2 * kTileN;  // two accumulators

// A pair's FP32 partial tile in the workspace, [CTA][group of 4 columns][row],
// and the flags of its 16 epilogue warps.
constexpr int64_t kSlotTile = 2 * 128 * kTileN * 4;
constexpr int64_t kSlotFlags = 2 * kEpiWarps * 8;

struct alignas(64) PairMaps {
  CUtensorMap a[2][2], b[2][2], out[2][2];  // [product][its second operand or output]
  CUtensorMap pre[2];
};

struct PairProduct {
  int m, n;              // of one output
  int tiles_m, tiles_n;  // of one output
  int tiles;             // of all outputs
  int kb_part, kb_total; // K blocks of the first contraction range, of all
  int a_mn, b_mn;        // operand orders
  int out_tma;
  void* out[2];
  long long ld_out;
};

struct PairArgs {
  PairProduct p[2];
  // K ranges per tile (SPLIT kernels), pairs per cluster.
  int split;
  // Schedule: tiles [0, whole) of p[0] go round the pairs whole; the blocks of
  // the others, p[0]'s then p[1]'s, are dealt to `runs` pairs in equal runs.
  int whole;
  int runs;
  long long run_blocks;  // blocks dealt in all
  float* partials;       // [runs] slots of kSlotTile bytes
  unsigned long long* flags;  // [runs][2][kEpiWarps]
  unsigned long long epoch;   // what a flag of this launch holds
  int group_m;           // tile rows that share a column of tiles in launch order
  int act;
  const void* bias[2];
  const void* residual;
  long long ld_residual;
  int residual_vec;      // residual rows are 16-byte aligned
  void* pre[2];
  long long ld_pre;
  int pre_tma;
  unsigned int* err;
};

// A piece of work of a pair: K blocks [kb_begin, kb_end) of one tile.
struct Piece {
  int product, part, m0, n0, kb_begin, kb_end;
  bool partial;  // starts inside the tile: its sums go to the workspace
  int helpers;   // further runs that hold the rest of the tile
};

// The pieces of pair `index` in order; every role of the kernel walks them
// alike.  Runs are dealt from the last pair down, so a pair that waits for a
// partial waits for one of a lower block index, which was started before it.
struct Walk {
  const PairArgs& args;
  int pairs, next_whole, run;
  long long lo, hi;
  int out_n;  // output columns per tile

  __device__ Walk(const PairArgs& a, int index, int pairs_, int out_n_)
      : args(a), pairs(pairs_), next_whole(index), run(a.runs - 1 - index), lo(0), hi(0), out_n(out_n_) {
    if (run >= 0) {
      lo = begin(run);
      hi = begin(run + 1);
    }
  }
  __device__ long long begin(int r) const { return static_cast<long long>(r) * args.run_blocks / args.runs; }

  // Tile t of product q: outputs one after the other; in each, groups of
  // group_m tile rows, rows fastest, so the tiles in flight share B columns
  // and A rows in L2.
  __device__ void place(Piece& c, int q, int t) const {
    const PairProduct& p = args.p[q];
    c.product = q;
    const int per = p.tiles_m * p.tiles_n;
    c.part = t / per;
    int r = t - c.part * per;
    const int group = r / (args.group_m * p.tiles_n);
    r -= group * args.group_m * p.tiles_n;
    const int first = group * args.group_m;
    const int rows = min(args.group_m, p.tiles_m - first);
    const int col = r / rows;
    c.m0 = (first + r - col * rows) * kTileM;
    c.n0 = col * out_n;
  }

  __device__ bool next(Piece& c) {
    if (next_whole < args.whole) {
      place(c, 0, next_whole);
      next_whole += pairs;
      c.kb_begin = 0;
      c.kb_end = args.p[0].kb_total;
      c.partial = false;
      c.helpers = 0;
      return true;
    }
    if (lo >= hi) return false;
    const long long blocks0 = static_cast<long long>(args.p[0].tiles - args.whole) * args.p[0].kb_total;
    const int q = lo < blocks0 ? 0 : 1;
    const long long base = q == 0 ? 0 : blocks0;
    const int kb = args.p[q].kb_total;
    const long long t = (lo - base) / kb;
    place(c, q, static_cast<int>(t) + (q == 0 ? args.whole : 0));
    const long long start = base + t * kb;
    c.kb_begin = static_cast<int>(lo - start);
    const long long end = min(start + kb, hi);
    c.kb_end = static_cast<int>(end - start);
    c.partial = c.kb_begin > 0;
    c.helpers = 0;
    if (!c.partial) {
      for (int r = run + 1; r < args.runs && begin(r) < start + kb; ++r) ++c.helpers;
    }
    lo = end;
    return true;
  }
};

// Calls f with the operand orders as constants: the loops that feed the tensor
// core are short of issue slots for anything else (with the orders looked up
// per block a K block took 0.34 us instead of 0.27).
template <typename F>
__device__ __forceinline__ void with_orders(const PairProduct& p, F&& f) {
  if (p.a_mn) {
    f(std::true_type(), std::true_type());
  } else if (p.b_mn) {
    f(std::false_type(), std::true_type());
  } else {
    f(std::false_type(), std::false_type());
  }
}

__device__ __forceinline__ float4 ld_global_cg(const float4* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void st_release_gpu(unsigned long long* p, unsigned long long v) {
  asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned long long ld_acquire_gpu(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

template <typename T, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairArgs args) {
  using E = Elem16<T>;
  constexpr int kOutN = GATED ? kTileN / 2 : kTileN;  // output columns of a tile

  extern __shared__ uint8_t smem_dyn[];
  const uint32_t raw = ptx::smem_addr(smem_dyn);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  uint8_t* smem = smem_dyn + pad;
  const uint32_t sbase = raw + pad;
  uint8_t* staging = smem + kRing;
  T* bias_smem = reinterpret_cast<T*>(staging + kStaging);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(bias_smem) + kBias);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
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
  const uint32_t leader = cluster_rank & ~1u;             // the CTA that issues the pair's MMAs
  const int range = static_cast<int>(cluster_rank >> 1);  // K range of this pair (SPLIT)
  const int split = SPLIT ? args.split : 1;
  auto raise = [&](unsigned int bit) {
    atomicOr(args.err, bit);
    *abort_flag = 1;
  };
  // Verdicts of a warp, so that its lanes stay together when a wait expires.
  auto all_ok = [&](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  auto going = [&]() { return all_ok(*abort_flag == 0); };

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
    ptx::prefetch_tensormap(&maps.a[0][0]);
    ptx::prefetch_tensormap(&maps.b[0][0]);
  }
  if (warp == 2) {
    ptx::tmem_alloc_pair(ptx::smem_addr(tmem_slot), kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync();  // both CTAs' barriers are initialised
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  Walk walk(args, static_cast<int>(blockIdx.x >> 1), static_cast<int>(gridDim.x >> 1), kOutN);
  Piece piece;
  bool first_piece = true;
  auto next_piece = [&]() {
    if constexpr (SPLIT) {  // this pair's K range of the cluster's tile
      if (!first_piece) return false;
      first_piece = false;
      walk.place(piece, 0, static_cast<int>(blockIdx.x >> 1) / split);
      const long long kb = args.p[0].kb_total;
      piece.kb_begin = static_cast<int>(range * kb / split);
      piece.kb_end = static_cast<int>((range + 1) * kb / split);
      piece.partial = false;
      piece.helpers = 0;
      return true;
    } else {
      return walk.next(piece);
    }
  };
  if (warp == 0) {
    // ---- TMA producer: this CTA's halves, counted on the leader's barriers.
    // (The whole warp walks and waits, one lane issues: a loop of one lane in a
    // diverged warp is slower.)
    int stage = 0, rounds = 0;
    const uint32_t signals = ptx::map_to_rank(full_bar(0), leader);
    while (going() && next_piece()) {
      // (in registers: the asm's memory clobbers would reload them per block)
      const PairProduct& p = args.p[piece.product];
      const int kb_part = p.kb_part;
      const int a_row = piece.m0 + static_cast<int>(rank) * 128;
      const int b_row = GATED ? piece.n0 : piece.n0 + static_cast<int>(rank) * 128;
      const CUtensorMap* maps_a = &maps.a[piece.product][piece.part];
      const CUtensorMap* maps_b = &maps.b[piece.product][GATED ? static_cast<int>(rank) : piece.part];
      const int kb_end = piece.kb_end;
      with_orders(p, [&](auto a_mn, auto b_mn) {
        for (int kb = piece.kb_begin; kb < kb_end; ++kb) {
          if (!all_ok(rounds == 0 ||
                      ptx::mbar_wait_bounded(empty_bar(stage), (rounds - 1) & 1, abort_flag, kWaitBudgetNs))) {
            raise(kErrTimeoutProducer);
            break;
          }
          const int half = kb >= kb_part ? 1 : 0;
          const int k0 = (kb - half * kb_part) * kBK;
          const CUtensorMap* map_a = maps_a + half;
          const CUtensorMap* map_b = GATED ? maps_b : maps_b + half;
          const uint32_t a_dst = sbase + stage * kStageBytes;
          const uint32_t b_dst = a_dst + kOperandBytes;
          if (ptx::elect_one()) {
            if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * kStageBytes);
            const uint32_t signal = signals + 8u * static_cast<uint32_t>(stage);
            if constexpr (decltype(a_mn)::value) {
              ptx::tma_load_2d_pair(a_dst, map_a, a_row, k0, signal);
              ptx::tma_load_2d_pair(a_dst + kMnBox, map_a, a_row + 64, k0, signal);
            } else {
              ptx::tma_load_2d_pair(a_dst, map_a, k0, a_row, signal);
            }
            if constexpr (decltype(b_mn)::value) {
              ptx::tma_load_2d_pair(b_dst, map_b, b_row, k0, signal);
              ptx::tma_load_2d_pair(b_dst + kMnBox, map_b, b_row + 64, k0, signal);
            } else {
              ptx::tma_load_2d_pair(b_dst, map_b, k0, b_row, signal);
            }
          }
          if (++stage == kStages) {
            stage = 0;
            ++rounds;
          }
        }
      });
    }
    if (lane == 0 && *abort_flag != 0) {
      // Give the copies in flight time to land before shared memory goes.
      const uint64_t t0 = ptx::globaltimer_ns();
      for (uint32_t i = 0; i < (1u << 20) && ptx::globaltimer_ns() - t0 < 2000000ull; ++i) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---- MMA issuer (leader CTA).
    int stage = 0, rounds = 0, local = 0;
    const uint16_t pair_mask = static_cast<uint16_t>(3u << leader);
    for (; going() && next_piece(); ++local) {
      const int acc = local & 1;
      if (!all_ok(local < 2 || ptx::mbar_wait_bounded_cluster(acc_empty(acc), ((local >> 1) - 1) & 1, abort_flag,
                                                              kWaitBudgetNs))) {
        raise(kErrTimeoutMma);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t d = tmem + acc * kTileN;
      bool ok = true;
      const int blocks = piece.kb_end - piece.kb_begin;
      with_orders(args.p[piece.product], [&](auto a_mn, auto b_mn) {
        constexpr bool kAMn = decltype(a_mn)::value, kBMn = decltype(b_mn)::value;
        constexpr uint32_t idesc = ptx::umma_idesc_f16_ab(kTileM, kTileN, E::kFormat, kAMn, kBMn);
        // Descriptor steps (16-byte units) per K = 16: 32 bytes along a
        // swizzled K-major row, or 16 K rows of 128 bytes.
        constexpr uint32_t kAStep = kAMn ? 128 : 2, kBStep = kBMn ? 128 : 2;
        for (int i = 0; i < blocks; ++i) {
          if (!all_ok(ptx::mbar_wait_bounded(full_bar(stage), rounds & 1, abort_flag, kWaitBudgetNs))) {
            raise(kErrTimeoutMma);
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t a_src = sbase + stage * kStageBytes, b_src = a_src + kOperandBytes;
          const uint64_t da = kAMn ? ptx::umma_desc_mn_sw128(a_src) : ptx::umma_desc_k_sw128(a_src);
          const uint64_t db = kBMn ? ptx::umma_desc_mn_sw128(b_src) : ptx::umma_desc_k_sw128(b_src);
          if (ptx::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk) {
              ptx::tc_mma_f16_pair(d, da + kAStep * kk, db + kBStep * kk, idesc, i > 0 || kk > 0 ? 1u : 0u);
            }
            ptx::tc_commit_pair(empty_bar(stage), pair_mask);
          }
          if (++stage == kStages) {
            stage = 0;
            ++rounds;
          }
        }
      });
      if (!ok) break;
      if (ptx::elect_one()) ptx::tc_commit_pair(acc_full(acc), pair_mask);
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
    // This warp's units of a tile; a split tile's are shared by its pairs.
    const int first_col = SPLIT ? 32 * (2 * range + half) : 32 * half;
    const int col_step = SPLIT ? 64 * split : 64;
    bool joined = false;
    // Run r's partial of this lane's row, and this warp's flag.
    auto partial_of = [&](int r) {
      return reinterpret_cast<float4*>(args.partials) + (static_cast<long long>(r) * 2 + rank) * (128 * kTileN / 4) +
             w * 32 + lane;
    };
    auto flag_of = [&](int r) { return args.flags + (static_cast<long long>(r) * 2 + rank) * kEpiWarps + (warp - 4); };
    for (int local = 0; next_piece(); ++local) {
      const PairProduct& p = args.p[piece.product];
      const int acc = local & 1;
      const int row0 = piece.m0 + static_cast<int>(rank) * 128 + w * 32;
      const int row = row0 + lane;
      // The residual of a unit is requested one unit ahead, the tile's first
      // before its accumulator is waited for.
      uint4 ahead[4] = {};
      [[maybe_unused]] auto request = [&](int c) {
        const int u0 = piece.n0 + c;
        if (!GATED && res != nullptr && args.residual_vec && c < kOutN && row < p.m && u0 + 32 <= p.n) {
          const uint4* rp = reinterpret_cast<const uint4*>(res + static_cast<long long>(row) * args.ld_residual + u0);
#pragma unroll
          for (int q = 0; q < 4; ++q) ahead[q] = rp[q];
        }
      };
      if (!piece.partial) request(first_col);
      if (!all_ok(ptx::mbar_wait_bounded(acc_full(acc), (local >> 1) & 1, abort_flag, kWaitBudgetNs))) {
        if (lane == 0) raise(kErrTimeoutEpilogue);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t src = lane_base + acc * kTileN;
      // This warp's share of the accumulator is in registers or written: the
      // leader may reuse it.
      auto release = [&]() {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_rank(acc_empty(acc), leader));
      };
      if (piece.partial) {
        float4* to = partial_of(walk.run);
#pragma unroll 1
        for (int c = first_col; c < kTileN; c += 64) {
          uint32_t r[32];
          ptx::tmem_ld_32x32b_x32(src + c, r);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            to[(c / 4 + q) * 128] = make_float4(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]),
                                                __uint_as_float(r[4 * q + 2]), __uint_as_float(r[4 * q + 3]));
          }
        }
        release();
        // (the release covers the other lanes' stores, ordered before by the
        // warp barrier)
        __syncwarp();
        if (lane == 0) st_release_gpu(flag_of(walk.run), args.epoch);
        continue;
      }
      if (piece.helpers > 0) {
        bool ready = true;
        if (lane < piece.helpers) {
          const unsigned long long* flag = flag_of(walk.run + 1 + lane);
          const uint64_t t0 = ptx::globaltimer_ns();
          for (uint32_t polls = 1; ld_acquire_gpu(flag) != args.epoch; ++polls) {
            if ((polls & 63u) == 0u &&
                (*abort_flag != 0 || ptx::globaltimer_ns() - t0 > kWaitBudgetNs || polls > (1u << 26))) {
              ready = false;
              break;
            }
          }
        }
        if (!all_ok(ready)) {
          if (lane == 0) raise(kErrTimeoutEpilogue);
          break;
        }
        __syncwarp();  // what the polling lanes acquired, the others may read
      }
      if constexpr (SPLIT) {
        // FP32 partials into the drained ring: [group of 4 columns][tile row].
        float4* part = reinterpret_cast<float4*>(smem) + w * 32 + lane;
#pragma unroll 1
        for (int c = 32 * half; c < kTileN; c += 64) {
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
      // 32 accumulator columns from `at`: from tensor memory (waited for
      // later), or the sums of the cluster's partials in range order.
      auto load32 = [&](int at, uint32_t(&r)[32]) {
        if constexpr (SPLIT) {
          const uint32_t local_at = sbase + static_cast<uint32_t>((at / 4 * 128 + w * 32 + lane) * 16);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float4 x[kMaxPairs];
#pragma unroll
            for (int k = 0; k < kMaxPairs; ++k) {
              if (k < split) x[k] = ptx::ld_dsmem_v4(ptx::map_to_rank(local_at + q * 128 * 16, 2 * k + rank));
            }
#pragma unroll
            for (int k = 1; k < kMaxPairs; ++k) {
              if (k < split) {
                x[0].x += x[k].x;
                x[0].y += x[k].y;
                x[0].z += x[k].z;
                x[0].w += x[k].w;
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
      // Other runs' partials, requested for the first of them before tensor
      // memory is waited for, added in run order.
      float4 other[8];
      auto request_partial = [&](int h, int at) {
        const float4* from = partial_of(walk.run + h) + at / 4 * 128;
#pragma unroll
        for (int q = 0; q < 8; ++q) other[q] = ld_global_cg(from + q * 128);
      };
      auto add_partials = [&](int at, uint32_t(&r)[32]) {  // other: the first helper's
        for (int h = 1;; ++h) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            r[4 * q] = __float_as_uint(__uint_as_float(r[4 * q]) + other[q].x);
            r[4 * q + 1] = __float_as_uint(__uint_as_float(r[4 * q + 1]) + other[q].y);
            r[4 * q + 2] = __float_as_uint(__uint_as_float(r[4 * q + 2]) + other[q].z);
            r[4 * q + 3] = __float_as_uint(__uint_as_float(r[4 * q + 3]) + other[q].w);
          }
          if (h == piece.helpers) break;
          request_partial(h + 1, at);
        }
      };
      const bool helped = !SPLIT && piece.helpers > 0;
      if (helped) request_partial(1, first_col);
      // Stores the unit in staging buffer `at` to its place.
      auto leave = [&](int at, int u0, const CUtensorMap* map, void* base, long long ld, bool tma) {
        const uint8_t* buf = slots + at * kSlotBytes;
        if (tma) {
          if (lane == 0 && row0 < p.m && u0 < p.n) ptx::tma_store_2d(map, ptx::smem_addr(buf), u0, row0);
        } else if (u0 + lane < p.n) {
          T* y = static_cast<T*>(base) + u0 + lane;
          for (int rr = 0; rr < 32 && row0 + rr < p.m; ++rr) {
            y[static_cast<long long>(row0 + rr) * ld] = *reinterpret_cast<const T*>(
                buf + rr * 64 + (((lane >> 3) ^ ((rr >> 1) & 3)) << 4) + (lane & 7) * 2);
          }
        }
      };
      const CUtensorMap* out_map = &maps.out[piece.product][piece.part];
      void* const out_base = p.out[piece.part];
      const long long ld_out = p.ld_out;
      const bool out_tma = p.out_tma != 0;
      // The staging buffers have been read by the stores before.
      auto reclaim = [&]() {
        if (lane == 0) ptx::bulk_wait_read<0>();
        __syncwarp();
      };
      reclaim();
      int filled = 0;
#pragma unroll 1
      for (int c = first_col; c < kOutN; c += col_step) {
        const int u0 = piece.n0 + c;  // first output column of the unit
        uint32_t r[32];
        load32(c, r);
        [[maybe_unused]] uint32_t r2[32];
        if constexpr (GATED) load32(kTileN / 2 + c, r2);
        if (biased) {
          __syncwarp();
          const bool in = u0 + lane < p.n;
          const T* b0 = static_cast<const T*>(args.bias[0]);
          sbias[lane] = b0 != nullptr && in ? b0[u0 + lane] : E::from_f(0.0f);
          if constexpr (GATED) {
            const T* b1 = static_cast<const T*>(args.bias[1]);
            sbias[32 + lane] = b1 != nullptr && in ? b1[u0 + lane] : E::from_f(0.0f);
          }
          __syncwarp();
        }
        if constexpr (!SPLIT) {
          ptx::tmem_ld_wait();
          if (c + 64 >= kOutN) release();
          if (helped) {
            add_partials(c, r);
            if constexpr (GATED) {
              request_partial(1, kTileN / 2 + c);
              add_partials(kTileN / 2 + c, r2);
            }
            if (c + 64 < kOutN) request_partial(1, c + 64);
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
        // The unit into a staging buffer, lane = row: 64-byte swizzle.
        auto put = [&](int at, const float(&x)[32]) {
          uint8_t* buf = slots + at * kSlotBytes;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 packed;
            packed.x = E::from_f2(x[8 * q], x[8 * q + 1]);
            packed.y = E::from_f2(x[8 * q + 2], x[8 * q + 3]);
            packed.z = E::from_f2(x[8 * q + 4], x[8 * q + 5]);
            packed.w = E::from_f2(x[8 * q + 6], x[8 * q + 7]);
            *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = packed;
          }
        };
        float v[32];
        with_bias(r, sbias, v);
        if (keep) put(1, v);
        if constexpr (GATED) {
          float v2[32];
          with_bias(r2, sbias + 32, v2);
          if (keep) put(2, v2);
          with_act(args.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_f<decltype(act)::value>(v[j]) * v2[j];
          });
        } else {
          with_act(args.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_f<decltype(act)::value>(v[j]);
          });
          if (res != nullptr && row < p.m) {
            if (args.residual_vec && u0 + 32 <= p.n) {
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
                if (u0 + j < p.n) v[j] += E::to_f(rp[j]);
              }
            }
          }
          request(c + col_step);
        }
        put(filled, v);
        if (keep) {
          // A unit's outputs leave together: one fence for the three.
          ptx::fence_proxy_async_smem();
          __syncwarp();
          leave(0, u0, out_map, out_base, ld_out, out_tma);
          leave(1, u0, &maps.pre[0], args.pre[0], args.ld_pre, args.pre_tma != 0);
          if constexpr (GATED) leave(2, u0, &maps.pre[1], args.pre[1], args.ld_pre, args.pre_tma != 0);
          if (lane == 0) ptx::bulk_commit();
          __syncwarp();
          reclaim();
        } else {
          ++filled;
        }
      }
      if (!keep) {
        // The tile's units leave together (a fence per unit made the epilogue
        // of a 128 x 256 half tile take 4.2 us).
        ptx::fence_proxy_async_smem();
        __syncwarp();
        for (int i = 0; i < filled; ++i) {
          leave(i, piece.n0 + first_col + i * col_step, out_map, out_base, ld_out, out_tma);
        }
        if (lane == 0) ptx::bulk_commit();
        __syncwarp();
      }
      // The flags are left as they were found, for a replay of this launch.
      __syncwarp();
      if (lane < piece.helpers) *flag_of(walk.run + 1 + lane) = 0ull;
    }
    // The staging buffers have been read; the grid's end completes the writes.
    if (lane == 0) ptx::bulk_wait_read<0>();
    if (SPLIT && !joined) {  // an aborted epilogue still takes its part in the join
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
    ptx::tmem_dealloc_pair(tmem, kTmemCols);
  }
}

// A value that no flag holds yet: launches number on from a start of their
// process's own, so what fresh workspace memory happens to hold is not it.
unsigned long long next_epoch() {
  static std::atomic<unsigned long long> epoch{
      static_cast<unsigned long long>(std::chrono::steady_clock::now().time_since_epoch().count()) *
      0x9E3779B97F4A7C15ull};
  const unsigned long long e = epoch.fetch_add(1);
  return e != 0 ? e : epoch.fetch_add(1);
}

bool aligned_rows(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * 2) % 16 == 0;
}

template <typename T, bool GATED, bool SPLIT>
cudaError_t launch_typed(const Product* products, int count, const PairPlan& plan, void* workspace, unsigned int* err,
                         cudaStream_t s) {
  constexpr int kOutN = GATED ? kTileN / 2 : kTileN;
  PairMaps maps;
  PairArgs args = {};
  bool ok = true;
  for (int q = 0; q < count; ++q) {
    const Product& p = products[q];
    const bool concat = p.parts == Parts::kConcatK, two = p.parts == Parts::kTwo;
    PairProduct& r = args.p[q];
    r.out_tma = aligned_rows(p.out[0], p.ld_out) && (!two || aligned_rows(p.out[1], p.ld_out)) ? 1 : 0;
    for (int i = 0; i < 2; ++i) {
      const Operand& a = concat || two ? p.a[i] : p.a[0];
      const Operand& b = concat || two || GATED ? p.b[i] : p.b[0];
      ok = ok && operand_map(&maps.a[q][i], p.dtype, a, p.m, p.k, 128);
      ok = ok && operand_map(&maps.b[q][i], p.dtype, b, p.n, p.k, 128);
      r.out[i] = p.out[two ? i : 0];
      maps.out[q][i] = maps.a[q][0];  // (a map that no store uses)
      if (r.out_tma) ok = ok && encode_tile_map(&maps.out[q][i], p.dtype, r.out[i], p.m, p.n, p.ld_out, 32, 32);
    }
    r.m = static_cast<int>(p.m);
    r.n = static_cast<int>(p.n);
    r.tiles_m = static_cast<int>((p.m + kTileM - 1) / kTileM);
    r.tiles_n = static_cast<int>((p.n + kOutN - 1) / kOutN);
    r.tiles = r.tiles_m * r.tiles_n * (two ? 2 : 1);
    r.kb_part = static_cast<int>((p.k + kBK - 1) / kBK);
    r.kb_total = r.kb_part * (concat ? 2 : 1);
    if (!p.a[0].k_major && p.b[0].k_major) return cudaErrorInvalidValue;  // does not occur
    r.a_mn = p.a[0].k_major ? 0 : 1;
    r.b_mn = p.b[0].k_major ? 0 : 1;
    r.ld_out = p.ld_out;
  }
  if (count == 1) {
    args.p[1] = args.p[0];
    for (int i = 0; i < 2; ++i) {
      maps.a[1][i] = maps.a[0][i];
      maps.b[1][i] = maps.b[0][i];
      maps.out[1][i] = maps.out[0][i];
    }
  }
  const Product& p = products[0];
  args.pre_tma = p.pre[0] != nullptr && aligned_rows(p.pre[0], p.ld_pre) &&
                         (!GATED || aligned_rows(p.pre[1], p.ld_pre))
                     ? 1
                     : 0;
  for (int i = 0; i < 2; ++i) {
    args.pre[i] = p.pre[i];
    args.bias[i] = p.bias[i];
    maps.pre[i] = maps.a[0][0];
    if (args.pre_tma && args.pre[i] != nullptr) {
      ok = ok && encode_tile_map(&maps.pre[i], p.dtype, args.pre[i], p.m, p.n, p.ld_pre, 32, 32);
    }
  }
  if (!ok) return cudaErrorInvalidValue;
  args.split = plan.split;
  args.whole = static_cast<int>(plan.whole);
  args.runs = plan.runs;
  args.run_blocks = plan.run_blocks;
  args.partials = static_cast<float*>(workspace);
  args.flags = reinterpret_cast<unsigned long long*>(static_cast<unsigned char*>(workspace) + plan.runs * kSlotTile);
  args.epoch = next_epoch();
  args.group_m = 8;
  args.act = p.act;
  args.residual = p.residual;
  args.ld_residual = p.ld_residual;
  args.residual_vec = aligned_rows(p.residual, p.ld_residual) ? 1 : 0;
  args.ld_pre = p.ld_pre;
  args.err = err;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * plan.pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(2 * plan.split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (p.flags & GLQ_FLAG_NO_PDL) ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, pair_kernel<T, GATED, SPLIT>, maps, args);
}

template <typename T>
cudaError_t launch_any(const Product* products, int count, const PairPlan& plan, void* workspace, unsigned int* err,
                       cudaStream_t s) {
  const bool gated = products[0].parts == Parts::kGated;
  if (plan.split > 1) {
    return gated ? launch_typed<T, true, true>(products, count, plan, workspace, err, s)
                 : launch_typed<T, false, true>(products, count, plan, workspace, err, s);
  }
  return gated ? launch_typed<T, true, false>(products, count, plan, workspace, err, s)
               : launch_typed<T, false, false>(products, count, plan, workspace, err, s);
}

template <typename T>
cudaError_t set_attrs() {
  constexpr cudaFuncAttribute kAttr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  const int bytes = static_cast<int>(kSmem);
  cudaError_t e = cudaFuncSetAttribute(pair_kernel<T, true, true>, kAttr, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(pair_kernel<T, true, false>, kAttr, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(pair_kernel<T, false, true>, kAttr, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(pair_kernel<T, false, false>, kAttr, bytes);
  return e;
}

struct Size {
  int64_t tiles, kb;
};

Size size_of(const Product& p) {
  const int out_n = p.parts == Parts::kGated ? kTileN / 2 : kTileN;
  return {(p.m + kTileM - 1) / kTileM * ((p.n + out_n - 1) / out_n) * (p.parts == Parts::kTwo ? 2 : 1),
          (p.k + kBK - 1) / kBK * (p.parts == Parts::kConcatK ? 2 : 1)};
}

// Clusters of 2 * split CTAs that run at once (one CTA per SM; a cluster stays
// inside a GPC): 33, 22 and 15 of 148 SMs.  An estimate for plans only.
int64_t resident_clusters(int split, int sm_count) {
  return split == 1 ? sm_count / 2 : sm_count * (split == 2 ? 33 : split == 3 ? 22 : 15) / 148;
}

// Estimated times in us, after the launch: a K block of a tile takes 0.25, a
// tile's epilogue 3.4; joining a split tile 1.5 (3 with two accumulators per
// unit), 1.2 more for clusters of over two pairs; dealt runs 4.5 for the
// hand-over and 4 for every further partial that a tile's owner adds.
constexpr double kBlockUs = 0.25, kEpilogueUs = 3.4, kLaunchUs = 4.0;

}  // namespace

PairPlan plan_pair(const Product* products, int count, int sm_count) {
  PairPlan plan;
  const int64_t most = std::max(sm_count / 2, 1);
  const Size s0 = size_of(products[0]);
  const Size s1 = count > 1 ? size_of(products[1]) : Size{0, 1};
  plan.pairs = static_cast<int>(std::min(most, s0.tiles + s1.tiles));
  plan.whole = s0.tiles;
  const int64_t rest = count > 1 ? s0.tiles : s0.tiles % most;
  const double wave_us = std::max(kBlockUs * static_cast<double>(s0.kb), kEpilogueUs);
  const double whole_us = static_cast<double>((s0.tiles - rest) / most) * wave_us;
  plan.us = whole_us + (rest > 0 ? wave_us : 0.0) + kEpilogueUs;
  if (rest == 0) return plan;
  // The last wave as it is; then each other way to compute its tiles.
  if (count == 1 && s0.tiles < most) {
    const double two = products[0].parts == Parts::kGated ? 2.0 : 1.0;
    for (int split = 2; split <= kMaxPairs && split <= s0.kb; ++split) {
      if (s0.tiles > resident_clusters(split, sm_count)) break;
      const double us = kBlockUs * static_cast<double>((s0.kb + split - 1) / split) + kEpilogueUs / split +
                        1.5 * two + (split > 2 ? 1.2 : 0.0);
      if (us < plan.us) {
        plan.us = us;
        plan.split = split;
      }
    }
    plan.pairs = static_cast<int>(s0.tiles * plan.split);
    return plan;
  }
  const int64_t blocks = rest * s0.kb + s1.tiles * s1.kb;
  const int64_t longest = std::max(s0.kb, s1.kb);
  int64_t best = 0;
  if (count > 1) plan.us = 1e30;
  for (int64_t runs = count > 1 ? 1 : rest + 1; runs <= std::min(most, blocks); ++runs) {
    const int64_t run = (blocks + runs - 1) / runs, helpers = (longest + run - 1) / run;
    if (helpers > 16) break;  // (a warp's lanes poll one helper's flag each)
    // A run through short tiles is paced by their epilogues.
    double loop_us = 0.0;
    for (const Size& z : {s0, s1}) {
      const double tiles = static_cast<double>(run) / static_cast<double>(z.kb);
      loop_us = std::max(loop_us, tiles * std::max(kBlockUs * static_cast<double>(z.kb), tiles > 1.0 ? kEpilogueUs : 0.0));
      if (count == 1) break;
    }
    const double us =
        whole_us + loop_us + kEpilogueUs + 4.5 + 4.0 * static_cast<double>(helpers - 1);
    if (us < plan.us) {
      plan.us = us;
      best = runs;
    }
  }
  if (best == 0) return plan;
  plan.whole = s0.tiles - rest;
  plan.runs = static_cast<int>(best);
  plan.run_blocks = blocks;
  plan.pairs = static_cast<int>(plan.whole > 0 ? most : best);
  plan.workspace_bytes = static_cast<size_t>(plan.runs * (kSlotTile + kSlotFlags));
  return plan;
}

// Two products in one launch when that is faster than one after the other
// (999 tokens through 4100 x 1032: 23 and 25 us alone, 37 together); many
// waves of tiles keep their order, which shares operands in L2.
bool share_launch(const Product* products, int sm_count) {
  if (size_of(products[0]).tiles + size_of(products[1]).tiles > 3 * std::max(sm_count / 2, 1)) return false;
  return plan_pair(products, 2, sm_count).us <
         plan_pair(products, 1, sm_count).us + plan_pair(products + 1, 1, sm_count).us + kLaunchUs;
}

cudaError_t pair_prepare_device() {
  const cudaError_t e = set_attrs<__half>();
  return e != cudaSuccess ? e : set_attrs<__nv_bfloat16>();
}

cudaError_t launch_pair(const Product* products, int count, void* workspace, int sm_count, unsigned int* err,
                        cudaStream_t s) {
  for (int i = 0; i < count; ++i) {
    if (products[i].m < 1 || products[i].n < 1 || products[i].k < 1) return cudaErrorInvalidValue;
  }
  const PairPlan plan = plan_pair(products, count, sm_count);
  return products[0].dtype == GLQ_DTYPE_BF16
             ? launch_any<__nv_bfloat16>(products, count, plan, workspace, err, s)
             : launch_any<__half>(products, count, plan, workspace, err, s);
}

}  // namespace glq
