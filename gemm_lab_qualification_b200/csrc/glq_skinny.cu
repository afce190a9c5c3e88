// glq_skinny.cu -- the feed-forward operators' matrix product for few tokens
// (decode batches, single tokens).
//
//   out[m, n] = epilogue(sum_k A[m, k] W[n, k]),  W = B^T
//
// Bound: the bytes of W, each read once.  So the weight rows fill the 128
// lanes of the MMA's M dimension, the tokens are its N dimension (16..192),
// and the work is spread so that every SM streams weights:
//   * One CTA owns 128 weight rows x one token tile x one contiguous range of
//     64-wide K blocks; two CTAs share an SM (about 100 KB of loads in flight
//     each).  The K ranges of a tile are the CTAs of one thread-block cluster.
//   * Gated pair: the 128 rows are 64 rows of Bg and the same 64 of Bu, so one
//     MMA computes both projections and the activations' product is formed
//     inside the CTA.
//   * Join: each CTA leaves its FP32 partial tile in its drained load ring as
//     [group of 4 tokens][row]; the CTAs of the cluster each own a share of
//     the groups and add the S partials in split order, so the result does not
//     depend on timing.  Up to 64 tokens the partials are pushed, one bulk
//     copy per owner, completing on the owner's barrier (1 x 4096 x 4096: 9.3
//     us when owners read them through distributed shared memory between two
//     cluster barriers); the receive buffer of 128 tokens would cost the second
//     CTA per SM, so those are read.  192 tokens take one CTA per SM.
//   * The epilogue (bias, activation, product, residual) runs on those sums
//     in FP32 with one rounding per output.
// The same kernel computes the input gradient for few tokens (W MN-major, and
// the two projections as one concatenated contraction).
#include <cuda.h>

#include <algorithm>

#include "glq_act.cuh"
#include "glq_ffn.h"
#include "glq_internal.h"
#include "glq_ptx_pair.cuh"

namespace glq {
namespace {

constexpr int kBK = 64;
constexpr int kThreads = 256;
constexpr int kRows = 128;  // weight rows per CTA
constexpr uint32_t kMnBox = 64 * kBK * 2;
constexpr uint32_t kTwoPerSm = 233472u / 2u - 1024u;
constexpr uint32_t kOnePerSm = 232448u;

template <int BT>
struct SkinnyConfig {
  static constexpr uint32_t kWBytes = kRows * kBK * 2;
  static constexpr uint32_t kABytes = BT * kBK * 2;
  static constexpr uint32_t kStageBytes = kWBytes + kABytes;
  // Two CTAs per SM up to 128 tokens, one beyond.
  static constexpr int kPerSm = BT <= 128 ? 2 : 1;
  static constexpr int kStages = BT == 16 || BT == 192 ? 5 : BT == 32 ? 4 : 3;
  static constexpr uint32_t kRing = kStages * kStageBytes;
  static constexpr bool kPush = BT <= 64;
  // Largest receive buffer: split - 1 partials of ceil(BT / 4 / split) groups.
  static constexpr uint32_t kReceive = !kPush ? 0 : BT <= 32 ? 7 * kRows * 16 : 7 * 2 * kRows * 16;
  static constexpr int kBars = 2 * kStages + 2;
  static constexpr uint32_t kSmem = 1024 + kRing + kReceive + kBars * 8 + 16;
  static constexpr uint32_t kTmemCols = BT < 32 ? 32 : BT == 192 ? 256 : BT;
  static_assert(kSmem <= (kPerSm == 2 ? kTwoPerSm : kOnePerSm), "shared memory");
  static_assert(kRows * BT * 4 <= kRing, "the partial tile reuses the ring");
};

struct alignas(64) SkinnyMaps {
  CUtensorMap w[2], a[2];
};

struct SkinnyArgs {
  int m, n;
  int kb_part, kb_total;
  int split;
  int act;
  const void* bias[2];
  const void* residual;
  long long ld_residual;
  void* out;
  long long ld_out;
  void* pre[2];
  long long ld_pre;
  unsigned int* err;
  unsigned int flags;
};

template <typename T, int BT, bool W_MN, bool GATED>
__global__ void __launch_bounds__(kThreads, SkinnyConfig<BT>::kPerSm)
    skinny_kernel(const __grid_constant__ SkinnyMaps maps, const __grid_constant__ SkinnyArgs args) {
  using Cfg = SkinnyConfig<BT>;
  using E = Elem16<T>;
  constexpr int kStages = Cfg::kStages;
  constexpr int kOutRows = GATED ? kRows / 2 : kRows;  // output columns per CTA

  extern __shared__ uint8_t smem_dyn[];
  const uint32_t raw = ptx::smem_addr(smem_dyn);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  uint8_t* smem = smem_dyn + pad;
  const uint32_t sbase = raw + pad;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kRing + Cfg::kReceive);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int i) { return ptx::smem_addr(&bars[i]); };
  auto empty_bar = [&](int i) { return ptx::smem_addr(&bars[kStages + i]); };
  const uint32_t done_bar = ptx::smem_addr(&bars[2 * kStages]);
  const uint32_t receive_bar = ptx::smem_addr(&bars[2 * kStages + 1]);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = args.split;
  const int s = blockIdx.x;  // K range == rank in the (split, 1, 1) cluster
  const int m0 = blockIdx.y * BT;
  const int n0 = blockIdx.z * kOutRows;
  const int kb_begin = static_cast<int>(static_cast<long long>(s) * args.kb_total / split);
  const int kb_end = static_cast<int>(static_cast<long long>(s + 1) * args.kb_total / split);
  const int nkb = kb_end - kb_begin;
  // The groups of 4 tokens that rank q of the cluster joins: [share(q),
  // share(q + 1)).
  const int tokens = min(BT, args.m - m0);
  const int groups = (tokens + 3) >> 2;
  auto share = [&](int q) { return q * groups / split; };
  const int own_lo = share(s);
  const int own = share(s + 1) - own_lo;
  auto raise = [&](unsigned int bit) {
    atomicOr(args.err, bit);
    *abort_flag = 1;
  };

  uint64_t pol_w = 0, pol_a = 0;
  auto issue_w = [&](int i) {
    const int stage = i % kStages;
    const int kb = kb_begin + i;
    const int half = kb >= args.kb_part ? 1 : 0;
    const int k0 = (kb - half * args.kb_part) * kBK;
    const uint32_t dst = sbase + stage * Cfg::kStageBytes;
    ptx::mbar_arrive_expect_tx(full_bar(stage), Cfg::kStageBytes);
    if constexpr (W_MN) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ptx::tma_load_2d(dst + j * kMnBox, &maps.w[GATED ? j : half], GATED ? n0 : n0 + 64 * j, k0, full_bar(stage),
                         pol_w);
      }
    } else if constexpr (GATED) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ptx::tma_load_2d(dst + j * (Cfg::kWBytes / 2), &maps.w[j], k0, n0, full_bar(stage), pol_w);
      }
    } else {
      ptx::tma_load_2d(dst, &maps.w[half], k0, n0, full_bar(stage), pol_w);
    }
  };
  auto issue_a = [&](int i) {
    const int stage = i % kStages;
    const int kb = kb_begin + i;
    const int half = kb >= args.kb_part ? 1 : 0;
    ptx::tma_load_2d(sbase + stage * Cfg::kStageBytes + Cfg::kWBytes, &maps.a[half], (kb - half * args.kb_part) * kBK,
                     m0, full_bar(stage), pol_a);
  };
  int issued = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full_bar(i), 1);
      ptx::mbar_init(empty_bar(i), 1);
    }
    ptx::mbar_init(done_bar, 1);
    ptx::mbar_init(receive_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    if (Cfg::kPush && split > 1) {
      ptx::mbar_arrive_expect_tx(receive_bar, static_cast<uint32_t>((split - 1) * own * kRows * 16));
    }
    if (nkb > 0) {
      ptx::prefetch_tensormap(&maps.w[0]);
      ptx::prefetch_tensormap(&maps.a[0]);
    }
    pol_w = ptx::policy_evict_first();
    pol_a = ptx::policy_evict_last();
    // The first stages need no wait: start the stream before anything else.
    // The weights wait for the preceding kernel unless declared static.
    const int first = min(nkb, kStages);
    const bool static_w = (args.flags & GLQ_FLAG_STATIC_WEIGHTS) != 0;
    if (static_w) {
      for (int i = 0; i < first; ++i) issue_w(i);
    }
    ptx::grid_dependency_wait();
    for (; issued < first; ++issued) {
      if (!static_w) issue_w(issued);
      issue_a(issued);
    }
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_addr(tmem_slot), Cfg::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // Waited for after the main loop: every receive barrier is initialised.
  if (Cfg::kPush && split > 1) ptx::cluster_arrive_relaxed();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  // (The feeding loops: a whole warp waits, one lane issues; loops of a single
  // lane in a diverged warp cost the pair kernel 3 to 6 %.)
  auto all_ok = [&](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  if (warp == 0) {
    issued = __shfl_sync(0xffffffffu, issued, 0);
    for (int i = issued; i < nkb; ++i) {
      if (!all_ok(ptx::mbar_wait_bounded(empty_bar(i % kStages), (i / kStages - 1) & 1, abort_flag, kWaitBudgetNs))) {
        raise(kErrTimeoutProducer);
        break;
      }
      if (lane == 0) {  // (the lane that has the cache policies)
        issue_w(i);
        issue_a(i);
      }
      issued = i + 1;
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = ptx::umma_idesc_f16_ab(kRows, BT, E::kFormat, W_MN ? 1 : 0, 0);
    constexpr uint32_t kWStep = W_MN ? 128 : 2;
    for (int i = 0; i < nkb; ++i) {
      const int stage = i % kStages;
      if (!all_ok(ptx::mbar_wait_bounded(full_bar(stage), (i / kStages) & 1, abort_flag, kWaitBudgetNs))) {
        raise(kErrTimeoutMma);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t w_src = sbase + stage * Cfg::kStageBytes;
      const uint64_t dw = W_MN ? ptx::umma_desc_mn_sw128(w_src) : ptx::umma_desc_k_sw128(w_src);
      const uint64_t da = ptx::umma_desc_k_sw128(w_src + Cfg::kWBytes);
      if (ptx::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
          ptx::tc_mma_f16(tmem, dw + kWStep * kk, da + 2u * kk, idesc, i > 0 || kk > 0 ? 1u : 0u);
        }
        ptx::tc_commit(empty_bar(stage));
      }
    }
    if (ptx::elect_one()) ptx::tc_commit(done_bar);
  }
  __syncwarp();
  if (!ptx::mbar_wait_bounded(done_bar, 0, abort_flag, kWaitBudgetNs)) raise(kErrTimeoutEpilogue);
  __syncthreads();
  const bool aborted = *abort_flag != 0;
  ptx::tc_fence_after_sync();

  // ---- Partial tile to shared memory: [group of 4 tokens][row], 16 bytes each.
  {
    const int row = (warp & 3) * 32 + lane;
    const uint32_t src = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float4* part = reinterpret_cast<float4*>(smem);
    for (int q = warp >> 2; q * 16 < tokens; q += 2) {
      uint32_t r[16];
      if (nkb > 0 && !aborted) {
        ptx::tmem_ld_32x32b_x16(src + q * 16, r);
        ptx::tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (4 * q + h < groups) {
          part[(4 * q + h) * kRows + row] =
              make_float4(__uint_as_float(r[4 * h]), __uint_as_float(r[4 * h + 1]), __uint_as_float(r[4 * h + 2]),
                          __uint_as_float(r[4 * h + 3]));
        }
      }
    }
  }
  bool joined = true;
  if (split > 1) {
    if constexpr (Cfg::kPush) {
      ptx::cluster_wait();
      ptx::fence_proxy_async_smem();
      __syncthreads();
      // Lane d ships the groups of rank s + d, so every owner is fed by a
      // different source at any moment; sources take receive slots in rank
      // order.
      if (warp == 0 && lane >= 1 && lane < split && !aborted) {
        const int owner = (s + lane) % split;
        const uint32_t bytes = static_cast<uint32_t>((share(owner + 1) - share(owner)) * kRows * 16);
        if (bytes > 0) {
          const uint32_t slot = static_cast<uint32_t>(s < owner ? s : s - 1);
          ptx::bulk_copy_to_peer(ptx::map_to_rank(sbase + Cfg::kRing + slot * bytes, owner),
                                 sbase + static_cast<uint32_t>(share(owner) * kRows * 16), bytes,
                                 ptx::map_to_rank(receive_bar, owner));
        }
      }
      joined = ptx::mbar_wait_bounded(receive_bar, 0, aborted ? abort_flag : nullptr, kWaitBudgetNs);
      if (!joined && !aborted) raise(kErrTimeoutEpilogue);
      // Arriving only after its own copies have landed, every CTA knows at
      // the last wait that none is in flight.
      ptx::cluster_arrive_relaxed();
    } else {
      __syncthreads();
      ptx::cluster_sync();
    }
  } else {
    __syncthreads();
  }

  // ---- Join and epilogue: this CTA's share of the groups.
  auto total = [&](int j, int row) {
    const int group = own_lo + j;
    const float4* mine = reinterpret_cast<const float4*>(smem) + group * kRows + row;
    if (split == 1) return *mine;
    const uint32_t at = sbase + static_cast<uint32_t>((group * kRows + row) * 16);
    const float4* received = reinterpret_cast<const float4*>(smem + Cfg::kRing) + j * kRows + row;
    float4 part[GLQ_MAX_SPLIT];
#pragma unroll
    for (int src = 0; src < GLQ_MAX_SPLIT; ++src) {
      if (src < split) {
        if constexpr (Cfg::kPush) {
          part[src] = src == s ? *mine : received[(src < s ? src : src - 1) * own * kRows];
        } else {
          part[src] = ptx::ld_dsmem_v4(ptx::map_to_rank(at, src));
        }
      }
    }
    float4 acc = part[0];
#pragma unroll
    for (int src = 1; src < GLQ_MAX_SPLIT; ++src) {
      if (src < split) {
        acc.x += part[src].x;
        acc.y += part[src].y;
        acc.z += part[src].z;
        acc.w += part[src].w;
      }
    }
    return acc;
  };
  T* out = static_cast<T*>(args.out);
  const T* res = static_cast<const T*>(args.residual);
  const bool keep = args.pre[0] != nullptr;
  if (!aborted && joined) {
    const int row = threadIdx.x % kOutRows;
    const int n = n0 + row;
    const bool n_ok = n < args.n;
    float b0 = 0.0f, b1 = 0.0f;
    if (n_ok && args.bias[0] != nullptr) b0 = E::to_f(static_cast<const T*>(args.bias[0])[n]);
    if (GATED && n_ok && args.bias[1] != nullptr) b1 = E::to_f(static_cast<const T*>(args.bias[1])[n]);
    for (int j = threadIdx.x / kOutRows; j < own; j += kThreads / kOutRows) {
      const float4 t0 = total(j, row);
      float v[4] = {t0.x + b0, t0.y + b0, t0.z + b0, t0.w + b0};
      [[maybe_unused]] float v2[4];
      if constexpr (GATED) {
        const float4 t1 = total(j, kOutRows + row);
        v2[0] = t1.x + b1;
        v2[1] = t1.y + b1;
        v2[2] = t1.z + b1;
        v2[3] = t1.w + b1;
      }
      const int m = m0 + 4 * (own_lo + j);
      if (keep && n_ok) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (m + e < args.m) {
            const long long at = static_cast<long long>(m + e) * args.ld_pre + n;
            static_cast<T*>(args.pre[0])[at] = E::from_f(v[e]);
            if constexpr (GATED) static_cast<T*>(args.pre[1])[at] = E::from_f(v2[e]);
          }
        }
      }
      with_act(args.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = act_f<decltype(act)::value>(v[e]);
      });
      if (n_ok) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (m + e < args.m) {
            float y = v[e];
            if constexpr (GATED) {
              y *= v2[e];
            } else {
              if (res != nullptr) y += E::to_f(res[static_cast<long long>(m + e) * args.ld_residual + n]);
            }
            out[static_cast<long long>(m + e) * args.ld_out + n] = E::from_f(y);
          }
        }
      }
    }
  }
  // After an abort, let this CTA's own loads land before shared memory goes.
  if (aborted && threadIdx.x == 0) {
    for (int i = max(0, issued - kStages); i < issued; ++i) {
      if (!ptx::mbar_wait_bounded(full_bar(i % kStages), (i / kStages) & 1, nullptr, kWaitBudgetNs)) {
        atomicOr(args.err, kErrTimeoutDrain);
        break;
      }
    }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (split > 1) {  // the peers have this CTA's partials
    if constexpr (Cfg::kPush) {
      ptx::cluster_wait();
    } else {
      ptx::cluster_sync();
    }
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, Cfg::kTmemCols);
  }
}

template <typename T, int BT, bool W_MN, bool GATED>
cudaError_t launch_typed(const Product& p, int sm_count, unsigned int* err, cudaStream_t s) {
  using Cfg = SkinnyConfig<BT>;
  constexpr int kOutRows = GATED ? kRows / 2 : kRows;
  const bool concat = p.parts == Parts::kConcatK;
  SkinnyMaps maps = {};
  SkinnyArgs args = {};
  if (p.k > 0) {
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
      ok = ok && operand_map(&maps.w[i], p.dtype, concat || GATED ? p.b[i] : p.b[0], p.n, p.k, kOutRows);
      ok = ok && operand_map(&maps.a[i], p.dtype, concat ? p.a[i] : p.a[0], p.m, p.k, BT);
    }
    if (!ok) return cudaErrorInvalidValue;
  }
  args.m = static_cast<int>(p.m);
  args.n = static_cast<int>(p.n);
  args.kb_part = static_cast<int>((p.k + kBK - 1) / kBK);
  args.kb_total = args.kb_part * (concat ? 2 : 1);
  args.act = p.act;
  args.residual = p.residual;
  args.ld_residual = p.ld_residual;
  args.out = p.out[0];
  args.ld_out = p.ld_out;
  args.ld_pre = p.ld_pre;
  args.err = err;
  args.flags = p.flags;
  for (int i = 0; i < 2; ++i) {
    args.bias[i] = p.bias[i];
    args.pre[i] = p.pre[i];
  }
  const int64_t tiles_n = (p.n + kOutRows - 1) / kOutRows, tiles_m = (p.m + BT - 1) / BT;
  if (tiles_m > 65535 || tiles_n > 65535) return cudaErrorInvalidValue;
  // As many K ranges as still run at once, each of at least four K blocks (a
  // shorter range is all latency).  The receive buffer is sized for these
  // counts; 3 fills the device where 2 leaves 40 % of it idle (32 x 11008 x
  // 4096: 19.2 us in 2 ranges, 17.8 in 3).  Clusters of 8 stay inside a GPC:
  // 33 of them run at once with two CTAs per SM, 15 with one.
  const int64_t eights = int64_t{sm_count} * (Cfg::kPerSm == 2 ? 33 : 15) / 148;
  int split = 1;
  for (int q : {2, 3, 4, 8}) {
    const int64_t tiles = tiles_n * tiles_m;
    if ((q == 8 ? tiles <= eights : tiles * q <= Cfg::kPerSm * sm_count) && args.kb_total / q >= 4) split = q;
  }
  args.split = split;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(split), static_cast<unsigned>(tiles_m), static_cast<unsigned>(tiles_n));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (p.flags & GLQ_FLAG_NO_PDL) ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, skinny_kernel<T, BT, W_MN, GATED>, maps, args);
}

template <typename T, int BT>
cudaError_t launch_order(const Product& p, int sm_count, unsigned int* err, cudaStream_t s) {
  const bool w_mn = !p.b[0].k_major;
  if (p.parts == Parts::kGated) {
    return w_mn ? launch_typed<T, BT, true, true>(p, sm_count, err, s)
                : launch_typed<T, BT, false, true>(p, sm_count, err, s);
  }
  return w_mn ? launch_typed<T, BT, true, false>(p, sm_count, err, s)
              : launch_typed<T, BT, false, false>(p, sm_count, err, s);
}

template <typename T>
cudaError_t launch_tokens(const Product& p, int sm_count, unsigned int* err, cudaStream_t s) {
  if (p.m <= 16) return launch_order<T, 16>(p, sm_count, err, s);
  if (p.m <= 32) return launch_order<T, 32>(p, sm_count, err, s);
  if (p.m <= 64) return launch_order<T, 64>(p, sm_count, err, s);
  if (p.m <= 128 || p.k == 0) return launch_order<T, 128>(p, sm_count, err, s);
  return launch_order<T, 192>(p, sm_count, err, s);
}

template <typename T, int BT>
cudaError_t set_attrs() {
  const int bytes = static_cast<int>(SkinnyConfig<BT>::kSmem);
  constexpr cudaFuncAttribute kAttr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(skinny_kernel<T, BT, false, false>, kAttr, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(skinny_kernel<T, BT, true, false>, kAttr, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(skinny_kernel<T, BT, false, true>, kAttr, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(skinny_kernel<T, BT, true, true>, kAttr, bytes);
  return e;
}

template <typename T>
cudaError_t set_attrs_all() {
  cudaError_t e = set_attrs<T, 16>();
  if (e == cudaSuccess) e = set_attrs<T, 32>();
  if (e == cudaSuccess) e = set_attrs<T, 64>();
  if (e == cudaSuccess) e = set_attrs<T, 128>();
  if (e == cudaSuccess) e = set_attrs<T, 192>();
  return e;
}

}  // namespace

cudaError_t skinny_prepare_device() {
  const cudaError_t e = set_attrs_all<__half>();
  return e != cudaSuccess ? e : set_attrs_all<__nv_bfloat16>();
}

cudaError_t launch_skinny(const Product& p, int sm_count, unsigned int* err, cudaStream_t s) {
  if (p.m < 1 || p.n < 1 || p.parts == Parts::kTwo || (p.k > 0 && !p.a[0].k_major)) return cudaErrorInvalidValue;
  return p.dtype == GLQ_DTYPE_BF16 ? launch_tokens<__nv_bfloat16>(p, sm_count, err, s)
                                   : launch_tokens<__half>(p, sm_count, err, s);
}

}  // namespace glq
