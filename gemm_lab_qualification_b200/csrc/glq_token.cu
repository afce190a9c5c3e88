// glq_token.cu -- the feed-forward operators' forward products for a single
// token: out[n] = epilogue(sum_k x[k] W[n, k]) with K-contiguous weight rows.
//
// Bound: the bytes of W (two multiply-adds per four bytes).  Tensor cores
// have nothing to add for one token, and what the skinny kernel spends on
// tensor memory, cluster joins and deep rings shows: a product of 33 MB took
// 9.0 us there, 180 MB (gated) 31.9 us.  Here each warp streams one weight row
// (gated: the gate row and the up row, sharing x) in 16-byte loads, four per
// row and lane in flight, x comes from L1, products are added in 32-bit pairs,
// and lanes join by shuffles.  Rows too few to fill the device are shared by
// 2, 4 or 8 warps of a block, joined in order through shared memory.
#include <cuda_runtime.h>

#include <algorithm>

#include "glq_act.cuh"
#include "glq_ffn.h"
#include "glq_internal.h"
#include "glq_ptx.cuh"

namespace glq {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 4;  // loads per row and lane in flight

struct TokenArgs {
  const void* x;
  const void* w[2];
  long long pitch[2];
  int n, k;
  int per_row;  // warps that share a row
  const void* bias[2];
  int act;
  const void* residual;
  void* out;
  void* pre[2];
};

// acc += the products of eight elements.
template <typename T>
__device__ __forceinline__ void dot8(const uint4& w, const float2 (&x)[4], float2& acc) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem16<T>::to_f2(v[i]);
    acc.x = fmaf(f.x, x[i].x, acc.x);
    acc.y = fmaf(f.y, x[i].y, acc.y);
  }
}

template <typename T>
__device__ __forceinline__ void widen(const uint4& x, float2 (&f)[4]) {
  f[0] = Elem16<T>::to_f2(x.x);
  f[1] = Elem16<T>::to_f2(x.y);
  f[2] = Elem16<T>::to_f2(x.z);
  f[3] = Elem16<T>::to_f2(x.w);
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kThreads, GATED ? 3 : 4) token_kernel(const TokenArgs a) {
  using E = Elem16<T>;
  constexpr int kRows = GATED ? 2 : 1;
  __shared__ float sums[kRows][kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = warp % a.per_row;
  const int n = blockIdx.x * (kWarps / a.per_row) + warp / a.per_row;
  const bool live = n < a.n;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  float2 acc[kRows] = {};
  if (live) {
    const T* x = static_cast<const T*>(a.x);
    const T* w[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) w[r] = static_cast<const T*>(a.w[r]) + static_cast<long long>(n) * a.pitch[r];
    const int whole = a.k & ~7;  // whole 16-byte chunks
    const int step = a.per_row * 256;
    int c = share * 256 + lane * 8;
    for (; c + (kAhead - 1) * step < whole; c += kAhead * step) {
      uint4 v[kRows][kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) v[r][i] = ptx::ldg_stream_v4(w[r] + c + i * step);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        float2 f[4];
        widen<T>(*reinterpret_cast<const uint4*>(x + c + i * step), f);
#pragma unroll
        for (int r = 0; r < kRows; ++r) dot8<T>(v[r][i], f, acc[r]);
      }
    }
    for (; c < whole; c += step) {
      float2 f[4];
      widen<T>(*reinterpret_cast<const uint4*>(x + c), f);
#pragma unroll
      for (int r = 0; r < kRows; ++r) dot8<T>(ptx::ldg_stream_v4(w[r] + c), f, acc[r]);
    }
    if (share == 0 && whole + lane < a.k) {  // the last elements of a row one by one
#pragma unroll
      for (int r = 0; r < kRows; ++r) acc[r].x = fmaf(E::to_f(w[r][whole + lane]), E::to_f(x[whole + lane]), acc[r].x);
    }
  }
  float s[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    s[r] = acc[r].x + acc[r].y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
  }
  if (a.per_row > 1) {
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) sums[r][warp] = s[r];
    }
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        for (int q = 1; q < a.per_row; ++q) s[r] += sums[r][warp + q];
      }
    }
  }
  if (live && share == 0 && lane == 0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (a.bias[r] != nullptr) s[r] += E::to_f(static_cast<const T*>(a.bias[r])[n]);
      if (a.pre[r] != nullptr) static_cast<T*>(a.pre[r])[n] = E::from_f(s[r]);
    }
    float y = s[0];
    with_act(a.act, [&](auto act) { y = act_f<decltype(act)::value>(y); });
    if constexpr (GATED) {
      y *= s[kRows - 1];
    } else {
      if (a.residual != nullptr) y += E::to_f(static_cast<const T*>(a.residual)[n]);
    }
    static_cast<T*>(a.out)[n] = E::from_f(y);
  }
}

template <typename T>
cudaError_t launch_typed(const TokenArgs& args, bool gated, unsigned int flags, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int rows = kWarps / args.per_row;
  cfg.gridDim = dim3(static_cast<unsigned>((args.n + rows - 1) / rows));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & GLQ_FLAG_NO_PDL) ? 0 : 1;
  return gated ? cudaLaunchKernelEx(&cfg, token_kernel<T, true>, args)
               : cudaLaunchKernelEx(&cfg, token_kernel<T, false>, args);
}

}  // namespace

cudaError_t launch_token(const Product& p, int sm_count, cudaStream_t s) {
  const bool gated = p.parts == Parts::kGated;
  if (p.m != 1 || p.n < 1 || p.k < 1 || (!gated && p.parts != Parts::kOne) || !p.a[0].k_major || !p.b[0].k_major ||
      (gated && !p.b[1].k_major)) {
    return cudaErrorInvalidValue;
  }
  TokenArgs args = {};
  args.x = p.a[0].base;
  args.n = static_cast<int>(p.n);
  args.k = static_cast<int>(p.k);
  args.act = p.act;
  args.residual = p.residual;
  args.out = p.out[0];
  for (int i = 0; i < 2; ++i) {
    args.w[i] = p.b[i].base;
    args.pitch[i] = p.b[i].pitch;
    args.bias[i] = p.bias[i];
    args.pre[i] = p.pre[i];
  }
  // The share of a row per warp with the fewest waves of work, each at least
  // one batch of loads; every doubling costs about a quarter (shorter streams
  // between a warp's start and its join).  1024 x 11008: 10.3, 7.5, 6.8 and 7.9
  // us with 1, 2, 4 and 8 warps per row; 4096 x 4096: 7.1, 7.7, 8.8 us.
  const int64_t at_once = int64_t{sm_count} * kWarps * (gated ? 3 : 4);
  int per_row = 1;
  double best = 0.0, toll = 1.0;
  for (int q = 1; q <= kWarps && (q == 1 || p.k >= int64_t{q} * 256 * kAhead); q *= 2, toll += 0.25) {
    const double waves = toll * static_cast<double>((p.n * q + at_once - 1) / at_once) / q;
    if (best == 0.0 || waves < best) {
      best = waves;
      per_row = q;
    }
  }
  args.per_row = per_row;
  return p.dtype == GLQ_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(args, gated, p.flags, s)
                                   : launch_typed<__half>(args, gated, p.flags, s);
}

}  // namespace glq
