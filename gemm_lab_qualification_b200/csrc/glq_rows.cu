// glq_rows.cu -- the memory-bound kernels of the feed-forward operators:
// layer norm forward and backward, the activations' backward pass, and the
// column sums (gradients of biases and of the norm's weight) that both share.
//
// All are bound by HBM: each tensor is read and written once, in 16-byte
// vectors where its rows allow, with every statistic and sum in FP32.
// Column sums are two fixed-order stages, rows of a block in registers and
// then the blocks' partial rows, so results do not depend on timing.
#include <cuda_runtime.h>

#include <algorithm>

#include "glq_act.cuh"
#include "glq_ptx.cuh"
#include "glq_rows.h"

namespace glq {
namespace {

// Eight consecutive elements of a row as floats; vec: 16-byte aligned and
// all inside, else `valid` of them element by element (the rest 0).
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int valid, float (&v)[8]) {
  if (vec) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem16<T>::to_f2(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? Elem16<T>::to_f(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int valid, const float (&v)[8]) {
  if (vec) {
    uint4 x;
    x.x = Elem16<T>::from_f2(v[0], v[1]);
    x.y = Elem16<T>::from_f2(v[2], v[3]);
    x.z = Elem16<T>::from_f2(v[4], v[5]);
    x.w = Elem16<T>::from_f2(v[6], v[7]);
    *reinterpret_cast<uint4*>(p) = x;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < valid) p[i] = Elem16<T>::from_f(v[i]);
    }
  }
}

// Sum of N values over the G threads of a row (all threads of the block call
// it; blocks of more than a warp per row use shared memory, red[2][32 N]).
template <int G, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& phase) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* buf = red + phase * 32 * N;  // two buffers: one barrier per sum
    phase ^= 1;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[warp * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += buf[w * N + i];
    }
  }
}

// ---------------------------------------------------------------- layer norm
//
// A row is held in registers by G threads (V vectors of 8 each), so x is read
// once and the variance is the mean of the squared deviations from the mean
// (no cancellation of large squares).  Rows of up to 512 columns take one
// warp each, four rows per block.

template <int G>
constexpr int kRowsPerBlock = G == 32 ? 4 : 1;

template <typename T, int G, int V>
__global__ void __launch_bounds__(G * kRowsPerBlock<G>)
    norm_kernel(const NormArgs a) {
  __shared__ float red[2 * 32];
  int phase = 0;
  const int in_row = threadIdx.x % G;
  const int first = blockIdx.x * kRowsPerBlock<G> + threadIdx.x / G;
  const int cols = a.cols;
  const float inv = 1.0f / static_cast<float>(cols);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const T* weight = static_cast<const T*>(a.weight);
  const T* bias = static_cast<const T*>(a.bias);
  for (long long r0 = first; r0 - threadIdx.x / G < a.rows; r0 += static_cast<long long>(gridDim.x) * kRowsPerBlock<G>) {
    const bool live = r0 < a.rows;  // whole warps: G >= 32
    const T* x = static_cast<const T*>(a.x) + r0 * a.ld_x;
    float v[V][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * G + in_row) * 8;
      load8(x + c, live && a.vec && c < cols, live ? cols - c : 0, v[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[0] += v[j][i];
    }
    row_sum<G>(sum, red, phase);
    const float mean = sum[0] * inv;
    float sq[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * G + in_row) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] -= mean;
        if (c + i < cols) sq[0] += v[j][i] * v[j][i];
      }
    }
    row_sum<G>(sq, red, phase);
    const float rstd = rsqrtf(sq[0] * inv + a.eps);
    if (!live) continue;
    T* y = static_cast<T*>(a.y) + r0 * a.ld_y;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * G + in_row) * 8;
      if (c >= cols) continue;
      float w[8], b[8];
      if (weight != nullptr) load8(weight + c, a.vec_w, cols - c, w);
      if (bias != nullptr) load8(bias + c, a.vec_w, cols - c, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] *= rstd;
        if (weight != nullptr) v[j][i] *= w[i];
        if (bias != nullptr) v[j][i] += b[i];
      }
      store8(y + c, a.vec, cols - c, v[j]);
    }
    if (in_row == 0 && a.mean != nullptr) {
      a.mean[r0] = mean;
      a.rstd[r0] = rstd;
    }
  }
}

// Rows longer than the register kernels hold: the same sums in three passes
// over the row (it stays in L2).
template <typename T>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormArgs a) {
  __shared__ float red[2 * 32];
  int phase = 0;
  const float inv = 1.0f / static_cast<float>(a.cols);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const T* weight = static_cast<const T*>(a.weight);
  const T* bias = static_cast<const T*>(a.bias);
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ld_x;
    T* y = static_cast<T*>(a.y) + r * a.ld_y;
    float sum[1] = {0.0f}, sq[1] = {0.0f}, v[8];
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      load8(x + c, a.vec, a.cols - c, v);
      for (int i = 0; i < 8; ++i) sum[0] += v[i];
    }
    row_sum<1024>(sum, red, phase);
    const float mean = sum[0] * inv;
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      load8(x + c, a.vec, a.cols - c, v);
      for (int i = 0; i < 8; ++i) {
        if (c + i < a.cols) sq[0] += (v[i] - mean) * (v[i] - mean);
      }
    }
    row_sum<1024>(sq, red, phase);
    const float rstd = rsqrtf(sq[0] * inv + a.eps);
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      float w[8], b[8];
      load8(x + c, a.vec, a.cols - c, v);
      if (weight != nullptr) load8(weight + c, a.vec_w, a.cols - c, w);
      if (bias != nullptr) load8(bias + c, a.vec_w, a.cols - c, b);
      for (int i = 0; i < 8; ++i) {
        v[i] = (v[i] - mean) * rstd;
        if (weight != nullptr) v[i] *= w[i];
        if (bias != nullptr) v[i] += b[i];
      }
      store8(y + c, a.vec, a.cols - c, v);
    }
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

// Backward.  With xhat = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  dw = sum_r dy xhat,
//   db = sum_r dy.
// A block walks rows blockIdx.x, + gridDim.x, ... and keeps its columns' dw
// and db sums in registers; partial rows go to part[block row][2][cols].
template <typename T, int G, int V>
__global__ void __launch_bounds__(G * kRowsPerBlock<G>)
    norm_backward_kernel(const NormBackwardArgs a) {
  __shared__ float red[2 * 32 * 2];
  int phase = 0;
  const int in_row = threadIdx.x % G;
  const int sub = threadIdx.x / G;
  const int cols = a.cols;
  const float inv = 1.0f / static_cast<float>(cols);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const T* weight = static_cast<const T*>(a.weight);
  float w[V][8], dw[V][8], db[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * G + in_row) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[j][i] = 1.0f;
      dw[j][i] = 0.0f;
      db[j][i] = 0.0f;
    }
    if (weight != nullptr && c < cols) load8(weight + c, a.vec_w, cols - c, w[j]);
  }
  for (long long r0 = static_cast<long long>(blockIdx.x) * kRowsPerBlock<G> + sub; r0 - sub < a.rows;
       r0 += static_cast<long long>(gridDim.x) * kRowsPerBlock<G>) {
    const bool live = r0 < a.rows;
    const T* x = static_cast<const T*>(a.x) + r0 * a.ld_x;
    const T* dy = static_cast<const T*>(a.dy) + r0 * a.ld_dy;
    const float mean = live ? a.mean[r0] : 0.0f;
    const float rstd = live ? a.rstd[r0] : 0.0f;
    float xh[V][8], g[V][8];
    float sum[2] = {0.0f, 0.0f};  // of g xhat and of g
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * G + in_row) * 8;
      load8(x + c, live && a.vec && c < cols, live ? cols - c : 0, xh[j]);
      load8(dy + c, live && a.vec && c < cols, live ? cols - c : 0, g[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xh[j][i] = (xh[j][i] - mean) * rstd;  // columns past the end: g is 0
        dw[j][i] += g[j][i] * xh[j][i];
        db[j][i] += g[j][i];
        g[j][i] *= w[j][i];
        sum[0] += g[j][i] * xh[j][i];
        sum[1] += g[j][i];
      }
    }
    row_sum<G>(sum, red, phase);
    const float c1 = sum[0] * inv, c2 = sum[1] * inv;
    if (!live) continue;
    T* dx = static_cast<T*>(a.dx) + r0 * a.ld_dx;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * G + in_row) * 8;
      if (c >= cols) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) g[j][i] = (g[j][i] - c2 - xh[j][i] * c1) * rstd;
      store8(dx + c, a.vec, cols - c, g[j]);
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + (static_cast<long long>(blockIdx.x) * kRowsPerBlock<G> + sub) * 2 * a.part_cols;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * G + in_row) * 8;
    if (c >= cols) continue;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {  // part_cols is a multiple of 8
      *reinterpret_cast<float4*>(part + c + i) = make_float4(dw[j][i], dw[j][i + 1], dw[j][i + 2], dw[j][i + 3]);
      *reinterpret_cast<float4*>(part + a.part_cols + c + i) =
          make_float4(db[j][i], db[j][i + 1], db[j][i + 2], db[j][i + 3]);
    }
  }
}

// Rows longer than the register kernels hold: dx by rows in two passes ...
template <typename T>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(const NormBackwardArgs a) {
  __shared__ float red[2 * 32 * 2];
  int phase = 0;
  const float inv = 1.0f / static_cast<float>(a.cols);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const T* weight = static_cast<const T*>(a.weight);
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ld_x;
    const T* dy = static_cast<const T*>(a.dy) + r * a.ld_dy;
    T* dx = static_cast<T*>(a.dx) + r * a.ld_dx;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sum[2] = {0.0f, 0.0f}, xv[8], g[8], w[8];
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      load8(x + c, a.vec, a.cols - c, xv);
      load8(dy + c, a.vec, a.cols - c, g);
      if (weight != nullptr) load8(weight + c, a.vec_w, a.cols - c, w);
      for (int i = 0; i < 8; ++i) {
        const float gw = weight != nullptr ? g[i] * w[i] : g[i];
        sum[0] += gw * (xv[i] - mean) * rstd;
        sum[1] += gw;
      }
    }
    row_sum<1024>(sum, red, phase);
    const float c1 = sum[0] * inv, c2 = sum[1] * inv;
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      load8(x + c, a.vec, a.cols - c, xv);
      load8(dy + c, a.vec, a.cols - c, g);
      if (weight != nullptr) load8(weight + c, a.vec_w, a.cols - c, w);
      for (int i = 0; i < 8; ++i) {
        const float gw = weight != nullptr ? g[i] * w[i] : g[i];
        g[i] = (gw - c2 - (xv[i] - mean) * rstd * c1) * rstd;
      }
      store8(dx + c, a.vec, a.cols - c, g);
    }
  }
}

// ... and the column sums by strips of rows.
template <typename T>
__global__ void __launch_bounds__(128) norm_columns_kernel(const NormBackwardArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int c = (blockIdx.x * 128 + threadIdx.x) * 8;
  if (c >= a.cols) return;
  const long long lo = static_cast<long long>(blockIdx.y) * a.rows / gridDim.y;
  const long long hi = static_cast<long long>(blockIdx.y + 1) * a.rows / gridDim.y;
  float dw[8] = {}, db[8] = {};
  for (long long r = lo; r < hi; ++r) {
    float xv[8], g[8];
    load8(static_cast<const T*>(a.x) + r * a.ld_x + c, a.vec, a.cols - c, xv);
    load8(static_cast<const T*>(a.dy) + r * a.ld_dy + c, a.vec, a.cols - c, g);
    const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[i] += g[i] * (xv[i] - mean) * rstd;
      db[i] += g[i];
    }
  }
  float* part = a.part + static_cast<long long>(blockIdx.y) * 2 * a.part_cols;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    part[c + i] = dw[i];
    part[a.part_cols + c + i] = db[i];
  }
}

// ---------------------------------------------------------------- column sums
//
// out[c] = sum over p of part[p][c], in order of p inside each of 8 strided
// ranges, then the 8 in order.  32 columns x 8 ranges per block.
template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const ColumnSumArgs a) {
  __shared__ float sums[8][33];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int which = blockIdx.y;  // sums side by side in a partial row
  float s = 0.0f;
  if (c < a.cols) {
    const float* p = a.part + static_cast<long long>(which) * a.part_cols + c;
    for (int i = q; i < a.parts; i += 8) s += p[static_cast<long long>(i) * a.sums * a.part_cols];
  }
  sums[q][lane] = s;
  __syncthreads();
  if (q == 0 && c < a.cols && a.out[which] != nullptr) {
    float t = sums[0][lane];
#pragma unroll
    for (int i = 1; i < 8; ++i) t += sums[i][lane];
    static_cast<T*>(a.out[which])[c] = Elem16<T>::from_f(t);
  }
}

// ---------------------------------------------------------------- activations
//
// Linear: dz = dy act'(z).  Gated: dg = dy u act'(g), du = dy act(g).  One
// block: 1024 columns x a strip of rows, 8 columns per thread; the bias
// gradients' partial sums of the strip (of the values before their rounding)
// stay in registers.  The rounding of dz to 16 bits is what the tensor-core
// products that follow read.
template <typename T, bool GATED>
__global__ void __launch_bounds__(128) act_backward_kernel(const ActBackwardArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int c = (blockIdx.x * 128 + threadIdx.x) * 8;
  if (c >= a.cols) return;
  const long long lo = static_cast<long long>(blockIdx.y) * a.rows / gridDim.y;
  const long long hi = static_cast<long long>(blockIdx.y + 1) * a.rows / gridDim.y;
  const int valid = a.cols - c;
  float s0[8] = {}, s1[8] = {};
  with_act(a.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
#pragma unroll 2
    for (long long r = lo; r < hi; ++r) {
      float g[8], z[8], u[8], d0[8], d1[8];
      load8(static_cast<const T*>(a.dy) + r * a.ld_dy + c, a.vec_dy, valid, g);
      if (GATED || ACT != GLQ_ACT_NONE) load8(static_cast<const T*>(a.pre[0]) + r * a.ld_pre + c, a.vec_pre, valid, z);
      if (GATED) load8(static_cast<const T*>(a.pre[1]) + r * a.ld_pre + c, a.vec_pre, valid, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float value = 0.0f, slope = 1.0f;
        if (GATED || ACT != GLQ_ACT_NONE) act_grad_f<ACT>(z[i], &value, &slope);
        if (GATED) {
          d0[i] = g[i] * u[i] * slope;
          d1[i] = g[i] * value;
          s1[i] += i < valid ? d1[i] : 0.0f;
        } else {
          d0[i] = g[i] * slope;
        }
        s0[i] += i < valid ? d0[i] : 0.0f;
      }
      if (a.dz[0] != nullptr) {  // null: column sums only
        store8(static_cast<T*>(a.dz[0]) + r * a.ld_dz + c, a.vec_dz, valid, d0);
        if (GATED) store8(static_cast<T*>(a.dz[1]) + r * a.ld_dz + c, a.vec_dz, valid, d1);
      }
    }
  });
  if (a.part != nullptr) {
    constexpr int kSums = GATED ? 2 : 1;
    float* part = a.part + static_cast<long long>(blockIdx.y) * kSums * a.part_cols + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[i] = s0[i];
      if (GATED) part[a.part_cols + i] = s1[i];
    }
  }
}

// ---------------------------------------------------------------- host

template <typename Kernel, typename Args>
cudaError_t launch(Kernel kernel, dim3 grid, int threads, const Args& args, unsigned int flags, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & GLQ_FLAG_NO_PDL) ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args);
}

bool vec_rows(const void* p, int64_t ld, int64_t cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && cols % 8 == 0;
}

// Threads per row and vectors per thread of the register kernels.
template <typename T, template <typename, int, int> class Launch, typename Args>
cudaError_t by_columns(const Args& a, int grid, unsigned int flags, cudaStream_t s) {
  if (a.cols <= 256) return Launch<T, 32, 1>::run(a, grid, flags, s);
  if (a.cols <= 512) return Launch<T, 32, 2>::run(a, grid, flags, s);
  if (a.cols <= 1024) return Launch<T, 128, 1>::run(a, grid, flags, s);
  if (a.cols <= 2048) return Launch<T, 128, 2>::run(a, grid, flags, s);
  if (a.cols <= 4096) return Launch<T, 256, 2>::run(a, grid, flags, s);
  if (a.cols <= 8192) return Launch<T, 512, 2>::run(a, grid, flags, s);
  return Launch<T, 1024, 2>::run(a, grid, flags, s);
}

template <typename T, int G, int V>
struct LaunchNorm {
  static cudaError_t run(const NormArgs& a, int grid, unsigned int flags, cudaStream_t s) {
    return launch(norm_kernel<T, G, V>, dim3(grid), G * kRowsPerBlock<G>, a, flags, s);
  }
};

template <typename T, int G, int V>
struct LaunchNormBackward {
  static cudaError_t run(const NormBackwardArgs& a, int grid, unsigned int flags, cudaStream_t s) {
    return launch(norm_backward_kernel<T, G, V>, dim3(grid), G * kRowsPerBlock<G>, a, flags, s);
  }
};

int rows_per_block(int cols) { return cols <= 512 ? 4 : 1; }

// Threads of the register kernels' blocks.
int block_threads(int cols) {
  return cols <= 2048 ? 128 : cols <= 4096 ? 256 : cols <= 8192 ? 512 : 1024;
}

// Blocks of the backward register kernel: as many as fill the SMs (about
// 1024 threads of it each at its register use), at most one per row group.
int64_t backward_blocks(int64_t rows, int64_t cols, int sm_count) {
  const int64_t groups = (rows + rows_per_block(static_cast<int>(cols)) - 1) / rows_per_block(static_cast<int>(cols));
  return std::max<int64_t>(1, std::min<int64_t>(groups, int64_t{sm_count} * (1024 / block_threads(static_cast<int>(cols)))));
}

int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }

// Row strips of the column kernels: enough blocks for four per SM.
int64_t strips(int64_t rows, int64_t cols, int sm_count) {
  const int64_t across = (cols + 1023) / 1024;
  return std::max<int64_t>(1, std::min<int64_t>(rows, std::min<int64_t>(4096, (int64_t{sm_count} * 8 + across - 1) / across)));
}

template <typename T>
cudaError_t norm_typed(const NormArgs& a, int sm_count, unsigned int flags, cudaStream_t s) {
  if (a.cols > kNormRegisterCols) {
    return launch(norm_long_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, 2 * sm_count))), 1024, a,
                  flags, s);
  }
  const int64_t groups = (a.rows + rows_per_block(a.cols) - 1) / rows_per_block(a.cols);
  return by_columns<T, LaunchNorm>(a, static_cast<int>(std::min<int64_t>(groups, 1 << 20)), flags, s);
}

template <typename T>
cudaError_t norm_backward_typed(NormBackwardArgs a, void* dweight, void* dbias, int sm_count, unsigned int flags,
                                cudaStream_t s) {
  int64_t parts = 0;
  cudaError_t e;
  if (a.cols > kNormRegisterCols) {
    e = launch(norm_backward_long_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, 2 * sm_count))),
               1024, a, flags, s);
    parts = strips(a.rows, a.cols, sm_count);
    if (e == cudaSuccess && a.part != nullptr) {
      e = launch(norm_columns_kernel<T>, dim3(static_cast<unsigned>((a.cols + 1023) / 1024), static_cast<unsigned>(parts)),
                 128, a, flags, s);
    }
  } else {
    const int64_t grid = backward_blocks(a.rows, a.cols, sm_count);
    parts = grid * rows_per_block(a.cols);
    e = by_columns<T, LaunchNormBackward>(a, static_cast<int>(grid), flags, s);
  }
  if (e != cudaSuccess || a.part == nullptr) return e;
  ColumnSumArgs c = {};
  c.part = a.part;
  c.part_cols = a.part_cols;
  c.parts = static_cast<int>(parts);
  c.sums = 2;
  c.cols = a.cols;
  c.out[0] = dweight;
  c.out[1] = dbias;
  return launch(column_sum_kernel<T>, dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), 256, c, flags, s);
}

template <typename T>
cudaError_t act_backward_typed(const ActBackwardArgs& a, bool gated, void* const* dbias, int64_t n_strips,
                               unsigned int flags, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.cols + 1023) / 1024), static_cast<unsigned>(n_strips));
  cudaError_t e = gated ? launch(act_backward_kernel<T, true>, grid, 128, a, flags, s)
                        : launch(act_backward_kernel<T, false>, grid, 128, a, flags, s);
  if (e != cudaSuccess || a.part == nullptr) return e;
  ColumnSumArgs c = {};
  c.part = a.part;
  c.part_cols = a.part_cols;
  c.parts = static_cast<int>(n_strips);
  c.sums = gated ? 2 : 1;
  c.cols = a.cols;
  c.out[0] = dbias[0];
  c.out[1] = gated ? dbias[1] : nullptr;
  return launch(column_sum_kernel<T>, dim3(static_cast<unsigned>((a.cols + 31) / 32), static_cast<unsigned>(c.sums)), 256,
                c, flags, s);
}

}  // namespace

size_t norm_backward_partial_bytes(int64_t rows, int64_t cols, int sm_count) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t parts = cols > kNormRegisterCols
                            ? strips(rows, cols, sm_count)
                            : backward_blocks(rows, cols, sm_count) * rows_per_block(static_cast<int>(cols));
  return static_cast<size_t>(parts * 2 * padded(cols)) * sizeof(float);
}

size_t act_backward_partial_bytes(int64_t rows, int64_t cols, int sums, int sm_count) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(strips(rows, cols, sm_count) * sums * padded(cols)) * sizeof(float);
}

cudaError_t launch_norm(int dtype, NormArgs a, int sm_count, unsigned int flags, cudaStream_t s) {
  a.vec = vec_rows(a.x, a.ld_x, a.cols) && vec_rows(a.y, a.ld_y, a.cols);
  a.vec_w = vec_rows(a.weight, 0, a.cols) && vec_rows(a.bias, 0, a.cols);
  return dtype == GLQ_DTYPE_BF16 ? norm_typed<__nv_bfloat16>(a, sm_count, flags, s)
                                 : norm_typed<__half>(a, sm_count, flags, s);
}

cudaError_t launch_norm_backward(int dtype, NormBackwardArgs a, void* dweight, void* dbias, int sm_count,
                                 unsigned int flags, cudaStream_t s) {
  a.vec = vec_rows(a.x, a.ld_x, a.cols) && vec_rows(a.dy, a.ld_dy, a.cols) && vec_rows(a.dx, a.ld_dx, a.cols);
  a.vec_w = vec_rows(a.weight, 0, a.cols);
  a.part_cols = padded(a.cols);
  return dtype == GLQ_DTYPE_BF16 ? norm_backward_typed<__nv_bfloat16>(a, dweight, dbias, sm_count, flags, s)
                                 : norm_backward_typed<__half>(a, dweight, dbias, sm_count, flags, s);
}

cudaError_t launch_act_backward(int dtype, bool gated, ActBackwardArgs a, void* const* dbias, int sm_count,
                                unsigned int flags, cudaStream_t s) {
  a.vec_dy = vec_rows(a.dy, a.ld_dy, a.cols);
  a.vec_pre = vec_rows(a.pre[0], a.ld_pre, a.cols) && vec_rows(a.pre[1], a.ld_pre, a.cols);
  a.vec_dz = vec_rows(a.dz[0], a.ld_dz, a.cols) && vec_rows(a.dz[1], a.ld_dz, a.cols);
  a.part_cols = padded(a.cols);
  const int64_t n = strips(a.rows, a.cols, sm_count);
  return dtype == GLQ_DTYPE_BF16 ? act_backward_typed<__nv_bfloat16>(a, gated, dbias, n, flags, s)
                                 : act_backward_typed<__half>(a, gated, dbias, n, flags, s);
}

}  // namespace glq
