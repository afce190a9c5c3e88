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
#include "glq_internal.h"
#include "glq_ptx.cuh"
#include "glq_rows.h"

namespace glq {
namespace {

// Eight consecutive 16-bit elements of a row.  align: bytes that every row's
// start is a multiple of (16, 8, 4 or 2); fewer than 8 valid elements are read
// and written one by one (the rest 0).
template <typename T>
__device__ __forceinline__ uint4 load8_raw(const T* p, int align, int valid) {
  if (valid >= 8 && align == 16) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
  if (valid >= 8 && align == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p), y = *reinterpret_cast<const uint2*>(p + 4);
    w[0] = x.x, w[1] = x.y, w[2] = y.x, w[3] = y.y;
  } else if (valid >= 8 && align == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 2 * i);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < valid ? q[2 * i] : 0u, hi = 2 * i + 1 < valid ? q[2 * i + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void store8_raw(T* p, int align, int valid, const uint4& x) {
  if (valid >= 8 && align == 16) {
    *reinterpret_cast<uint4*>(p) = x;
    return;
  }
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if (valid >= 8 && align == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(p + 4) = make_uint2(w[2], w[3]);
  } else if (valid >= 8 && align == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(p + 2 * i) = w[i];
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < valid) q[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
    }
  }
}

// The same as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int align, int valid, float (&v)[8]) {
  const uint4 x = load8_raw(p, align, valid);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem16<T>::to_f2(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int align, int valid, const float (&v)[8]) {
  store8_raw(p, align, valid,
             make_uint4(Elem16<T>::from_f2(v[0], v[1]), Elem16<T>::from_f2(v[2], v[3]), Elem16<T>::from_f2(v[4], v[5]),
                        Elem16<T>::from_f2(v[6], v[7])));
}

// Which columns of a row a thread of its group of G holds: in its vector j of 8
// the pair i begins at column(j, i).  VEC (rows of whole 16-byte vectors): 8
// consecutive columns.  Other rows: a warp's 256 columns of a vector are dealt
// out in pairs, so that each of its loads and stores covers 128 bytes in a row
// (consecutive columns there, 2 to 8 bytes at a time from 512 bytes: 8192 x
// 4095 forward 117 us, backward 173 us; 61 and 111 so).
template <int G, bool VEC>
struct Columns {
  int first;
  __device__ __forceinline__ Columns() {
    const int t = threadIdx.x % G;
    first = VEC ? t * 8 : (t / 32) * 256 + (t % 32) * 2;
  }
  __device__ __forceinline__ int column(int j, int i) const { return first + j * G * 8 + (VEC ? 2 : 64) * i; }
};

// Loads and stores under a predicate instead of a branch: none waits for the
// one before it.
__device__ __forceinline__ uint32_t ld_u32_if(const void* p, bool on) {
  uint32_t v;
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n mov.b32 %0, 0;\n @q ld.global.b32 %0, [%1];\n}"
               : "=&r"(v) : "l"(p), "r"(static_cast<int>(on)));
  return v;
}
__device__ __forceinline__ uint32_t ld_u16_if(const void* p, bool on) {
  uint16_t v;
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n mov.b16 %0, 0;\n @q ld.global.b16 %0, [%1];\n}"
               : "=&h"(v) : "l"(p), "r"(static_cast<int>(on)));
  return v;
}
__device__ __forceinline__ void st_u32_if(void* p, bool on, uint32_t v) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q st.global.b32 [%0], %1;\n}"
               :: "l"(p), "r"(v), "r"(static_cast<int>(on)) : "memory");
}
__device__ __forceinline__ void st_u16_if(void* p, bool on, uint32_t v) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q st.global.b16 [%0], %1;\n}"
               :: "l"(p), "h"(static_cast<uint16_t>(v)), "r"(static_cast<int>(on)) : "memory");
}

__device__ __forceinline__ bool in_words(const void* row) { return (reinterpret_cast<uintptr_t>(row) & 3) == 0; }

// The pairs of vectors first to first + V of a row (0 past its end), by whole
// words where the row begins at one.
template <typename T, int V, typename C>
__device__ __forceinline__ void load_pairs(const T* row, const C& mine, int cols, uint4 (&out)[V], int first = 0) {
  const bool words = in_words(row);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    uint32_t w[4];
    if (words) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = mine.column(first + j, i);
        w[i] = ld_u32_if(row + c, c + 1 < cols);
      }
      if (cols & 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = mine.column(first + j, i);
          w[i] |= ld_u16_if(row + c, c + 1 == cols);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = mine.column(first + j, i);
        w[i] = ld_u16_if(row + c, c < cols) | (ld_u16_if(row + c + 1, c + 1 < cols) << 16);
      }
    }
    out[j] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T, typename C>
__device__ __forceinline__ void store_pairs(T* row, const C& mine, int cols, int j, const uint4& x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if (in_words(row)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = mine.column(j, i);
      st_u32_if(row + c, c + 1 < cols, w[i]);
      st_u16_if(row + c, c + 1 == cols, w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = mine.column(j, i);
      st_u16_if(row + c, c < cols, w[i]);
      st_u16_if(row + c + 1, c + 1 < cols, w[i] >> 16);
    }
  }
}

// Sum of N values over the G threads of a row.  Groups of more than a warp
// join through red[2][G / 32][N], their own, behind the group's named barrier;
// every thread adds the warps' sums in the same order.
template <int G, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& phase, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if constexpr (G > 32) {
    constexpr int kWarps = G / 32;
    const int warp = (threadIdx.x % G) >> 5, lane = threadIdx.x & 31;
    float* buf = red + phase * kWarps * N;  // two buffers: one barrier per sum
    phase ^= 1;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[warp * N + i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(G) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += buf[w * N + i];
    }
  }
}

// Two floats in one 64-bit register pair: one instruction adds or multiplies
// both, which the row kernels need to stay bound by memory.
using Two = unsigned long long;

__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& x, Two (&v)[4]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem16<T>::to_f2(w[i]);
    v[i] = two(f.x, f.y);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const Two (&v)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = halves(v[i]);
    w[i] = Elem16<T>::from_f2(f.x, f.y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows on their way to a group of threads: STAGES slots of ROWS tensors' rows
// in shared memory, filled by bulk copies that the group's first thread
// starts, so the bytes in flight do not depend on registers or on how long a
// row's joins take.  An expired wait raises the error word and lets the group
// go on (with what the slot holds), so no barrier is missed.
template <int ROWS, int STAGES>
struct RowRing {
  uint32_t slots, bars;  // shared-memory addresses
  uint32_t row_bytes;
  unsigned int* err;
  uint64_t policy;
  int fill = 0, use = 0;

  __device__ __forceinline__ void start(const void* const (&rows)[ROWS]) {
    const int s = fill % STAGES;
    ptx::mbar_arrive_expect_tx(bars + 8 * s, ROWS * row_bytes);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      ptx::bulk_load_1d(slots + (s * ROWS + i) * row_bytes, rows[i], row_bytes, bars + 8 * s, policy);
    }
    ++fill;
  }
  // Waits for the next slot and returns its address.
  __device__ uint32_t wait() {
    const int s = use % STAGES;
    if (!ptx::mbar_wait_bounded(bars + 8 * s, (use / STAGES) & 1, nullptr, kWaitBudgetNs)) {
      atomicOr(err, kErrTimeoutProducer);
    }
    ++use;
    return slots + s * ROWS * row_bytes;
  }
};

__device__ __forceinline__ uint4 ld_smem_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// ---------------------------------------------------------------- layer norm
//
// A row is held in registers by G threads (V vectors of 8 each), so x is read
// once and the variance is the mean of the squared deviations from the mean
// (no cancellation of large squares).  What bounds it is HBM, as long as loads
// are in flight while a row's two joins wait and the instructions per element
// stay below about a dozen: persistent groups of threads walk rows group,
// + groups, ..., each requesting its next row before it reduces the present
// one (one row per block instead: 159 us at 16384 x 8192; rows by bulk copies
// through shared memory: 123 us, the joins' latency then has too few groups
// per SM to hide behind), and arithmetic is paired.  VEC: rows of whole
// 16-byte vectors; other rows are held in pairs of columns (Columns).

// sum / n with inv = 1 / n rounded: the product and its remainder's share, so
// that the mean of a constant row is its value (sum * inv can be one bit off,
// which rstd magnifies).  A division here costs 2 % at 16384 x 8192.
__device__ __forceinline__ float quotient(float sum, float n, float inv) {
  const float q = sum * inv;
  const float exact = fmaf(fmaf(-q, n, sum), inv, q);
  return fabsf(q) <= 3.402823466e38f ? exact : q;  // (infinity has no remainder)
}

constexpr int kNormThreads = 256;

template <typename T, int G, int V, bool VEC>
__global__ void __launch_bounds__(G < kNormThreads ? kNormThreads : G, G < 512 ? 3 : 1) norm_kernel(const NormArgs a) {
  constexpr int kGroups = G < kNormThreads ? kNormThreads / G : 1;  // rows per block at a time
  __shared__ float red[kGroups * 2 * (G / 32)];
  int phase = 0;
  const int group = threadIdx.x / G;
  const Columns<G, VEC> mine;
  const int cols = a.cols;
  const float inv = 1.0f / static_cast<float>(cols);
  float* my_red = red + group * 2 * (G / 32);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const T* weight = static_cast<const T*>(a.weight);
  const T* bias = static_cast<const T*>(a.bias);
  const T* x = static_cast<const T*>(a.x);
  const long long step = static_cast<long long>(gridDim.x) * kGroups;
  long long r = static_cast<long long>(blockIdx.x) * kGroups + group;
  uint4 next[V];
  auto request = [&](long long row) {
    const T* from = x + row * a.ld_x;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = mine.column(j, 0);
        next[j] = c < cols ? ptx::ldg_stream_v4(from + c) : make_uint4(0, 0, 0, 0);
      }
    } else {
      load_pairs(from, mine, cols, next);
    }
  };
  if (r < a.rows) request(r);
  for (; r < a.rows; r += step) {
    Two v[V][4];
    Two acc = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      unpack<T>(next[j], v[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc = add2(acc, v[j][i]);
    }
    if (r + step < a.rows) request(r + step);
    float sum[1] = {halves(acc).x + halves(acc).y};
    row_sum<G>(sum, my_red, phase, group);
    const float mean = quotient(sum[0], static_cast<float>(cols), inv);
    const Two minus_mean = two(-mean, -mean);
    acc = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = mine.column(j, VEC ? 0 : i);
        v[j][i] = add2(v[j][i], minus_mean);
        if (!VEC && c + 1 >= cols) {  // past the end, or the last of an odd number
          v[j][i] = two(c < cols ? halves(v[j][i]).x : 0.0f, 0.0f);
        }
        if (!VEC || c < cols) acc = fma2(v[j][i], v[j][i], acc);
      }
    }
    sum[0] = halves(acc).x + halves(acc).y;
    row_sum<G>(sum, my_red, phase, group);
    const float rstd = rsqrtf(sum[0] * inv + a.eps);
    const Two scale = two(rstd, rstd);
    T* y = static_cast<T*>(a.y) + r * a.ld_y;
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = mul2(v[j][i], scale);
      if constexpr (VEC) {  // (align_w is 16)
        const int c = mine.column(j, 0);
        if (c >= cols) continue;
        Two w[4];
        if (weight != nullptr) {
          unpack<T>(*reinterpret_cast<const uint4*>(weight + c), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = mul2(v[j][i], w[i]);
        }
        if (bias != nullptr) {
          unpack<T>(*reinterpret_cast<const uint4*>(bias + c), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = add2(v[j][i], w[i]);
        }
        *reinterpret_cast<uint4*>(y + c) = pack<T>(v[j]);
      } else {
        uint4 raw[1];
        Two w[4];
        if (weight != nullptr) {
          load_pairs(weight, mine, cols, raw, j);
          unpack<T>(raw[0], w);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = mul2(v[j][i], w[i]);
        }
        if (bias != nullptr) {
          load_pairs(bias, mine, cols, raw, j);
          unpack<T>(raw[0], w);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = add2(v[j][i], w[i]);
        }
        store_pairs(y, mine, cols, j, pack<T>(v[j]));
      }
    }
    if (threadIdx.x % G == 0 && a.mean != nullptr) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
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
      load8(x + c, a.align, a.cols - c, v);
      for (int i = 0; i < 8; ++i) sum[0] += v[i];
    }
    row_sum<1024>(sum, red, phase, 0);
    const float mean = quotient(sum[0], static_cast<float>(a.cols), inv);
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      load8(x + c, a.align, a.cols - c, v);
      for (int i = 0; i < 8; ++i) {
        if (c + i < a.cols) sq[0] += (v[i] - mean) * (v[i] - mean);
      }
    }
    row_sum<1024>(sq, red, phase, 0);
    const float rstd = rsqrtf(sq[0] * inv + a.eps);
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      float w[8], b[8];
      load8(x + c, a.align, a.cols - c, v);
      if (weight != nullptr) load8(weight + c, a.align_w, a.cols - c, w);
      if (bias != nullptr) load8(bias + c, a.align_w, a.cols - c, b);
      for (int i = 0; i < 8; ++i) {
        v[i] = (v[i] - mean) * rstd;
        if (weight != nullptr) v[i] *= w[i];
        if (bias != nullptr) v[i] += b[i];
      }
      store8(y + c, a.align, a.cols - c, v);
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
// One block per SM.  Its groups of G threads walk the rows, the next ones on
// their way to shared memory (RowRing) and their statistics to registers, and
// keep their columns' dw and db sums in registers; a row is read twice from
// its slot (sums, then dx).  The weight waits as floats in shared memory.  At
// the end the groups' sums are added in order in shared memory, so a block
// leaves one partial row: part[block][2][part_cols].  (16384 x 8192: 243 us
// with rows requested into registers and unpaired arithmetic; two rows per
// join with half the columns per thread spills and is slower on most widths.)
constexpr int kRowThreads = 512;
template <int G>
constexpr int kBackwardStages = G < 512 ? 3 : 2;

template <typename T, int G, int V, bool VEC>
__global__ void __launch_bounds__(kRowThreads, 1) norm_backward_kernel(const NormBackwardArgs a) {
  constexpr int kGroups = kRowThreads / G;
  constexpr int kStages = kBackwardStages<G>;
  __shared__ float red[kGroups * 2 * (G / 32) * 2];
  __shared__ alignas(8) uint64_t bars[kGroups * kStages];
  extern __shared__ __align__(128) uint8_t dyn_smem[];  // weight, rings; at the end: float [groups][2][part_cols]
  int phase = 0;
  const int group = threadIdx.x / G;
  const Columns<G, VEC> mine;
  const bool leads = threadIdx.x % G == 0;
  const int cols = a.cols;
  float* weight = reinterpret_cast<float*>(dyn_smem);
  const float inv = 1.0f / static_cast<float>(cols);
  float* my_red = red + group * 2 * (G / 32) * 2;
  if (VEC && threadIdx.x < kGroups * kStages) ptx::mbar_init(ptx::smem_addr(&bars[threadIdx.x]), 1);
  ptx::fence_mbar_init();
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  Two dw[V][4] = {}, db[V][4] = {};
  const long long step = static_cast<long long>(gridDim.x) * kGroups;
  long long r = static_cast<long long>(blockIdx.x) * kGroups + group;
  RowRing<2, kStages> ring;
  ring.row_bytes = static_cast<uint32_t>(cols) * 2u;
  ring.slots = ptx::smem_addr(weight + a.part_cols) + group * kStages * 2 * ring.row_bytes;
  ring.bars = ptx::smem_addr(&bars[group * kStages]);
  ring.err = a.err;
  ring.policy = ptx::policy_evict_first();
  auto start = [&](long long row) { ring.start({x + row * a.ld_x, dy + row * a.ld_dy}); };
  if (VEC && leads) {
    for (int i = 0; i < kStages && r + i * step < a.rows; ++i) start(r + i * step);
  }
  float next_mean = 0.0f, next_rstd = 0.0f;
  if (r < a.rows) {
    next_mean = a.mean[r];
    next_rstd = a.rstd[r];
  }
  {
    const T* from = static_cast<const T*>(a.weight);
    for (int c = threadIdx.x * 8; c < cols; c += kRowThreads * 8) {
      float f[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
      if (from != nullptr) load8(from + c, a.align_w, cols - c, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) weight[c + i] = f[i];  // part_cols is a multiple of 8
    }
  }
  __syncthreads();
  for (; r < a.rows; r += step) {
    const float rstd = next_rstd;
    const float mean = next_mean;
    if (r + step < a.rows) {
      next_mean = a.mean[r + step];
      next_rstd = a.rstd[r + step];
    }
    [[maybe_unused]] const uint32_t slot = VEC ? ring.wait() : 0u;
    [[maybe_unused]] uint4 x_raw[VEC ? 1 : V], dy_raw[VEC ? 1 : V];
    if constexpr (!VEC) {
      load_pairs(x + r * a.ld_x, mine, cols, x_raw);
      load_pairs(dy + r * a.ld_dy, mine, cols, dy_raw);
    }
    // x and dy of vector j (0 past the row's end).
    auto at = [&](int j, Two(&xv)[4], Two(&gv)[4]) {
      if constexpr (VEC) {
        const int c = mine.column(j, 0);
        unpack<T>(ld_smem_v4(slot + 2 * c), xv);
        unpack<T>(ld_smem_v4(slot + ring.row_bytes + 2 * c), gv);
      } else {
        unpack<T>(x_raw[j], xv);
        unpack<T>(dy_raw[j], gv);
      }
    };
    auto weights = [&](int j, Two(&w)[4]) {
      if constexpr (VEC) {
        const ulonglong2* p = reinterpret_cast<const ulonglong2*>(weight + mine.column(j, 0));
        const ulonglong2 lo = p[0], hi = p[1];
        w[0] = lo.x, w[1] = lo.y, w[2] = hi.x, w[3] = hi.y;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = mine.column(j, i);
          w[i] = c < cols ? *reinterpret_cast<const Two*>(weight + c) : 0;  // (part_cols is even)
        }
      }
    };
    // (x - mean is formed first: x rstd - mean rstd cancels in rows far off centre)
    const Two rstd2 = two(rstd, rstd), minus_mean = two(-mean, -mean);
    Two s0 = 0, s1 = 0;  // sums of dy w xhat and of dy w
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (VEC && mine.column(j, 0) >= cols) continue;
      Two xv[4], g[4], w[4];
      at(j, xv, g);
      weights(j, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Two t = mul2(g[i], mul2(add2(xv[i], minus_mean), rstd2));
        dw[j][i] = add2(dw[j][i], t);
        db[j][i] = add2(db[j][i], g[i]);
        s0 = fma2(t, w[i], s0);
        s1 = fma2(g[i], w[i], s1);
      }
    }
    float sum[2] = {halves(s0).x + halves(s0).y, halves(s1).x + halves(s1).y};
    row_sum<G>(sum, my_red, phase, group);
    // Past this join the whole group is done with the row before this one:
    // its slot takes the row kStages - 1 ahead.
    if (VEC && leads && ring.use > 1 && r + (kStages - 1) * step < a.rows) start(r + (kStages - 1) * step);
    // dx = (rstd w) dy - rstd^2 mean(g xhat) (x - mean) - rstd mean(g)
    const float k1 = -rstd * (sum[0] * inv), k2 = -rstd * (sum[1] * inv);
    const Two slope = two(k1 * rstd, k1 * rstd), level = two(k2, k2);
    T* dx = static_cast<T*>(a.dx) + r * a.ld_dx;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (VEC && mine.column(j, 0) >= cols) continue;
      Two xv[4], g[4], w[4];
      at(j, xv, g);
      weights(j, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = fma2(g[i], mul2(w[i], rstd2), fma2(add2(xv[i], minus_mean), slope, level));
      const uint4 raw = pack<T>(g);
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(dx + mine.column(j, 0)) = raw;
      } else {
        store_pairs(dx, mine, cols, j, raw);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + static_cast<long long>(blockIdx.x) * 2 * a.part_cols;
  // One group writes its sums; several leave them side by side in shared
  // memory (over their drained rings), added per column in group order.
  float* joined = reinterpret_cast<float*>(dyn_smem);
  if (kGroups > 1) __syncthreads();
  float* to = kGroups > 1 ? joined + static_cast<size_t>(group) * 2 * a.part_cols : part;
#pragma unroll
  for (int j = 0; j < V; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // part_cols is a multiple of 8
      const int c = mine.column(j, i);
      if (c >= a.part_cols) continue;
      *reinterpret_cast<Two*>(to + c) = dw[j][i];
      *reinterpret_cast<Two*>(to + a.part_cols + c) = db[j][i];
    }
  }
  if (kGroups > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.part_cols; c += kRowThreads) {
      float t = joined[c];
#pragma unroll
      for (int g = 1; g < kGroups; ++g) t += joined[static_cast<size_t>(g) * 2 * a.part_cols + c];
      part[c] = t;
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
      load8(x + c, a.align, a.cols - c, xv);
      load8(dy + c, a.align, a.cols - c, g);
      if (weight != nullptr) load8(weight + c, a.align_w, a.cols - c, w);
      for (int i = 0; i < 8; ++i) {
        const float gw = weight != nullptr ? g[i] * w[i] : g[i];
        sum[0] += gw * (xv[i] - mean) * rstd;
        sum[1] += gw;
      }
    }
    row_sum<1024>(sum, red, phase, 0);
    const float c1 = sum[0] * inv, c2 = sum[1] * inv;
    for (int c = threadIdx.x * 8; c < a.cols; c += 1024 * 8) {
      load8(x + c, a.align, a.cols - c, xv);
      load8(dy + c, a.align, a.cols - c, g);
      if (weight != nullptr) load8(weight + c, a.align_w, a.cols - c, w);
      for (int i = 0; i < 8; ++i) {
        const float gw = weight != nullptr ? g[i] * w[i] : g[i];
        g[i] = (gw - c2 - (xv[i] - mean) * rstd * c1) * rstd;
      }
      store8(dx + c, a.align, a.cols - c, g);
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
    load8(static_cast<const T*>(a.x) + r * a.ld_x + c, a.align, a.cols - c, xv);
    load8(static_cast<const T*>(a.dy) + r * a.ld_dy + c, a.align, a.cols - c, g);
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
// out[c] = sum over p of part[p][c], in order of p inside each of 16 strided
// ranges, then the 16 in order.  32 columns x 16 ranges per block; a range's
// loads are requested eight at a time (bound by their latency).
constexpr int kSumRanges = 16;

template <typename T>
__global__ void __launch_bounds__(32 * kSumRanges) column_sum_kernel(const ColumnSumArgs a) {
  __shared__ float sums[kSumRanges][33];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int which = blockIdx.y;  // sums side by side in a partial row
  float s = 0.0f;
  if (c < a.cols) {
    const float* p = a.part + static_cast<long long>(which) * a.part_cols + c;
    const long long step = static_cast<long long>(a.sums) * a.part_cols;
#pragma unroll 8
    for (int i = q; i < a.parts; i += kSumRanges) s += p[i * step];
  }
  sums[q][lane] = s;
  __syncthreads();
  T* out = static_cast<T*>(which == 0 ? a.out[0] : a.out[1]);
  if (q == 0 && c < a.cols && out != nullptr) {
    float t = sums[0][lane];
#pragma unroll
    for (int i = 1; i < kSumRanges; ++i) t += sums[i][lane];
    out[c] = Elem16<T>::from_f(t);
  }
}

// ---------------------------------------------------------------- activations
//
// Linear: dz = dy act'(z).  Gated: dg = dy u act'(g), du = dy act(g).  One
// block: 512 columns (8 per thread) x a strip of rows, four rows at a time;
// each thread has its next two rows requested while it works on one (4096 x
// 11008 gated: 141 us row by row, since stores to dz keep the compiler from
// moving loads up; 97 us in pairs of rows that were waited for).  SUMS: the
// bias gradients' sums of the strip (of the values before their rounding) stay
// in registers and are added over the four row threads in order at the end.
// The rounding of dz to 16 bits is what the tensor-core products that follow
// read.
constexpr int kActCols = 64;  // column threads
constexpr int kActRows = 4;   // row threads

template <typename T, bool GATED, bool SUMS>
__global__ void __launch_bounds__(kActCols * kActRows, GATED && SUMS ? 2 : 3)
    act_backward_kernel(const ActBackwardArgs a) {
  constexpr int kSums = GATED ? 2 : 1;
  __shared__ float sums[SUMS ? kActRows - 1 : 1][kSums][kActCols * 8];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int tc = threadIdx.x % kActCols, tr = threadIdx.x / kActCols;
  const int c = (blockIdx.x * kActCols + tc) * 8;
  const bool live = c < a.cols;
  const long long lo = static_cast<long long>(blockIdx.y) * a.rows / gridDim.y + tr;
  const long long hi = live ? static_cast<long long>(blockIdx.y + 1) * a.rows / gridDim.y : 0;
  const int valid = a.cols - c;
  const T* dy = static_cast<const T*>(a.dy) + c;
  const T* pre0 = static_cast<const T*>(a.pre[0]) + c;
  const T* pre1 = static_cast<const T*>(a.pre[1]) + c;
  [[maybe_unused]] float s0[8] = {}, s1[8] = {};
  with_act(a.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    constexpr bool kReadsPre = GATED || ACT != GLQ_ACT_NONE;
    struct Row {
      uint4 g, z, u;
    };
    auto request = [&](long long row, Row& x) {
      if (row < hi) {
        x.g = load8_raw(dy + row * a.ld_dy, a.align_dy, valid);
        if (kReadsPre) x.z = load8_raw(pre0 + row * a.ld_pre, a.align_pre, valid);
        if (GATED) x.u = load8_raw(pre1 + row * a.ld_pre, a.align_pre, valid);
      }
    };
    auto work = [&](long long row, const Row& x) {
      const uint32_t gw[4] = {x.g.x, x.g.y, x.g.z, x.g.w};
      const uint32_t zw[4] = {x.z.x, x.z.y, x.z.z, x.z.w};
      const uint32_t uw[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
      uint32_t d0[4], d1[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // elements past the row's end are zeros: so are their products
        const float2 g = Elem16<T>::to_f2(gw[i]);
        float2 value = {0.0f, 0.0f}, slope = {1.0f, 1.0f};
        if (kReadsPre) {
          const float2 z = Elem16<T>::to_f2(zw[i]);
          act_grad_f<ACT>(z.x, &value.x, &slope.x);
          act_grad_f<ACT>(z.y, &value.y, &slope.y);
        }
        float2 p = {g.x * slope.x, g.y * slope.y};
        if (GATED) {
          const float2 u = Elem16<T>::to_f2(uw[i]);
          p = {p.x * u.x, p.y * u.y};
          const float2 q = {g.x * value.x, g.y * value.y};
          d1[i] = Elem16<T>::from_f2(q.x, q.y);
          if (SUMS) {
            s1[2 * i] += q.x;
            s1[2 * i + 1] += q.y;
          }
        }
        d0[i] = Elem16<T>::from_f2(p.x, p.y);
        if (SUMS) {
          s0[2 * i] += p.x;
          s0[2 * i + 1] += p.y;
        }
      }
      if (a.dz[0] != nullptr) {  // null: column sums only
        store8_raw(static_cast<T*>(a.dz[0]) + row * a.ld_dz + c, a.align_dz, valid,
                   make_uint4(d0[0], d0[1], d0[2], d0[3]));
        if (GATED) {
          store8_raw(static_cast<T*>(a.dz[1]) + row * a.ld_dz + c, a.align_dz, valid,
                     make_uint4(d1[0], d1[1], d1[2], d1[3]));
        }
      }
    };
    Row even, odd;
    request(lo, even);
    request(lo + kActRows, odd);
    for (long long r = lo; r < hi; r += 2 * kActRows) {
      const Row now = even;
      request(r + 2 * kActRows, even);
      work(r, now);
      if (r + kActRows < hi) {
        const Row then = odd;
        request(r + 3 * kActRows, odd);
        work(r + kActRows, then);
      }
    }
  });
  if constexpr (SUMS) {
    if (tr > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sums[tr - 1][0][tc * 8 + i] = s0[i];
        if (GATED) sums[tr - 1][kSums - 1][tc * 8 + i] = s1[i];
      }
    }
    __syncthreads();
    if (tr == 0 && live) {
      float* part = a.part + static_cast<long long>(blockIdx.y) * kSums * a.part_cols + c;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int q = 0; q < kActRows - 1; ++q) {
          s0[i] += sums[q][0][tc * 8 + i];
          if (GATED) s1[i] += sums[q][kSums - 1][tc * 8 + i];
        }
        part[i] = s0[i];
        if (GATED) part[a.part_cols + i] = s1[i];
      }
    }
  }
}

// ---------------------------------------------------------------- host

template <typename Kernel, typename Args>
cudaError_t launch(Kernel kernel, dim3 grid, int threads, size_t smem, const Args& args, unsigned int flags,
                   cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
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

int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }

// Largest of 16, 8, 4, 2 that every row's start is a multiple of.
int row_align(const void* p, int64_t ld) {
  const uintptr_t both = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * 2);
  return both % 16 == 0 ? 16 : both % 8 == 0 ? 8 : both % 4 == 0 ? 4 : 2;
}

// Threads per row and vectors per thread of the register kernels: four
// vectors, a warp at least.
int group_threads(int64_t cols) {
  return cols <= 1024 ? 32 : cols <= 2048 ? 64 : cols <= 4096 ? 128 : cols <= 8192 ? 256 : 512;
}

template <typename T, int G, int V>
cudaError_t launch_rows(const NormArgs& a, int grid, unsigned int flags, cudaStream_t s) {
  constexpr int kThreads = G < kNormThreads ? kNormThreads : G;
  return a.vec ? launch(norm_kernel<T, G, V, true>, dim3(grid), kThreads, 0, a, flags, s)
               : launch(norm_kernel<T, G, V, false>, dim3(grid), kThreads, 0, a, flags, s);
}

template <typename T>
cudaError_t norm_by_columns(const NormArgs& a, int grid, unsigned int flags, cudaStream_t s) {
  if (a.cols <= 256) return launch_rows<T, 32, 1>(a, grid, flags, s);
  if (a.cols <= 512) return launch_rows<T, 32, 2>(a, grid, flags, s);
  switch (group_threads(a.cols)) {
    case 32: return launch_rows<T, 32, 4>(a, grid, flags, s);
    case 64: return launch_rows<T, 64, 4>(a, grid, flags, s);
    case 128: return launch_rows<T, 128, 4>(a, grid, flags, s);
    case 256: return launch_rows<T, 256, 4>(a, grid, flags, s);
    default: return launch_rows<T, 512, 4>(a, grid, flags, s);
  }
}

template <typename T, int G, int V, bool VEC>
cudaError_t launch_rows_backward(const NormBackwardArgs& a, int grid, unsigned int flags, cudaStream_t s) {
  constexpr int kGroups = kRowThreads / G;
  // Weight and rings (at most 224 KB), then the groups' sums (at most 128 KB).
  const size_t one = static_cast<size_t>(a.part_cols) * sizeof(float);
  const size_t ring = VEC ? static_cast<size_t>(kGroups) * kBackwardStages<G> * 2 * a.cols * 2 : 0;
  const size_t smem = std::max(one + ring, kGroups > 1 ? kGroups * 2 * one : 0);
  return launch(norm_backward_kernel<T, G, V, VEC>, dim3(grid), kRowThreads, smem, a, flags, s);
}

template <typename T>
cudaError_t norm_backward_by_columns(const NormBackwardArgs& a, int grid, unsigned int flags, cudaStream_t s) {
  if (a.cols <= 256) return a.vec ? launch_rows_backward<T, 32, 1, true>(a, grid, flags, s)
                                : launch_rows_backward<T, 32, 1, false>(a, grid, flags, s);
  if (a.cols <= 512) return a.vec ? launch_rows_backward<T, 32, 2, true>(a, grid, flags, s)
                                : launch_rows_backward<T, 32, 2, false>(a, grid, flags, s);
  if (!a.vec) {  // a row waits in registers: half of it per thread where a block is enough
    switch (group_threads(a.cols)) {
      case 32: return launch_rows_backward<T, 64, 2, false>(a, grid, flags, s);
      case 64: return launch_rows_backward<T, 128, 2, false>(a, grid, flags, s);
      case 128: return launch_rows_backward<T, 256, 2, false>(a, grid, flags, s);
      case 256: return launch_rows_backward<T, 512, 2, false>(a, grid, flags, s);
      default: return launch_rows_backward<T, 512, 4, false>(a, grid, flags, s);
    }
  }
  switch (group_threads(a.cols)) {
    case 32: return launch_rows_backward<T, 32, 4, true>(a, grid, flags, s);
    case 64: return launch_rows_backward<T, 64, 4, true>(a, grid, flags, s);
    case 128: return launch_rows_backward<T, 128, 4, true>(a, grid, flags, s);
    case 256: return launch_rows_backward<T, 256, 4, true>(a, grid, flags, s);
    default: return launch_rows_backward<T, 512, 4, true>(a, grid, flags, s);
  }
}

// Blocks of the backward register kernel: one per SM, at most one per rows
// that a block takes at a time.
int64_t backward_blocks(int64_t rows, int64_t cols, int sm_count) {
  const int64_t at_a_time = kRowThreads / group_threads(cols);
  return std::min<int64_t>((rows + at_a_time - 1) / at_a_time, sm_count);
}

template <typename T, int G, int V, bool VEC>
cudaError_t set_attr() {
  return cudaFuncSetAttribute(norm_backward_kernel<T, G, V, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              VEC ? 229376 : 131072);
}

template <typename T>
cudaError_t set_attrs() {
  cudaError_t e = set_attr<T, 32, 1, true>();
  if (e == cudaSuccess) e = set_attr<T, 32, 2, true>();
  if (e == cudaSuccess) e = set_attr<T, 32, 4, true>();
  if (e == cudaSuccess) e = set_attr<T, 64, 4, true>();
  if (e == cudaSuccess) e = set_attr<T, 128, 4, true>();
  if (e == cudaSuccess) e = set_attr<T, 256, 4, true>();
  if (e == cudaSuccess) e = set_attr<T, 512, 4, true>();
  if (e == cudaSuccess) e = set_attr<T, 32, 1, false>();
  if (e == cudaSuccess) e = set_attr<T, 32, 2, false>();
  if (e == cudaSuccess) e = set_attr<T, 64, 2, false>();
  if (e == cudaSuccess) e = set_attr<T, 128, 2, false>();
  if (e == cudaSuccess) e = set_attr<T, 256, 2, false>();
  if (e == cudaSuccess) e = set_attr<T, 512, 2, false>();
  if (e == cudaSuccess) e = set_attr<T, 512, 4, false>();
  return e;
}

// Row strips of norm_columns_kernel: four blocks of 128 threads per SM.
int64_t strips(int64_t rows, int64_t cols, int sm_count) {
  const int64_t across = (cols + 1023) / 1024;
  return std::max<int64_t>(1, std::min<int64_t>(rows, std::min<int64_t>(4096, (int64_t{sm_count} * 4 + across - 1) / across)));
}

// Row strips of act_backward_kernel: one wave of blocks (three per SM, two
// with the gated sums) if whole strips fill most of it, else a few; at least
// the rows that a block's threads take in two steps each.
int64_t act_strips(int64_t rows, int64_t cols, int64_t sums, int sm_count) {
  const int64_t across = (cols + kActCols * 8 - 1) / (kActCols * 8);
  const int64_t wave = int64_t{sm_count} * (sums == 2 ? 2 : 3);
  int64_t n = wave / across;
  if (n * across * 5 < wave * 4) n = (4 * wave + across - 1) / across;
  const int64_t most = (rows + 2 * kActRows - 1) / (2 * kActRows);
  return std::max<int64_t>(1, std::min<int64_t>(most, std::min<int64_t>(4096, n)));
}

template <typename T>
cudaError_t norm_typed(const NormArgs& a, int sm_count, unsigned int flags, cudaStream_t s) {
  if (a.cols > kNormRegisterCols) {
    return launch(norm_long_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, 2 * sm_count))), 1024, 0, a,
                  flags, s);
  }
  // As many blocks as an SM holds: three of 256 threads, one of 512.
  const int g = group_threads(a.cols);
  const int64_t at_a_time = g < kNormThreads ? kNormThreads / g : 1;
  const int64_t blocks =
      std::min<int64_t>((a.rows + at_a_time - 1) / at_a_time, int64_t{sm_count} * (g < 512 ? 3 : 1));
  return norm_by_columns<T>(a, static_cast<int>(blocks), flags, s);
}

template <typename T>
cudaError_t norm_backward_typed(NormBackwardArgs a, void* dweight, void* dbias, int sm_count, unsigned int flags,
                                cudaStream_t s) {
  int64_t parts = 0;
  cudaError_t e;
  if (a.cols > kNormRegisterCols) {
    e = launch(norm_backward_long_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, 2 * sm_count))),
               1024, 0, a, flags, s);
    parts = strips(a.rows, a.cols, sm_count);
    if (e == cudaSuccess && a.part != nullptr) {
      e = launch(norm_columns_kernel<T>, dim3(static_cast<unsigned>((a.cols + 1023) / 1024), static_cast<unsigned>(parts)),
                 128, 0, a, flags, s);
    }
  } else {
    const int64_t grid = backward_blocks(a.rows, a.cols, sm_count);
    parts = grid;
    e = norm_backward_by_columns<T>(a, static_cast<int>(grid), flags, s);
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
  return launch(column_sum_kernel<T>, dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), 32 * kSumRanges, 0, c, flags, s);
}

template <typename T>
cudaError_t act_backward_typed(const ActBackwardArgs& a, bool gated, void* const* dbias, int64_t n_strips,
                               unsigned int flags, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.cols + kActCols * 8 - 1) / (kActCols * 8)), static_cast<unsigned>(n_strips));
  constexpr int kThreads = kActCols * kActRows;
  cudaError_t e;
  if (a.part != nullptr) {
    e = gated ? launch(act_backward_kernel<T, true, true>, grid, kThreads, 0, a, flags, s)
              : launch(act_backward_kernel<T, false, true>, grid, kThreads, 0, a, flags, s);
  } else {
    e = gated ? launch(act_backward_kernel<T, true, false>, grid, kThreads, 0, a, flags, s)
              : launch(act_backward_kernel<T, false, false>, grid, kThreads, 0, a, flags, s);
  }
  if (e != cudaSuccess || a.part == nullptr) return e;
  ColumnSumArgs c = {};
  c.part = a.part;
  c.part_cols = a.part_cols;
  c.parts = static_cast<int>(n_strips);
  c.sums = gated ? 2 : 1;
  c.cols = a.cols;
  c.out[0] = dbias[0];
  c.out[1] = gated ? dbias[1] : nullptr;
  return launch(column_sum_kernel<T>, dim3(static_cast<unsigned>((a.cols + 31) / 32), static_cast<unsigned>(c.sums)),
                32 * kSumRanges, 0, c, flags, s);
}

}  // namespace

cudaError_t rows_prepare_device() {
  const cudaError_t e = set_attrs<__half>();
  return e != cudaSuccess ? e : set_attrs<__nv_bfloat16>();
}

size_t norm_backward_partial_bytes(int64_t rows, int64_t cols, int sm_count) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t parts = cols > kNormRegisterCols
                            ? strips(rows, cols, sm_count)
                            : backward_blocks(rows, cols, sm_count);
  return static_cast<size_t>(parts * 2 * padded(cols)) * sizeof(float);
}

size_t act_backward_partial_bytes(int64_t rows, int64_t cols, int sums, int sm_count) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(act_strips(rows, cols, sums, sm_count) * sums * padded(cols)) * sizeof(float);
}

cudaError_t launch_norm(int dtype, NormArgs a, int sm_count, unsigned int flags, cudaStream_t s) {
  a.align = std::min(row_align(a.x, a.ld_x), row_align(a.y, a.ld_y));
  a.align_w = std::min(row_align(a.weight, 0), row_align(a.bias, 0));
  a.vec = a.align == 16 && a.align_w == 16 && a.cols % 8 == 0;
  return dtype == GLQ_DTYPE_BF16 ? norm_typed<__nv_bfloat16>(a, sm_count, flags, s)
                                 : norm_typed<__half>(a, sm_count, flags, s);
}

cudaError_t launch_norm_backward(int dtype, NormBackwardArgs a, void* dweight, void* dbias, int sm_count,
                                 unsigned int flags, cudaStream_t s) {
  a.align = std::min(row_align(a.x, a.ld_x), std::min(row_align(a.dy, a.ld_dy), row_align(a.dx, a.ld_dx)));
  a.align_w = row_align(a.weight, 0);
  a.vec = a.align == 16 && a.cols % 8 == 0;
  a.part_cols = padded(a.cols);
  return dtype == GLQ_DTYPE_BF16 ? norm_backward_typed<__nv_bfloat16>(a, dweight, dbias, sm_count, flags, s)
                                 : norm_backward_typed<__half>(a, dweight, dbias, sm_count, flags, s);
}

cudaError_t launch_act_backward(int dtype, bool gated, ActBackwardArgs a, void* const* dbias, int sm_count,
                                unsigned int flags, cudaStream_t s) {
  a.align_dy = row_align(a.dy, a.ld_dy);
  a.align_pre = std::min(row_align(a.pre[0], a.ld_pre), row_align(a.pre[1], a.ld_pre));
  a.align_dz = std::min(row_align(a.dz[0], a.ld_dz), row_align(a.dz[1], a.ld_dz));
  a.part_cols = padded(a.cols);
  const int64_t n = act_strips(a.rows, a.cols, a.part == nullptr ? 0 : gated ? 2 : 1, sm_count);
  return dtype == GLQ_DTYPE_BF16 ? act_backward_typed<__nv_bfloat16>(a, gated, dbias, n, flags, s)
                                 : act_backward_typed<__half>(a, gated, dbias, n, flags, s);
}

}  // namespace glq
