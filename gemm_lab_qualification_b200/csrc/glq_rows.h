// glq_rows.h -- launchers of the memory-bound kernels of glq_rows.cu.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace glq {

// Longest row the register-resident norm kernels hold.
constexpr int kNormRegisterCols = 16384;

// Tensors are [rows, cols] with unit column stride and row pitch ld_*
// (elements); the align and vec fields are set by the launchers.
struct NormArgs {
  const void* x;
  long long ld_x;
  const void* weight;  // [cols] or null
  const void* bias;    // [cols] or null
  void* y;
  long long ld_y;
  float* mean;  // [rows] or null (then rstd too)
  float* rstd;
  long long rows;
  int cols;
  float eps;
  int align, align_w;  // bytes that rows, weight and bias start at multiples of
  int vec;             // rows of whole 16-byte vectors
};

struct NormBackwardArgs {
  const void* dy;
  long long ld_dy;
  const void* x;
  long long ld_x;
  const void* weight;
  const float* mean;
  const float* rstd;
  void* dx;
  long long ld_dx;
  float* part;  // norm_backward_partial_bytes, or null: no dweight, no dbias
  long long part_cols;
  long long rows;
  int cols;
  unsigned int* err;
  int align, align_w, vec;
};

struct ColumnSumArgs {
  const float* part;  // [parts][sums][part_cols]
  long long part_cols;
  int parts, sums, cols;
  void* out[2];
};

struct ActBackwardArgs {
  const void* dy;
  long long ld_dy;
  const void* pre[2];  // z, or gate and up
  long long ld_pre;
  void* dz[2];  // dz, or dgate and dup; dz[0] null: column sums only
  long long ld_dz;
  float* part;  // act_backward_partial_bytes, or null: no bias gradients
  long long part_cols;
  long long rows;
  int cols;
  int act;
  int align_dy, align_pre, align_dz;
};

// Per-device one-time set-up (shared memory opt-in).
cudaError_t rows_prepare_device();

size_t norm_backward_partial_bytes(int64_t rows, int64_t cols, int sm_count);
size_t act_backward_partial_bytes(int64_t rows, int64_t cols, int sums, int sm_count);

// rows, cols >= 1.
cudaError_t launch_norm(int dtype, NormArgs a, int sm_count, unsigned int flags, cudaStream_t s);
cudaError_t launch_norm_backward(int dtype, NormBackwardArgs a, void* dweight, void* dbias, int sm_count,
                                 unsigned int flags, cudaStream_t s);
// Writes dz and, with a.part, the bias gradients dbias[0] (and dbias[1]).
cudaError_t launch_act_backward(int dtype, bool gated, ActBackwardArgs a, void* const* dbias, int sm_count,
                                unsigned int flags, cudaStream_t s);

}  // namespace glq
