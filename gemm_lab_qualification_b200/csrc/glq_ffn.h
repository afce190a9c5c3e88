// glq_ffn.h -- declarations shared by the feed-forward operators' kernels
// (glq_pair.cu, glq_skinny.cu, glq_token.cu, glq_rows.cu) and their C-ABI layer
// (glq_ffn_api.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/glq.h"

namespace glq {

// Set-up of the current device by glq_api.cu: a glq_status, the SM count and
// the sticky error word.
int current_device(int* sm_count, unsigned int** error_word);

// A matrix a TMA kernel reads: `rows` x `k` with k the contraction, element
// (r, c) at base + r * pitch + c when k-major, base + c * pitch + r when not.
// 16-byte aligned base and pitch.
struct Operand {
  const void* base = nullptr;
  int64_t pitch = 0;
  bool k_major = true;
};

// out[m, n] = epilogue(sum over parts p of A_p[m, :] . B_p[n, :]).
//
// kParts says what the second A / B / output stands for:
//   kOne      there is none;
//   kConcatK  a second contraction range: out = A_0 B_0^T + A_1 B_1^T;
//   kTwo      a second product of the same sizes, A_1 B_1^T into out[1];
//   kGated    a second B with the same A: out[0] = act(A B_0^T + bias[0]) *
//             (A B_1^T + bias[1]).
enum class Parts : int { kOne, kConcatK, kTwo, kGated };

struct Product {
  int dtype = 0;  // glq_dtype
  Parts parts = Parts::kOne;
  int64_t m = 0, n = 0, k = 0;
  Operand a[2], b[2];
  const void* bias[2] = {nullptr, nullptr};
  int act = GLQ_ACT_NONE;
  const void* residual = nullptr;
  int64_t ld_residual = 0;
  void* out[2] = {nullptr, nullptr};
  int64_t ld_out = 0;
  // Pre-activations, if kept: z, or gate and up.
  void* pre[2] = {nullptr, nullptr};
  int64_t ld_pre = 0;
  unsigned int flags = 0;  // glq_flags
};

// Largest token tile of the skinny kernel.
constexpr int kSkinnyTokens = 192;

// How a launch of the pair kernel is scheduled (see glq_pair.cu).
struct PairPlan {
  int pairs = 0;           // CTA pairs launched
  int split = 1;           // pairs per cluster that share a tile's K range
  int64_t whole = 0;       // tiles of the first product computed whole
  int runs = 0;            // pairs that the other tiles' K blocks are dealt to
  int64_t run_blocks = 0;  // those blocks
  size_t workspace_bytes = 0;
  double us = 0.0;         // estimate, after the launch
};
PairPlan plan_pair(const Product* products, int count, int sm_count);
bool share_launch(const Product* products, int sm_count);

// One launch of the pair kernel for one product (any m, k >= 1), or for two
// without epilogue of their own; workspace: plan_pair's bytes, 256-byte
// aligned.
cudaError_t launch_pair(const Product* products, int count, void* workspace, int sm_count, unsigned int* err,
                        cudaStream_t s);
// One call of the skinny kernel: k-major A, parts other than kTwo, k >= 0.
cudaError_t launch_skinny(const Product& p, int sm_count, unsigned int* err, cudaStream_t s);
// One call of the single-token kernel: m == 1, k >= 1, every operand k-major,
// parts kOne or kGated.
cudaError_t launch_token(const Product& p, int sm_count, cudaStream_t s);
cudaError_t pair_prepare_device();
cudaError_t skinny_prepare_device();

// Tensor map of a row-major matrix rows x cols (row pitch in elements of two
// bytes), boxes of box_rows x box_cols (64 columns with 128-byte swizzle, or 32
// with 64-byte swizzle), zero fill.
bool encode_tile_map(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t cols, int64_t pitch,
                     uint32_t box_rows, uint32_t box_cols = 64);

// The map of an operand with `rows` output rows and contraction `k`: boxes of
// box_rows rows x 64 K, or 64 rows x 64 K when MN-major.
bool operand_map(CUtensorMap* map, int dtype, const Operand& o, int64_t rows, int64_t k, uint32_t box_rows);

}  // namespace glq
