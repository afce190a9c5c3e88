// glq_ffn_api.cu -- the extern "C" boundary of the feed-forward operators
// (declared in include/glq.h): argument checks, operand preparation (aligned
// copies in the caller's workspace), the choice of kernel and the launches.
//
// Nothing here allocates device memory and no C++ exception crosses the
// boundary.  Each *_workspace_bytes function runs the same planning code as
// its operator, with an arena that only counts.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "glq_ffn.h"
#include "glq_internal.h"
#include "glq_rows.h"

namespace glq {
namespace {

constexpr int64_t kEsz = 2;

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool odd(const void* p) { return p != nullptr && !aligned(p, 2); }

// Workspace bytes handed out in 256-byte steps; base null: counting only.
struct Arena {
  unsigned char* base = nullptr;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base != nullptr ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

// A matrix as the caller has it: element (r, c) at ptr + r * rs + c * cs.
struct Matrix {
  const void* ptr;
  int64_t rows, cols, rs, cs;
};

struct Copy {
  Matrix from;
  void* to = nullptr;  // rows at sector_pitch(cols)
};

struct Copies {
  Copy list[3];
  int count = 0;
};

// Whether rows of m can be TMA rows as they are: unit column stride, 16-byte
// base and pitch, rows that do not overlap.
bool row_addressable(const Matrix& m) {
  return (m.cs == 1 || m.cols == 1) && aligned(m.ptr, 16) &&
         (m.rows == 1 || (m.rs > 0 && m.rs * kEsz % 16 == 0 && m.rs >= m.cols));
}

int64_t row_pitch(const Matrix& m) { return m.rows == 1 ? repack_pitch(m.cols) : m.rs; }

Matrix transposed(const Matrix& m) { return {m.ptr, m.cols, m.rows, m.cs, m.rs}; }

enum class Major { kAny, kK, kMn };

// Rows that begin at multiples of 16 bytes but not of 32 load at two thirds of
// the rate: the TMA splits their 32-byte sectors.  One such operand slows the
// pair kernel by an eighth, two by almost a half (512 tokens through 22528 x
// 7104: 122 us; pitch of A, of B, of both off by 16 bytes: 146, 134, 175; 2048
// tokens: 413, and 499, 481, 639), which a copy of the smaller one can be worth.
constexpr double kOffSector[3] = {1.0, 1.12, 1.45};
int64_t sector_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }

// The rows that operand() reads m by where it lies: those of m, or of its
// transpose, or none (it is copied, to whole sectors).
enum class Rows { kOwn, kTransposed, kCopied };
Rows rows_of(const Matrix& m, Major want) {
  if (want != Major::kMn && row_addressable(m)) return Rows::kOwn;
  return want != Major::kK && row_addressable(transposed(m)) ? Rows::kTransposed : Rows::kCopied;
}
bool off_sector(const Matrix& m, Major want) {
  const Rows rows = rows_of(m, want);
  if (rows == Rows::kCopied) return false;
  return !aligned(m.ptr, 32) || row_pitch(rows == Rows::kOwn ? m : transposed(m)) % 16 != 0;
}
// Estimated times in us: a launch and the bytes both ways at 5.5 TB/s; a
// product at 1.5 PFLOP/s.
double copy_us(const Matrix& m) { return 2.5 + static_cast<double>(m.rows * m.cols * 2 * kEsz) / 5.5e6; }
double product_us(int64_t m, int64_t n, int64_t k) {
  return 2.0 * static_cast<double>(m) * static_cast<double>(n) * static_cast<double>(k) / 1.5e9;
}

// Whether a copy is MN-major: in the order that reads m along its contiguous
// dimension if `want` leaves the choice.
bool copied_mn(const Matrix& m, Major want) {
  return want == Major::kMn || (want == Major::kAny && m.cs != 1 && m.rs == 1);
}

// m as an operand with m.cols the contraction; `copy`: one whose rows can be
// read as they are is copied all the same.
Operand operand(const Matrix& m, Major want, Arena* arena, Copies* copies, bool copy = false) {
  const Matrix t = transposed(m);
  const Rows rows = copy ? Rows::kCopied : rows_of(m, want);
  if (rows == Rows::kOwn) return {m.ptr, row_pitch(m), true};
  if (rows == Rows::kTransposed) return {m.ptr, row_pitch(t), false};
  const bool mn = copied_mn(m, want);
  const Matrix from = mn ? t : m;
  const int64_t pitch = sector_pitch(from.cols);
  void* to = arena->take(static_cast<size_t>(from.rows) * pitch * kEsz);
  copies->list[copies->count].from = from;
  copies->list[copies->count++].to = to;
  return {to, pitch, !mn};
}

cudaError_t run_copies(const Copies& c, int sm_count, cudaStream_t s) {
  for (int i = 0; i < c.count; ++i) {
    const Matrix& f = c.list[i].from;
    const cudaError_t e = launch_repack(f.ptr, f.rows, f.cols, f.rs, f.cs, c.list[i].to, sm_count, s, sector_pitch(f.cols));
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

int check_common(int dtype, int activation, int64_t m, int64_t n, int64_t k, unsigned int flags) {
  if (dtype != GLQ_DTYPE_F16 && dtype != GLQ_DTYPE_BF16) return GLQ_ERR_INVALID_ARGUMENT;
  if (activation < GLQ_ACT_NONE || activation >= GLQ_ACT_COUNT) return GLQ_ERR_INVALID_ARGUMENT;
  if ((flags & ~(GLQ_FLAG_NO_PDL | GLQ_FLAG_STATIC_WEIGHTS)) != 0) return GLQ_ERR_INVALID_ARGUMENT;
  if (m < 0 || n < 0 || k < 0) return GLQ_ERR_SHAPE;
  // The skinny kernel's grid: 64 output columns (rows) per block, 65535 blocks.
  constexpr int64_t kMax = 65535 * 64;
  if (m > kMax || n > kMax || k > kMax) return GLQ_ERR_SHAPE;
  return GLQ_OK;
}

// Strides of a matrix with unit column stride.
bool bad_pitch(const void* p, int64_t rows, int64_t cols, int64_t ld) { return p != nullptr && rows > 1 && ld < cols; }

int status_of(cudaError_t e) {
  if (e == cudaSuccess) return GLQ_OK;
  cudaGetLastError();
  return GLQ_ERR_CUDA;
}

int check_workspace(const Arena& need, const void* workspace, size_t bytes) {
  if (need.used == 0) return GLQ_OK;
  return workspace == nullptr || !aligned(workspace, 256) || bytes < need.used ? GLQ_ERR_WORKSPACE : GLQ_OK;
}

// The current device's SM count (148 without one: sizes can be asked anywhere).
int device_sms() {
  int sm_count = 0;
  unsigned int* err = nullptr;
  return current_device(&sm_count, &err) == GLQ_OK ? sm_count : 148;
}

// Few tokens (or no sums at all): the skinny kernel, which wants A k-major.
// Its 192-token tiles (one CTA per SM) serve products of one wave of them: 131
// tokens through 4096 x 4096 take 13.1 us there and 17.6 in the pair kernel,
// 192 through 28672 x 8192 (224 CTAs) 108.8 and 104.7.
bool is_skinny(const Product& p, int sm_count) {
  if (p.parts == Parts::kTwo) return false;
  if (p.k == 0) return true;
  if (!p.a[0].k_major) return false;
  const int64_t rows = p.parts == Parts::kGated ? 64 : 128;
  return p.m <= 128 || (p.m <= kSkinnyTokens && (p.n + rows - 1) / rows <= sm_count);
}

// One token, weights with K-contiguous rows: the single-token kernel.
bool is_token(const Product& p) {
  return p.m == 1 && p.k > 0 && (p.parts == Parts::kOne || p.parts == Parts::kGated) && p.a[0].k_major &&
         p.b[0].k_major && (p.parts == Parts::kOne || p.b[1].k_major);
}

size_t product_workspace(const Product& p, int sm_count) {
  return is_skinny(p, sm_count) ? 0 : plan_pair(&p, 1, sm_count).workspace_bytes;
}

// The pitch of a single row means nothing: one the TMA takes.
void settle_pitches(Product* p) {
  if (p->m == 1) p->ld_out = p->ld_pre = p->ld_residual = repack_pitch(p->n);
}

// One product by the kernel for its size.
cudaError_t run_product(Product p, void* workspace, int sm_count, unsigned int* err, cudaStream_t s) {
  settle_pitches(&p);
  if (is_token(p)) return launch_token(p, sm_count, s);
  return is_skinny(p, sm_count) ? launch_skinny(p, sm_count, err, s) : launch_pair(&p, 1, workspace, sm_count, err, s);
}

// rows x cols zeros.
cudaError_t zero_rows(void* p, int64_t rows, int64_t cols, int64_t ld, cudaStream_t s) {
  if (p == nullptr || rows <= 0 || cols <= 0) return cudaSuccess;
  const size_t width = static_cast<size_t>(cols) * kEsz;
  const size_t pitch = rows == 1 ? width : static_cast<size_t>(ld) * kEsz;
  return cudaMemset2DAsync(p, pitch, 0, width, static_cast<size_t>(rows), s);
}

// ---- forward

// A forward call's operands (A k-major, the weights in one order) and the
// product's workspace.
struct ForwardPlan {
  Copies copies;
  void* workspace = nullptr;
};

ForwardPlan plan_forward(Product* p, const Matrix& a, const Matrix& b0, const Matrix* b1, int sm_count,
                         Arena* arena) {
  ForwardPlan plan;
  bool copy_a = false, copy_b = false;
  p->a[0].k_major = true;
  if (!is_skinny(*p, sm_count)) {
    // (the second weight follows the first one's order)
    const Rows rows = rows_of(b0, Major::kAny);
    const bool mn = rows == Rows::kTransposed || (rows == Rows::kCopied && copied_mn(b0, Major::kAny));
    const Major want = mn ? Major::kMn : Major::kK;
    const bool off_a = off_sector(a, Major::kK);
    const bool off_b = off_sector(b0, Major::kAny) || (b1 != nullptr && off_sector(*b1, want));
    double copy_b_us = rows == Rows::kCopied ? 0.0 : copy_us(b0);
    if (b1 != nullptr && rows_of(*b1, want) != Rows::kCopied) copy_b_us += copy_us(*b1);
    const double us = product_us(p->m, (b1 != nullptr ? 2 : 1) * p->n, p->k);
    double best = us * kOffSector[off_a + off_b];
    for (int c = 1; c < 4; ++c) {
      const bool ca = (c & 1) != 0, cb = (c & 2) != 0;
      if ((ca && !off_a) || (cb && !off_b)) continue;
      const double t = us * kOffSector[(off_a && !ca) + (off_b && !cb)] + (ca ? copy_us(a) : 0.0) +
                       (cb ? copy_b_us : 0.0);
      if (t < best) best = t, copy_a = ca, copy_b = cb;
    }
  }
  p->a[0] = operand(a, Major::kK, arena, &plan.copies, copy_a);
  p->b[0] = operand(b0, Major::kAny, arena, &plan.copies, copy_b);
  if (b1 != nullptr) p->b[1] = operand(*b1, p->b[0].k_major ? Major::kK : Major::kMn, arena, &plan.copies, copy_b);
  plan.workspace = arena->take(product_workspace(*p, sm_count));
  return plan;
}

int run_forward(Product p, const Matrix& a, const Matrix& b0, const Matrix* b1, void* workspace, size_t bytes,
                cudaStream_t s) {
  int sm_count = device_sms();
  ForwardPlan plan;
  if (p.k > 0) {
    Arena arena;
    plan_forward(&p, a, b0, b1, sm_count, &arena);
    const int w = check_workspace(arena, workspace, bytes);
    if (w != GLQ_OK) return w;
    arena = Arena{static_cast<unsigned char*>(workspace), 0};
    plan = plan_forward(&p, a, b0, b1, sm_count, &arena);
  }
  unsigned int* err = nullptr;
  const int d = current_device(&sm_count, &err);
  if (d != GLQ_OK) return d;
  // A copied weight is written just before the product reads it.
  if (plan.copies.count > 0) p.flags &= ~static_cast<unsigned int>(GLQ_FLAG_STATIC_WEIGHTS);
  cudaError_t e = run_copies(plan.copies, sm_count, s);
  if (e == cudaSuccess) e = run_product(p, plan.workspace, sm_count, err, s);
  return status_of(e);
}

Matrix weight_rows(const void* b, int64_t ks, int64_t ns, int64_t n, int64_t k) { return {b, n, k, ns, ks}; }

// ---- backward

// What a backward call computes and from what; pairs are gate and up (gated)
// or have only their first entry.
struct Backward {
  int dtype;
  bool gated;
  int act;
  int64_t m, n, k;
  const void* dy;
  int64_t ld_dy;
  const void* pre[2];
  int64_t ld_pre;
  Matrix a;     // [m, k]
  Matrix b[2];  // [k, n]
  void* da;
  int64_t ld_da;
  void* db[2];
  int64_t db_ks, db_ns;
  void* dbias[2];
  bool want_da, want_db, want_dbias;  // what the workspace has to serve
};

// Whether dB is laid out as rows of B^T (a weight's gradient [n, k]) rather
// than rows of B.
bool gradient_nk(const Backward& q) { return q.db_ks == 1 && (q.n == 1 || q.db_ns >= q.k); }

struct BackwardPlan {
  bool make_dz;       // dz is written to the workspace (else it is dy)
  Operand dz[2];      // rows m, contraction n
  float* part = nullptr;
  Copies copies;
  Product products[2];  // the input's gradient, the weights' gradient
  int count = 0;
  bool together = false;  // one launch
  void* workspace = nullptr;
};

BackwardPlan plan_backward(const Backward& q, unsigned int flags, int sm_count, Arena* arena) {
  BackwardPlan p;
  const int pair = q.gated ? 2 : 1;
  const Matrix dy = {q.dy, q.m, q.n, q.ld_dy, 1};
  const bool products = q.k > 0 && (q.want_da || q.want_db);
  p.make_dz = products && (q.gated || q.act != GLQ_ACT_NONE || !row_addressable(dy));
  if (p.make_dz) {
    for (int i = 0; i < pair; ++i) {
      const int64_t pitch = sector_pitch(q.n);
      p.dz[i] = {arena->take(static_cast<size_t>(q.m) * pitch * kEsz), pitch, true};
    }
  } else {
    p.dz[0] = {q.dy, row_pitch(dy), true};
  }
  if (products && q.want_da) {
    Product& r = p.products[p.count++];
    r.parts = q.gated ? Parts::kConcatK : Parts::kOne;
    r.m = q.m;
    r.n = q.k;
    r.k = q.n;
    r.out[0] = q.da;
    r.ld_out = q.ld_da;
    r.b[0] = operand(q.b[0], Major::kAny, arena, &p.copies);
    if (q.gated) r.b[1] = operand(q.b[1], r.b[0].k_major ? Major::kK : Major::kMn, arena, &p.copies);
    for (int i = 0; i < pair; ++i) r.a[i] = p.dz[i];
  }
  if (products && q.want_db) {
    // dB^T [n, k] = dz^T A, or dB [k, n] = A^T dz: rows as the gradient lies.
    const bool nk = gradient_nk(q);
    const Operand a = operand(transposed(q.a), Major::kMn, arena, &p.copies);
    Product& r = p.products[p.count++];
    r.parts = q.gated ? Parts::kTwo : Parts::kOne;
    r.m = nk ? q.n : q.k;
    r.n = nk ? q.k : q.n;
    r.k = q.m;
    r.ld_out = nk ? q.db_ns : q.db_ks;
    for (int i = 0; i < pair; ++i) {
      const Operand dz = {p.dz[i].base, p.dz[i].pitch, false};
      r.a[i] = nk ? dz : a;
      r.b[i] = nk ? a : dz;
      r.out[i] = q.db[i];
    }
  }
  if (q.want_dbias) p.part = static_cast<float*>(arena->take(act_backward_partial_bytes(q.m, q.n, pair, sm_count)));
  for (int i = 0; i < p.count; ++i) {
    p.products[i].dtype = q.dtype;
    p.products[i].flags = flags;
    settle_pitches(&p.products[i]);
  }
  p.together = p.count == 2 && !is_skinny(p.products[0], sm_count) && share_launch(p.products, sm_count);
  // Launches follow one another, so they share it; a size that was asked for
  // both gradients serves a call for one.
  size_t bytes = p.together ? plan_pair(p.products, 2, sm_count).workspace_bytes : 0;
  for (int i = 0; i < p.count; ++i) bytes = std::max(bytes, product_workspace(p.products[i], sm_count));
  p.workspace = arena->take(bytes);
  return p;
}

int run_backward(const Backward& q, unsigned int flags, void* workspace, size_t bytes, cudaStream_t s) {
  const int pair = q.gated ? 2 : 1;
  int sm_count = 0;
  unsigned int* err = nullptr;
  const int d = current_device(&sm_count, &err);
  if (d != GLQ_OK) return d;
  if (q.m == 0 || q.n == 0) {
    // Empty sums: the gradients that have elements are zero.
    cudaError_t e = zero_rows(q.da, q.m, q.k, q.ld_da, s);
    for (int i = 0; i < pair && e == cudaSuccess; ++i) {
      if (q.db[i] != nullptr) {
        e = gradient_nk(q) ? zero_rows(q.db[i], q.n, q.k, q.db_ns, s) : zero_rows(q.db[i], q.k, q.n, q.db_ks, s);
      }
      if (e == cudaSuccess) e = zero_rows(q.dbias[i], 1, q.n, q.n, s);
    }
    return status_of(e);
  }
  flags &= ~static_cast<unsigned int>(GLQ_FLAG_STATIC_WEIGHTS);
  Arena arena;
  plan_backward(q, flags, sm_count, &arena);
  const int w = check_workspace(arena, workspace, bytes);
  if (w != GLQ_OK) return w;
  arena = Arena{static_cast<unsigned char*>(workspace), 0};
  const BackwardPlan p = plan_backward(q, flags, sm_count, &arena);

  cudaError_t e = cudaSuccess;
  if (p.make_dz || q.want_dbias) {
    ActBackwardArgs a = {};
    a.dy = q.dy;
    a.ld_dy = q.ld_dy;
    a.ld_pre = q.ld_pre;
    a.ld_dz = sector_pitch(q.n);
    a.rows = q.m;
    a.cols = static_cast<int>(q.n);
    a.act = q.act;
    a.part = q.want_dbias ? p.part : nullptr;
    for (int i = 0; i < pair; ++i) {
      a.pre[i] = q.pre[i];
      a.dz[i] = p.make_dz ? const_cast<void*>(p.dz[i].base) : nullptr;
    }
    e = launch_act_backward(q.dtype, q.gated, a, q.dbias, sm_count, flags, s);
  }
  if (e == cudaSuccess) e = run_copies(p.copies, sm_count, s);
  if (p.together) {
    if (e == cudaSuccess) e = launch_pair(p.products, 2, p.workspace, sm_count, err, s);
  } else {
    for (int i = 0; i < p.count && e == cudaSuccess; ++i) {
      e = run_product(p.products[i], p.workspace, sm_count, err, s);
    }
  }
  return status_of(e);
}

// Checks that both backward entry points share.
int check_backward(const Backward& q) {
  const int pair = q.gated ? 2 : 1;
  if (odd(q.dy) || odd(q.a.ptr) || odd(q.da)) return GLQ_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < pair; ++i) {
    if (odd(q.pre[i]) || odd(q.b[i].ptr) || odd(q.db[i]) || odd(q.dbias[i])) return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (q.want_db && q.n > 0 && q.k > 0) {
    const bool kn = q.db_ns == 1 && (q.k == 1 || q.db_ks >= q.n);
    if (!gradient_nk(q) && !kn) return GLQ_ERR_OUTPUT_LAYOUT;
  }
  if (bad_pitch(q.da, q.m, q.k, q.ld_da)) return GLQ_ERR_OUTPUT_LAYOUT;
  if (q.m == 0 || q.n == 0) return GLQ_OK;
  if (q.dy == nullptr) return GLQ_ERR_INVALID_ARGUMENT;
  const bool needs_pre = q.gated || q.act != GLQ_ACT_NONE;
  for (int i = 0; i < pair; ++i) {
    if (needs_pre && q.pre[i] == nullptr) return GLQ_ERR_INVALID_ARGUMENT;
    if (needs_pre && bad_pitch(q.pre[i], q.m, q.n, q.ld_pre)) return GLQ_ERR_SHAPE;
    if (q.k > 0 && q.want_da && q.b[i].ptr == nullptr) return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (q.k > 0 && q.want_db && q.a.ptr == nullptr) return GLQ_ERR_INVALID_ARGUMENT;
  if (bad_pitch(q.dy, q.m, q.n, q.ld_dy)) return GLQ_ERR_SHAPE;
  return GLQ_OK;
}

}  // namespace
}  // namespace glq

using glq::Matrix;
using glq::Parts;
using glq::Product;

extern "C" {

int glq_fused_linear(int dtype, const void* A, int64_t a_row_stride, int64_t a_col_stride, const void* B,
                     int64_t b_k_stride, int64_t b_n_stride, const void* bias, int activation, const void* residual,
                     int64_t residual_row_stride, void* Z, int64_t z_row_stride, void* Y, int64_t y_row_stride,
                     int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream,
                     unsigned int flags) {
  const int v = glq::check_common(dtype, activation, M, N, K, flags);
  if (v != GLQ_OK) return v;
  if (M == 0 || N == 0) return GLQ_OK;
  if (Y == nullptr || (K > 0 && (A == nullptr || B == nullptr))) return GLQ_ERR_INVALID_ARGUMENT;
  if (glq::odd(A) || glq::odd(B) || glq::odd(bias) || glq::odd(residual) || glq::odd(Z) || glq::odd(Y)) {
    return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (glq::bad_pitch(Y, M, N, y_row_stride) || glq::bad_pitch(Z, M, N, z_row_stride)) return GLQ_ERR_OUTPUT_LAYOUT;
  if (residual != nullptr && M > 1 && residual_row_stride < 0) return GLQ_ERR_SHAPE;
  Product p;
  p.dtype = dtype;
  p.m = M;
  p.n = N;
  p.k = K;
  p.bias[0] = bias;
  p.act = activation;
  p.residual = residual;
  p.ld_residual = residual_row_stride;
  p.out[0] = Y;
  p.ld_out = y_row_stride;
  p.pre[0] = Z;
  p.ld_pre = z_row_stride;
  p.flags = flags;
  return glq::run_forward(p, Matrix{A, M, K, a_row_stride, a_col_stride},
                          glq::weight_rows(B, b_k_stride, b_n_stride, N, K), nullptr, workspace, workspace_bytes,
                          static_cast<cudaStream_t>(stream));
}

size_t glq_fused_linear_workspace_bytes(int dtype, const void* A, int64_t a_row_stride, int64_t a_col_stride,
                                        const void* B, int64_t b_k_stride, int64_t b_n_stride, int64_t M, int64_t N,
                                        int64_t K) {
  if (glq::check_common(dtype, GLQ_ACT_NONE, M, N, K, 0) != GLQ_OK || M == 0 || N == 0 || K == 0) return 0;
  Product p;
  p.m = M;
  p.n = N;
  p.k = K;
  glq::Arena arena;
  glq::plan_forward(&p, Matrix{A, M, K, a_row_stride, a_col_stride},
                    glq::weight_rows(B, b_k_stride, b_n_stride, N, K), nullptr, glq::device_sms(), &arena);
  return arena.used;
}

int glq_gated_linear(int dtype, const void* A, int64_t a_row_stride, int64_t a_col_stride, const void* Bg,
                     int64_t bg_k_stride, int64_t bg_n_stride, const void* Bu, int64_t bu_k_stride,
                     int64_t bu_n_stride, const void* bias_g, const void* bias_u, int activation, void* G, void* U,
                     int64_t gu_row_stride, void* Y, int64_t y_row_stride, int64_t M, int64_t N, int64_t K,
                     void* workspace, size_t workspace_bytes, void* stream, unsigned int flags) {
  const int v = glq::check_common(dtype, activation, M, N, K, flags);
  if (v != GLQ_OK) return v;
  if ((G == nullptr) != (U == nullptr)) return GLQ_ERR_INVALID_ARGUMENT;
  if (M == 0 || N == 0) return GLQ_OK;
  if (Y == nullptr || (K > 0 && (A == nullptr || Bg == nullptr || Bu == nullptr))) return GLQ_ERR_INVALID_ARGUMENT;
  if (glq::odd(A) || glq::odd(Bg) || glq::odd(Bu) || glq::odd(bias_g) || glq::odd(bias_u) || glq::odd(G) ||
      glq::odd(U) || glq::odd(Y)) {
    return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (glq::bad_pitch(Y, M, N, y_row_stride) || glq::bad_pitch(G, M, N, gu_row_stride)) return GLQ_ERR_OUTPUT_LAYOUT;
  Product p;
  p.dtype = dtype;
  p.parts = Parts::kGated;
  p.m = M;
  p.n = N;
  p.k = K;
  p.bias[0] = bias_g;
  p.bias[1] = bias_u;
  p.act = activation;
  p.out[0] = Y;
  p.ld_out = y_row_stride;
  p.pre[0] = G;
  p.pre[1] = U;
  p.ld_pre = gu_row_stride;
  p.flags = flags;
  const Matrix up = glq::weight_rows(Bu, bu_k_stride, bu_n_stride, N, K);
  return glq::run_forward(p, Matrix{A, M, K, a_row_stride, a_col_stride},
                          glq::weight_rows(Bg, bg_k_stride, bg_n_stride, N, K), &up, workspace, workspace_bytes,
                          static_cast<cudaStream_t>(stream));
}

size_t glq_gated_linear_workspace_bytes(int dtype, const void* A, int64_t a_row_stride, int64_t a_col_stride,
                                        const void* Bg, int64_t bg_k_stride, int64_t bg_n_stride, const void* Bu,
                                        int64_t bu_k_stride, int64_t bu_n_stride, int64_t M, int64_t N, int64_t K) {
  if (glq::check_common(dtype, GLQ_ACT_NONE, M, N, K, 0) != GLQ_OK || M == 0 || N == 0 || K == 0) return 0;
  Product p;
  p.parts = Parts::kGated;
  p.m = M;
  p.n = N;
  p.k = K;
  glq::Arena arena;
  const Matrix up = glq::weight_rows(Bu, bu_k_stride, bu_n_stride, N, K);
  glq::plan_forward(&p, Matrix{A, M, K, a_row_stride, a_col_stride},
                    glq::weight_rows(Bg, bg_k_stride, bg_n_stride, N, K), &up, glq::device_sms(), &arena);
  return arena.used;
}

int glq_fused_linear_backward(int dtype, const void* dY, int64_t dy_row_stride, const void* Z, int64_t z_row_stride,
                              const void* A, int64_t a_row_stride, int64_t a_col_stride, const void* B,
                              int64_t b_k_stride, int64_t b_n_stride, int activation, void* dA, int64_t da_row_stride,
                              void* dB, int64_t db_k_stride, int64_t db_n_stride, void* dbias, int64_t M, int64_t N,
                              int64_t K, void* workspace, size_t workspace_bytes, void* stream, unsigned int flags) {
  int v = glq::check_common(dtype, activation, M, N, K, flags);
  if (v != GLQ_OK) return v;
  glq::Backward q = {};
  q.dtype = dtype;
  q.act = activation;
  q.m = M;
  q.n = N;
  q.k = K;
  q.dy = dY;
  q.ld_dy = dy_row_stride;
  q.pre[0] = activation == GLQ_ACT_NONE ? nullptr : Z;
  q.ld_pre = z_row_stride;
  q.a = Matrix{A, M, K, a_row_stride, a_col_stride};
  q.b[0] = Matrix{B, K, N, b_k_stride, b_n_stride};
  q.da = dA;
  q.ld_da = da_row_stride;
  q.db[0] = dB;
  q.db_ks = db_k_stride;
  q.db_ns = db_n_stride;
  q.dbias[0] = dbias;
  q.want_da = dA != nullptr;
  q.want_db = dB != nullptr;
  q.want_dbias = dbias != nullptr;
  v = glq::check_backward(q);
  return v != GLQ_OK ? v : glq::run_backward(q, flags, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t glq_fused_linear_backward_workspace_bytes(int dtype, const void* dY, int64_t dy_row_stride, const void* A,
                                                 int64_t a_row_stride, int64_t a_col_stride, const void* B,
                                                 int64_t b_k_stride, int64_t b_n_stride, int activation, int has_bias,
                                                 int64_t M, int64_t N, int64_t K) {
  if (glq::check_common(dtype, activation, M, N, K, 0) != GLQ_OK || M == 0 || N == 0) return 0;
  glq::Backward q = {};
  q.act = activation;
  q.m = M;
  q.n = N;
  q.k = K;
  q.dy = dY;
  q.ld_dy = dy_row_stride;
  q.a = Matrix{A, M, K, a_row_stride, a_col_stride};
  q.b[0] = Matrix{B, K, N, b_k_stride, b_n_stride};
  q.want_da = q.want_db = true;
  q.want_dbias = has_bias != 0;
  glq::Arena arena;
  glq::plan_backward(q, 0, glq::device_sms(), &arena);
  return arena.used;
}

int glq_gated_linear_backward(int dtype, const void* dY, int64_t dy_row_stride, const void* G, const void* U,
                              int64_t gu_row_stride, const void* A, int64_t a_row_stride, int64_t a_col_stride,
                              const void* Bg, int64_t bg_k_stride, int64_t bg_n_stride, const void* Bu,
                              int64_t bu_k_stride, int64_t bu_n_stride, int activation, void* dA,
                              int64_t da_row_stride, void* dBg, void* dBu, int64_t db_k_stride, int64_t db_n_stride,
                              void* dbias_g, void* dbias_u, int64_t M, int64_t N, int64_t K, void* workspace,
                              size_t workspace_bytes, void* stream, unsigned int flags) {
  int v = glq::check_common(dtype, activation, M, N, K, flags);
  if (v != GLQ_OK) return v;
  if ((dBg == nullptr) != (dBu == nullptr) || (dbias_g == nullptr) != (dbias_u == nullptr)) {
    return GLQ_ERR_INVALID_ARGUMENT;
  }
  glq::Backward q = {};
  q.dtype = dtype;
  q.gated = true;
  q.act = activation;
  q.m = M;
  q.n = N;
  q.k = K;
  q.dy = dY;
  q.ld_dy = dy_row_stride;
  q.pre[0] = G;
  q.pre[1] = U;
  q.ld_pre = gu_row_stride;
  q.a = Matrix{A, M, K, a_row_stride, a_col_stride};
  q.b[0] = Matrix{Bg, K, N, bg_k_stride, bg_n_stride};
  q.b[1] = Matrix{Bu, K, N, bu_k_stride, bu_n_stride};
  q.da = dA;
  q.ld_da = da_row_stride;
  q.db[0] = dBg;
  q.db[1] = dBu;
  q.db_ks = db_k_stride;
  q.db_ns = db_n_stride;
  q.dbias[0] = dbias_g;
  q.dbias[1] = dbias_u;
  q.want_da = dA != nullptr;
  q.want_db = dBg != nullptr;
  q.want_dbias = dbias_g != nullptr;
  v = glq::check_backward(q);
  return v != GLQ_OK ? v : glq::run_backward(q, flags, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t glq_gated_linear_backward_workspace_bytes(int dtype, const void* A, int64_t a_row_stride,
                                                 int64_t a_col_stride, const void* Bg, int64_t bg_k_stride,
                                                 int64_t bg_n_stride, const void* Bu, int64_t bu_k_stride,
                                                 int64_t bu_n_stride, int has_bias, int64_t M, int64_t N, int64_t K) {
  if (glq::check_common(dtype, GLQ_ACT_NONE, M, N, K, 0) != GLQ_OK || M == 0 || N == 0) return 0;
  glq::Backward q = {};
  q.gated = true;
  q.m = M;
  q.n = N;
  q.k = K;
  q.a = Matrix{A, M, K, a_row_stride, a_col_stride};
  q.b[0] = Matrix{Bg, K, N, bg_k_stride, bg_n_stride};
  q.b[1] = Matrix{Bu, K, N, bu_k_stride, bu_n_stride};
  q.want_da = q.want_db = true;
  q.want_dbias = has_bias != 0;
  glq::Arena arena;
  glq::plan_backward(q, 0, glq::device_sms(), &arena);
  return arena.used;
}

int glq_layer_norm(int dtype, const void* X, int64_t x_row_stride, const void* weight, const void* bias, double eps,
                   void* Y, int64_t y_row_stride, float* mean, float* rstd, int64_t M, int64_t N, void* stream,
                   unsigned int flags) {
  const int v = glq::check_common(dtype, GLQ_ACT_NONE, 0, N, 0, flags);
  if (v != GLQ_OK) return v;
  if (M < 0 || M > INT_MAX) return GLQ_ERR_SHAPE;
  if (!(eps >= 0.0) || (mean == nullptr) != (rstd == nullptr)) return GLQ_ERR_INVALID_ARGUMENT;
  if (M == 0 || (N == 0 && mean == nullptr)) return GLQ_OK;
  if (N > 0 && (X == nullptr || Y == nullptr)) return GLQ_ERR_INVALID_ARGUMENT;
  if (glq::odd(X) || glq::odd(Y) || glq::odd(weight) || glq::odd(bias) || !glq::aligned(mean, 4) ||
      !glq::aligned(rstd, 4)) {
    return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (M > 1 && x_row_stride < 0) return GLQ_ERR_SHAPE;
  if (glq::bad_pitch(Y, M, N, y_row_stride)) return GLQ_ERR_OUTPUT_LAYOUT;
  int sm_count = 0;
  unsigned int* err = nullptr;
  const int d = glq::current_device(&sm_count, &err);
  if (d != GLQ_OK) return d;
  if (N == 0) {
    // Statistics of no values, 0 / 0: all bits set are a NaN.
    const size_t bytes = static_cast<size_t>(M) * sizeof(float);
    cudaError_t e = cudaMemsetAsync(mean, 0xff, bytes, static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) e = cudaMemsetAsync(rstd, 0xff, bytes, static_cast<cudaStream_t>(stream));
    return glq::status_of(e);
  }
  glq::NormArgs a = {};
  a.x = X;
  a.ld_x = x_row_stride;
  a.weight = weight;
  a.bias = bias;
  a.y = Y;
  a.ld_y = y_row_stride;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = M;
  a.cols = static_cast<int>(N);
  a.eps = static_cast<float>(eps);
  return glq::status_of(glq::launch_norm(dtype, a, sm_count, flags, static_cast<cudaStream_t>(stream)));
}

int glq_layer_norm_backward(int dtype, const void* dY, int64_t dy_row_stride, const void* X, int64_t x_row_stride,
                            const void* weight, const float* mean, const float* rstd, void* dX, int64_t dx_row_stride,
                            void* dweight, void* dbias, int64_t M, int64_t N, void* workspace, size_t workspace_bytes,
                            void* stream, unsigned int flags) {
  const int v = glq::check_common(dtype, GLQ_ACT_NONE, 0, N, 0, flags);
  if (v != GLQ_OK) return v;
  if (M < 0 || M > INT_MAX) return GLQ_ERR_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (glq::odd(dY) || glq::odd(X) || glq::odd(weight) || glq::odd(dX) || glq::odd(dweight) || glq::odd(dbias) ||
      !glq::aligned(mean, 4) || !glq::aligned(rstd, 4)) {
    return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (N == 0) return GLQ_OK;
  int sm_count = 0;
  unsigned int* err = nullptr;
  if (M == 0) {
    const int d = glq::current_device(&sm_count, &err);
    if (d != GLQ_OK) return d;
    cudaError_t e = glq::zero_rows(dweight, 1, N, N, s);
    if (e == cudaSuccess) e = glq::zero_rows(dbias, 1, N, N, s);
    return glq::status_of(e);
  }
  if (dY == nullptr || X == nullptr || mean == nullptr || rstd == nullptr || dX == nullptr) {
    return GLQ_ERR_INVALID_ARGUMENT;
  }
  if (M > 1 && (x_row_stride < 0 || dy_row_stride < 0)) return GLQ_ERR_SHAPE;
  if (glq::bad_pitch(dX, M, N, dx_row_stride)) return GLQ_ERR_OUTPUT_LAYOUT;
  const int d = glq::current_device(&sm_count, &err);
  if (d != GLQ_OK) return d;
  glq::NormBackwardArgs a = {};
  if (dweight != nullptr || dbias != nullptr) {
    glq::Arena need;
    need.take(glq::norm_backward_partial_bytes(M, N, sm_count));
    const int w = glq::check_workspace(need, workspace, workspace_bytes);
    if (w != GLQ_OK) return w;
    a.part = static_cast<float*>(workspace);
  }
  a.dy = dY;
  a.ld_dy = dy_row_stride;
  a.x = X;
  a.ld_x = x_row_stride;
  a.weight = weight;
  a.mean = mean;
  a.rstd = rstd;
  a.dx = dX;
  a.ld_dx = dx_row_stride;
  a.rows = M;
  a.cols = static_cast<int>(N);
  a.err = err;
  return glq::status_of(glq::launch_norm_backward(dtype, a, dweight, dbias, sm_count, flags, s));
}

size_t glq_layer_norm_backward_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || N > INT_MAX) return 0;
  glq::Arena arena;
  arena.take(glq::norm_backward_partial_bytes(M, N, glq::device_sms()));
  return arena.used;
}

}  // extern "C"
