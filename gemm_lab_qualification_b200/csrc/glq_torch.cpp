// glq_torch.cpp -- the operator API's call path into libglq.so, in C++.
//
// The Python operators of kernels.py (triton_matmul_into, triton_bias_silu_into,
// triton_splitk_matmul_into and the Plans) check their arguments and call
// glq_linear_ex.  Doing both through Python attribute access and ctypes cost
// ~15 us per call on the host, more than the kernel itself, so a dependent
// chain of calls was host-bound.  This module does the same checks (same
// ValueError texts as kernels.py:132-145, 150-153, 259-262, 403-409, minus the
// contiguity rule) and the launch in one native call on torch's current
// stream.  Library failures come back as the glq_status so that Python raises
// the same GlqError as the ctypes binding.
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/extension.h>

#include <sstream>
#include <string>
#include <tuple>
#include <vector>

#include <pybind11/stl.h>

#include "glq.h"

namespace {

std::string shape_str(const at::Tensor& t) {
  std::ostringstream s;
  s << '(';
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  if (t.dim() == 1) s << ',';
  s << ')';
  return s.str();
}

void check_inputs(const at::Tensor& a, const at::Tensor& b, const std::string& op) {
  if (a.dim() != 2 || b.dim() != 2) throw py::value_error(op + " expects two rank-2 tensors");
  if (a.size(1) != b.size(0)) {
    throw py::value_error("incompatible dimensions: " + shape_str(a) + " and " + shape_str(b));
  }
  if (!a.is_cuda() || !b.is_cuda()) throw py::value_error(op + " requires CUDA tensors");
  if (a.device() != b.device()) throw py::value_error("input tensors must be on the same CUDA device");
  if (a.scalar_type() != b.scalar_type() ||
      (a.scalar_type() != at::kHalf && a.scalar_type() != at::kBFloat16)) {
    throw py::value_error("inputs must share dtype float16 or bfloat16");
  }
}

void check_output(const at::Tensor& out, const at::Tensor& a, int64_t m, int64_t n) {
  if (out.dim() != 2 || out.size(0) != m || out.size(1) != n || out.device() != a.device() ||
      out.scalar_type() != a.scalar_type()) {
    throw py::value_error("output tensor has the wrong shape, device, or dtype");
  }
  if (m && n && ((n > 1 && out.stride(1) != 1) || (m > 1 && out.stride(0) < n))) {
    throw py::value_error("output tensor must be contiguous");
  }
}

void check_bias(const at::Tensor& bias, const at::Tensor& a, int64_t n) {
  if (bias.dim() != 1 || bias.size(0) != n || bias.device() != a.device() || bias.scalar_type() != a.scalar_type()) {
    throw py::value_error("bias tensor has the wrong shape, device, or dtype");
  }
  if (n > 1 && bias.stride(0) != 1) throw py::value_error("bias tensor must be contiguous");
}

// What the kernels write through a raw pointer: autograd compares the version
// of a tensor it saved with the present one (inference tensors have none).
void wrote(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Returns (glq_status, path, split).  `op` names the operator in messages.
std::tuple<int, int, int> linear(const std::string& op, const at::Tensor& a, const at::Tensor& b, at::Tensor& out,
                                 const c10::optional<at::Tensor>& bias, int epilogue, int split_k,
                                 const c10::optional<at::Tensor>& partial, int64_t flags) {
  check_inputs(a, b, op);
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  if (bias.has_value()) check_bias(*bias, a, n);
  check_output(out, a, m, n);
  const int dtype = a.scalar_type() == at::kHalf ? GLQ_DTYPE_F16 : GLQ_DTYPE_BF16;
  void* ws = nullptr;
  size_t ws_bytes = 0;
  at::Tensor repack_ws;
  if (partial.has_value()) {
    ws = partial->data_ptr();
    ws_bytes = static_cast<size_t>(partial->numel()) * partial->element_size();
  } else if (m && n && k) {
    // Strided or unaligned operands: aligned copies in a workspace from
    // torch's caching allocator (stream-ordered, so it may be released as
    // soon as the launches are queued), then the tcgen05 / GEMV kernel.
    const size_t need = glq_linear_workspace_bytes(dtype, a.data_ptr(), a.stride(0), a.stride(1), b.data_ptr(),
                                                   b.stride(0), b.stride(1), m, n, k);
    if (need) {
      repack_ws = at::empty({static_cast<int64_t>(need)}, a.options().dtype(at::kByte));
      ws = repack_ws.data_ptr();
      ws_bytes = need;
    }
  }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(a.device().index()).stream();
  int path = -1, split = 0;
  const int status = glq_linear_ex(dtype, a.data_ptr(),
                                   a.stride(0), a.stride(1), b.data_ptr(), b.stride(0), b.stride(1),
                                   bias.has_value() ? bias->data_ptr() : nullptr, epilogue, out.data_ptr(),
                                   out.stride(0), m, n, k, split_k, ws, ws_bytes, stream,
                                   static_cast<unsigned int>(flags), &path, &split);
  wrote(out);
  return {status, path, split};
}

// The fused-gather launch of the column-parallel layer (glq_linear_gather):
// per-rank output and signal-slot pointers as integers (peer mappings from
// torch symmetric memory).  Returns (glq_status, path, split).
std::tuple<int, int, int> linear_gather(const at::Tensor& a, const at::Tensor& b, const c10::optional<at::Tensor>& bias,
                                        int epilogue, const std::vector<int64_t>& y_ptrs, int64_t y_row_stride,
                                        int64_t y_col_offset, int rank, const std::vector<int64_t>& signal_ptrs,
                                        int64_t counter, int64_t epoch, int split_k, int64_t flags) {
  check_inputs(a, b, "linear_gather");
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  if (bias.has_value()) check_bias(*bias, a, n);
  if (y_ptrs.size() != signal_ptrs.size() || y_ptrs.empty() || y_ptrs.size() > GLQ_MAX_RANKS) {
    throw py::value_error("one output and one signal pointer per rank, at most GLQ_MAX_RANKS ranks");
  }
  void* ys[GLQ_MAX_RANKS];
  uint64_t* sigs[GLQ_MAX_RANKS];
  for (size_t r = 0; r < y_ptrs.size(); ++r) {
    ys[r] = reinterpret_cast<void*>(y_ptrs[r]);
    sigs[r] = reinterpret_cast<uint64_t*>(signal_ptrs[r]);
  }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(a.device().index()).stream();
  int path = -1, split = 0;
  const int status = glq_linear_gather(
      a.scalar_type() == at::kHalf ? GLQ_DTYPE_F16 : GLQ_DTYPE_BF16, a.data_ptr(), a.stride(0), a.stride(1),
      b.data_ptr(), b.stride(0), b.stride(1), bias.has_value() ? bias->data_ptr() : nullptr, epilogue, ys,
      y_row_stride, y_col_offset, m, n, k, split_k, rank, static_cast<int>(y_ptrs.size()), sigs,
      reinterpret_cast<unsigned int*>(counter), static_cast<uint64_t>(epoch), stream,
      static_cast<unsigned int>(flags), &path, &split);
  return {status, path, split};
}

// ---------------------------------------------------------------- feed-forward operators
//
// Each allocates its outputs and workspace from torch's caching allocator on
// the current stream of the operands' device (made current for the call) and
// returns (glq_status, outputs...).

using OptTensor = c10::optional<at::Tensor>;

int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? GLQ_DTYPE_F16 : GLQ_DTYPE_BF16; }

cudaStream_t stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// The operators have no forward-mode derivative: an output without a tangent
// would stand for a derivative of zero.
bool dual(const at::Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool dual(const OptTensor& t) { return t.has_value() && dual(*t); }

template <typename... Tensors>
void check_no_tangent(const char* op, const Tensors&... tensors) {
  // (outside of every dual level there are none; asking each tensor costs views 0.1 us)
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr) return;
  if ((dual(tensors) || ...) && c10::AutogradState::get_tls_state().get_fw_grad_mode()) {
    throw py::value_error(std::string(op) + " has no forward-mode derivative");
  }
}

void check_vector(const OptTensor& v, const at::Tensor& a, int64_t n, const char* name) {
  if (!v.has_value()) return;
  if (v->dim() != 1 || v->size(0) != n || v->device() != a.device() || v->scalar_type() != a.scalar_type()) {
    throw py::value_error(std::string(name) + " tensor has the wrong shape, device, or dtype");
  }
  if (n > 1 && v->stride(0) != 1) throw py::value_error(std::string(name) + " tensor must be contiguous");
}

void check_matrix(const at::Tensor& t, const at::Tensor& a, int64_t m, int64_t n, const char* name) {
  if (t.dim() != 2 || t.size(0) != m || t.size(1) != n || t.device() != a.device() ||
      t.scalar_type() != a.scalar_type()) {
    throw py::value_error(std::string(name) + " tensor has the wrong shape, device, or dtype");
  }
}

// A caller's output.  One that autograd follows would keep the history, and so
// the gradients, of the values that the call overwrites.
void check_written(const at::Tensor& out, const at::Tensor& a, int64_t m, int64_t n) {
  check_output(out, a, m, n);
  if (at::GradMode::is_enabled() && out.requires_grad()) {
    throw py::value_error("an output tensor requires gradients; write it under torch.no_grad()");
  }
}

// An input read by rows: itself if its columns are contiguous and its rows
// do not overlap, else a contiguous copy.
at::Tensor by_rows(const at::Tensor& t) {
  const bool rows = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
  return rows ? t : t.contiguous();
}

void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// A workspace of `bytes`; keep it alive until the launches are queued.
struct Workspace {
  at::Tensor t;
  size_t bytes;
  Workspace(size_t n, const at::Tensor& like) : bytes(n) {
    if (n) t = at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
  }
  void* data() const { return bytes ? t.data_ptr() : nullptr; }
};

// Gradient of b [k, n] in b's own order: the transpose of [n, k] rows for a
// weight's W.t(), else [k, n] rows.
at::Tensor empty_like_weight(const at::Tensor& b) {
  const int64_t k = b.size(0), n = b.size(1);
  const bool nk = b.stride(0) == 1 && !(b.stride(1) == 1 && k > 1 && n > 1);
  return nk ? at::empty({n, k}, b.options()).t() : at::empty({k, n}, b.options());
}

std::tuple<int, at::Tensor, OptTensor> fused_linear(const at::Tensor& a, const at::Tensor& b, const OptTensor& bias,
                                                    int activation, const OptTensor& residual, const OptTensor& output,
                                                    const OptTensor& preact, bool return_preact, int64_t flags) {
  check_no_tangent("fused_linear", a, b, bias, residual, output, preact);
  check_inputs(a, b, "fused_linear");
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  check_vector(bias, a, n, "bias");
  at::Tensor res;
  if (residual.has_value()) {
    check_matrix(*residual, a, m, n, "residual");
    res = by_rows(*residual);
  }
  at::Tensor y = output.has_value() ? *output : at::empty({m, n}, a.options());
  if (output.has_value()) check_written(y, a, m, n);
  OptTensor z = preact;
  if (z.has_value()) {
    check_written(*z, a, m, n);
  } else if (return_preact) {
    z = at::empty({m, n}, a.options());
  }
  const Workspace ws(glq_fused_linear_workspace_bytes(dtype_of(a), a.data_ptr(), a.stride(0), a.stride(1), b.data_ptr(),
                                                      b.stride(0), b.stride(1), m, n, k),
                     a);
  const int status = glq_fused_linear(
      dtype_of(a), a.data_ptr(), a.stride(0), a.stride(1), b.data_ptr(), b.stride(0), b.stride(1), ptr(bias), activation,
      res.defined() ? res.data_ptr() : nullptr, res.defined() ? res.stride(0) : 0, ptr(z), z.has_value() ? z->stride(0) : 0,
      y.data_ptr(), y.stride(0), m, n, k, ws.data(), ws.bytes, stream_of(a), static_cast<unsigned int>(flags));
  if (output.has_value()) wrote(y);
  if (preact.has_value()) wrote(*z);
  return {status, y, z};
}

std::tuple<int, OptTensor, OptTensor, OptTensor> fused_linear_backward(const at::Tensor& grad, const at::Tensor& a,
                                                                       const at::Tensor& b, const OptTensor& preact,
                                                                       int activation, bool want_a, bool want_b,
                                                                       bool has_bias, int64_t flags) {
  check_no_tangent("fused_linear_backward", grad, a, b, preact);
  check_inputs(a, b, "fused_linear_backward");
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  check_matrix(grad, a, m, n, "grad_output");
  const at::Tensor dy = by_rows(grad);
  at::Tensor z;
  if (activation != GLQ_ACT_NONE) {
    if (!preact.has_value()) throw py::value_error("the backward pass of an activation needs preact");
    check_matrix(*preact, a, m, n, "preact");
    z = by_rows(*preact);
  }
  OptTensor da, db, dbias;
  if (want_a) da = at::empty({m, k}, a.options());
  if (want_b) db = empty_like_weight(b);
  if (has_bias) dbias = at::empty({n}, a.options());
  const Workspace ws(glq_fused_linear_backward_workspace_bytes(dtype_of(a), dy.data_ptr(), dy.stride(0), a.data_ptr(),
                                                               a.stride(0), a.stride(1), b.data_ptr(), b.stride(0),
                                                               b.stride(1), activation, has_bias ? 1 : 0, m, n, k),
                     a);
  const int status = glq_fused_linear_backward(
      dtype_of(a), dy.data_ptr(), dy.stride(0), z.defined() ? z.data_ptr() : nullptr, z.defined() ? z.stride(0) : 0,
      a.data_ptr(), a.stride(0), a.stride(1), b.data_ptr(), b.stride(0), b.stride(1), activation,
      ptr(da), da.has_value() ? da->stride(0) : 0, ptr(db),
      db.has_value() ? db->stride(0) : 0, db.has_value() ? db->stride(1) : 0, ptr(dbias), m, n, k,
      ws.data(), ws.bytes, stream_of(a), static_cast<unsigned int>(flags));
  return {status, da, db, dbias};
}

void check_pair(const at::Tensor& a, const at::Tensor& b_gate, const at::Tensor& b_up, const std::string& op) {
  check_inputs(a, b_gate, op);
  check_inputs(a, b_up, op);
  if (b_gate.size(1) != b_up.size(1)) {
    throw py::value_error("incompatible dimensions: " + shape_str(b_gate) + " and " + shape_str(b_up));
  }
}

std::tuple<int, at::Tensor, OptTensor, OptTensor> gated_linear(const at::Tensor& a, const at::Tensor& b_gate,
                                                               const at::Tensor& b_up, const OptTensor& bias_gate,
                                                               const OptTensor& bias_up, int activation,
                                                               const OptTensor& output, const OptTensor& gate,
                                                               const OptTensor& up, bool return_preact, int64_t flags) {
  check_no_tangent("gated_linear", a, b_gate, b_up, bias_gate, bias_up, output, gate, up);
  check_pair(a, b_gate, b_up, "gated_linear");
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = b_gate.size(1);
  check_vector(bias_gate, a, n, "bias_gate");
  check_vector(bias_up, a, n, "bias_up");
  at::Tensor y = output.has_value() ? *output : at::empty({m, n}, a.options());
  if (output.has_value()) check_written(y, a, m, n);
  OptTensor g = gate, u = up;
  if (g.has_value() != u.has_value()) throw py::value_error("gate and up are given together");
  if (g.has_value()) {
    check_written(*g, a, m, n);
    check_written(*u, a, m, n);
    if (m > 1 && g->stride(0) != u->stride(0)) throw py::value_error("gate and up need one row stride");
  } else if (return_preact) {
    g = at::empty({m, n}, a.options());
    u = at::empty({m, n}, a.options());
  }
  const int dtype = dtype_of(a);
  const Workspace ws(
      glq_gated_linear_workspace_bytes(dtype, a.data_ptr(), a.stride(0), a.stride(1), b_gate.data_ptr(),
                                       b_gate.stride(0), b_gate.stride(1), b_up.data_ptr(), b_up.stride(0),
                                       b_up.stride(1), m, n, k),
      a);
  const int status = glq_gated_linear(
      dtype, a.data_ptr(), a.stride(0), a.stride(1), b_gate.data_ptr(), b_gate.stride(0), b_gate.stride(1),
      b_up.data_ptr(), b_up.stride(0), b_up.stride(1), ptr(bias_gate), ptr(bias_up), activation,
      ptr(g), ptr(u), g.has_value() ? g->stride(0) : 0, y.data_ptr(), y.stride(0),
      m, n, k, ws.data(), ws.bytes, stream_of(a), static_cast<unsigned int>(flags));
  if (output.has_value()) wrote(y);
  if (gate.has_value()) {
    wrote(*g);
    wrote(*u);
  }
  return {status, y, g, u};
}

std::tuple<int, OptTensor, OptTensor, OptTensor, OptTensor, OptTensor> gated_linear_backward(
    const at::Tensor& grad, const at::Tensor& a, const at::Tensor& b_gate, const at::Tensor& b_up,
    const at::Tensor& gate, const at::Tensor& up, int activation, bool want_a, bool want_b, bool has_bias,
    int64_t flags) {
  check_no_tangent("gated_linear_backward", grad, a, b_gate, b_up, gate, up);
  check_pair(a, b_gate, b_up, "gated_linear_backward");
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = b_gate.size(1);
  check_matrix(grad, a, m, n, "grad_output");
  check_matrix(gate, a, m, n, "gate");
  check_matrix(up, a, m, n, "up");
  const at::Tensor dy = by_rows(grad);
  at::Tensor g = by_rows(gate), u = by_rows(up);
  if (m > 1 && g.stride(0) != u.stride(0)) {
    g = g.contiguous();
    u = u.contiguous();
  }
  OptTensor da, dbg, dbu, dbias_g, dbias_u;
  if (want_a) da = at::empty({m, k}, a.options());
  if (want_b) {
    dbg = empty_like_weight(b_gate);
    dbu = at::empty_strided(dbg->sizes(), dbg->strides(), dbg->options());
  }
  if (has_bias) {
    dbias_g = at::empty({n}, a.options());
    dbias_u = at::empty({n}, a.options());
  }
  const int dtype = dtype_of(a);
  const Workspace ws(
      glq_gated_linear_backward_workspace_bytes(dtype, a.data_ptr(), a.stride(0), a.stride(1), b_gate.data_ptr(),
                                                b_gate.stride(0), b_gate.stride(1), b_up.data_ptr(), b_up.stride(0),
                                                b_up.stride(1), has_bias ? 1 : 0, m, n, k),
      a);
  const int status = glq_gated_linear_backward(
      dtype, dy.data_ptr(), dy.stride(0), g.data_ptr(), u.data_ptr(), g.stride(0), a.data_ptr(), a.stride(0),
      a.stride(1), b_gate.data_ptr(), b_gate.stride(0), b_gate.stride(1), b_up.data_ptr(), b_up.stride(0),
      b_up.stride(1), activation, ptr(da), da.has_value() ? da->stride(0) : 0,
      ptr(dbg), ptr(dbu), dbg.has_value() ? dbg->stride(0) : 0,
      dbg.has_value() ? dbg->stride(1) : 0, ptr(dbias_g), ptr(dbias_u), m, n, k,
      ws.data(), ws.bytes, stream_of(a), static_cast<unsigned int>(flags));
  return {status, da, dbg, dbu, dbias_g, dbias_u};
}

void check_norm(const at::Tensor& x, const std::string& op) {
  if (x.dim() != 2) throw py::value_error(op + " expects a rank-2 tensor");
  if (!x.is_cuda()) throw py::value_error(op + " requires CUDA tensors");
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16) {
    throw py::value_error("inputs must share dtype float16 or bfloat16");
  }
}

std::tuple<int, at::Tensor, OptTensor, OptTensor> layer_norm(const at::Tensor& x, const OptTensor& weight,
                                                             const OptTensor& bias, double eps,
                                                             const OptTensor& output, bool return_stats,
                                                             int64_t flags) {
  check_no_tangent("layer_norm", x, weight, bias, output);
  check_norm(x, "layer_norm");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), n = x.size(1);
  check_vector(weight, x, n, "weight");
  check_vector(bias, x, n, "bias");
  const at::Tensor rows = by_rows(x);
  at::Tensor y = output.has_value() ? *output : at::empty({m, n}, x.options());
  if (output.has_value()) check_written(y, x, m, n);
  OptTensor mean, rstd;
  if (return_stats) {
    mean = at::empty({m}, x.options().dtype(at::kFloat));
    rstd = at::empty({m}, x.options().dtype(at::kFloat));
  }
  const int status = glq_layer_norm(dtype_of(x), rows.data_ptr(), rows.stride(0), ptr(weight), ptr(bias), eps,
                                    y.data_ptr(), y.stride(0), return_stats ? mean->data_ptr<float>() : nullptr,
                                    return_stats ? rstd->data_ptr<float>() : nullptr, m, n, stream_of(x),
                                    static_cast<unsigned int>(flags));
  if (output.has_value()) wrote(y);
  return {status, y, mean, rstd};
}

std::tuple<int, at::Tensor, OptTensor, OptTensor> layer_norm_backward(const at::Tensor& grad, const at::Tensor& x,
                                                                      const at::Tensor& mean, const at::Tensor& rstd,
                                                                      const OptTensor& weight, bool has_bias,
                                                                      bool need_weight, int64_t flags) {
  check_no_tangent("layer_norm_backward", grad, x, mean, rstd, weight);
  check_norm(x, "layer_norm_backward");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), n = x.size(1);
  check_matrix(grad, x, m, n, "grad_output");
  check_vector(weight, x, n, "weight");
  for (const at::Tensor* t : {&mean, &rstd}) {
    if (t->dim() != 1 || t->size(0) != m || t->device() != x.device() || t->scalar_type() != at::kFloat ||
        !t->is_contiguous()) {
      throw py::value_error("mean and rstd are contiguous float32 vectors of one value per row");
    }
  }
  const at::Tensor dy = by_rows(grad), rows = by_rows(x);
  at::Tensor dx = at::empty({m, n}, x.options());
  OptTensor dweight, dbias;
  if (weight.has_value() && need_weight) dweight = at::empty({n}, x.options());
  if (has_bias) dbias = at::empty({n}, x.options());
  const Workspace ws(dweight.has_value() || has_bias ? glq_layer_norm_backward_workspace_bytes(m, n) : 0, x);
  const int status = glq_layer_norm_backward(
      dtype_of(x), dy.data_ptr(), dy.stride(0), rows.data_ptr(), rows.stride(0), ptr(weight), mean.data_ptr<float>(),
      rstd.data_ptr<float>(), dx.data_ptr(), dx.stride(0), ptr(dweight),
      ptr(dbias), m, n, ws.data(), ws.bytes, stream_of(x), static_cast<unsigned int>(flags));
  return {status, dx, dweight, dbias};
}

}  // namespace

PYBIND11_MODULE(_glq_torch, mod) {
  mod.doc() = "Checks and launches of the gemm_lab operator API on libglq.so (torch current stream).";
  mod.def("linear", &linear, py::arg("op"), py::arg("a"), py::arg("b"), py::arg("out"), py::arg("bias"),
          py::arg("epilogue"), py::arg("split_k"), py::arg("partial"), py::arg("flags"));
  mod.def("linear_gather", &linear_gather, py::arg("a"), py::arg("b"), py::arg("bias"), py::arg("epilogue"),
          py::arg("y_ptrs"), py::arg("y_row_stride"), py::arg("y_col_offset"), py::arg("rank"),
          py::arg("signal_ptrs"), py::arg("counter"), py::arg("epoch"), py::arg("split_k"), py::arg("flags"));
  mod.def("fused_linear", &fused_linear);
  mod.def("fused_linear_backward", &fused_linear_backward);
  mod.def("gated_linear", &gated_linear);
  mod.def("gated_linear_backward", &gated_linear_backward);
  mod.def("layer_norm", &layer_norm);
  mod.def("layer_norm_backward", &layer_norm_backward);
}
