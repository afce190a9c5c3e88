"""The feed-forward half of a transformer block on the native sm_100a kernels.

Beside the lab's ``act(a @ b + bias)`` operators (``kernels``), with the same
conventions -- rank-2 float16 / bfloat16 CUDA tensors, ``b`` a [K, N] operand
that is either a linear layer's weight as ``W.t()`` or N-contiguous, outputs
allocated or passed to the ``*_into`` forms, ``ValueError`` for a broken
contract, ``launch_options`` for the launch flags, the current stream of the
operands' device:

* ``fused_linear`` -- ``act(a @ b + bias) + residual``;
* ``gated_linear`` -- ``act(a @ b_gate + bias_gate) * (a @ b_up + bias_up)``
  in one pass over ``a``;
* ``layer_norm`` -- row normalisation with weight and bias;
* ``feed_forward`` -- the pre-norm block that they make up.

Rows, columns and contraction of the products go up to 65535 * 64.
``activation`` is None, "silu", "gelu" (exact), "gelu_tanh" or "relu".

Called on tensors that require gradients, they are differentiable: the call
goes through the custom op ``gemm_lab::<name>`` (with fake kernels for
tracing), which keeps what its backward pass reads.  The ``*_backward``
functions are those passes for callers that run their own.  Gradients have
the inputs' 16-bit type; every sum is FP32 with one rounding, except that the
gradient of the pre-activations is rounded to 16 bits before the products that
read it (in float16 it overflows beyond 65504).  The backward passes
themselves are not differentiable, and forward-mode tangents
(``torch.autograd.forward_ad``) are refused.

The ``*_into`` forms write in place and raise the version of what they wrote,
as torch's own operations do: a pending backward pass that saved the tensor
then ends with torch's error instead of with wrong gradients.  They are not
differentiable, and while gradients are recorded they refuse an output that
requires them.

Results are the same bits on every run of the same call; which gradients are
asked for together may change the order of their sums.  All calls can be
captured into CUDA graphs after a first call on the device.  To capture a
``.backward()``, let no eager graph of the same leaves live at that time (torch
keeps the leaves' gradient nodes on the stream they were made on), or capture
the ``*_backward`` functions.

The reference has no counterpart (its fused epilogue is bias + SiLU,
kernels.py:191-249, inference only).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _native
from .kernels import _binding, _flags

__all__ = [
    "fused_linear", "fused_linear_into", "fused_linear_backward",
    "gated_linear", "gated_linear_into", "gated_linear_backward",
    "layer_norm", "layer_norm_into", "layer_norm_backward", "feed_forward",
]


def _activation(name: str | None) -> int:
    try:
        return _native.ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError("activation must be None, 'silu', 'gelu', 'gelu_tanh' or 'relu'") from None


def _check(status: int, what: str) -> None:
    if status != _native.STATUS_OK:
        raise _native.GlqError(status, what)


def _differentiable(*tensors: Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ---------------------------------------------------------------- linear + bias + activation + residual

def _fused_linear(a, b, bias, activation, residual, output=None, preact=None, return_preact=False):
    status, y, z = _binding().fused_linear(a, b, bias, _activation(activation), residual, output, preact,
                                           return_preact, _flags())
    _check(status, "glq_fused_linear")
    return y, z


def fused_linear_into(a: Tensor, b: Tensor, output: Tensor, bias: Tensor | None = None,
                      activation: str | None = None, residual: Tensor | None = None,
                      preact: Tensor | None = None) -> Tensor:
    """output = act(a @ b + bias) + residual; preact, if given, receives
    ``a @ b + bias``.  ``output`` may be the residual itself (the residual
    stream updated in place); apart from that, outputs overlap no operand.
    Not differentiable."""
    return _fused_linear(a, b, bias, activation, residual, output, preact)[0]


def fused_linear(a: Tensor, b: Tensor, bias: Tensor | None = None, activation: str | None = None,
                 residual: Tensor | None = None, return_preact: bool = False):
    """act(a @ b + bias) + residual; with return_preact, also ``a @ b + bias``
    (what the backward pass of an activation reads; differentiable only
    through the first output)."""
    if _differentiable(a, b, bias, residual):
        y, z = fused_linear_op(a, b, bias, activation, residual, return_preact)
    else:
        y, z = _fused_linear(a, b, bias, activation, residual, return_preact=return_preact)
    return (y, z) if return_preact else y


def fused_linear_backward(grad_output: Tensor, a: Tensor, b: Tensor, preact: Tensor | None = None,
                          activation: str | None = None, has_bias: bool = False, need_a: bool = True,
                          need_b: bool = True) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """(grad a, grad b, grad bias) of ``fused_linear``; the residual's gradient
    is grad_output.  preact is required with an activation.  grad b has b's
    memory order."""
    status, da, db, dbias = _binding().fused_linear_backward(grad_output, a, b, preact, _activation(activation),
                                                             need_a, need_b, has_bias, _flags())
    _check(status, "glq_fused_linear_backward")
    return da, db, dbias


# ---------------------------------------------------------------- gated pair

def _gated_linear(a, b_gate, b_up, bias_gate, bias_up, activation, output=None, gate=None, up=None,
                  return_preact=False):
    status, y, g, u = _binding().gated_linear(a, b_gate, b_up, bias_gate, bias_up, _activation(activation), output,
                                              gate, up, return_preact, _flags())
    _check(status, "glq_gated_linear")
    return y, g, u


def gated_linear_into(a: Tensor, b_gate: Tensor, b_up: Tensor, output: Tensor, bias_gate: Tensor | None = None,
                      bias_up: Tensor | None = None, activation: str | None = "silu", gate: Tensor | None = None,
                      up: Tensor | None = None) -> Tensor:
    """output = act(a @ b_gate + bias_gate) * (a @ b_up + bias_up); gate and up,
    if given (both, one row stride), receive the two projections.  Outputs
    overlap no other operand.  Not differentiable."""
    return _gated_linear(a, b_gate, b_up, bias_gate, bias_up, activation, output, gate, up)[0]


def gated_linear(a: Tensor, b_gate: Tensor, b_up: Tensor, bias_gate: Tensor | None = None,
                 bias_up: Tensor | None = None, activation: str | None = "silu", return_preact: bool = False):
    """act(a @ b_gate + bias_gate) * (a @ b_up + bias_up); with return_preact,
    also the two projections (what the backward pass reads; differentiable
    only through the first output)."""
    if _differentiable(a, b_gate, b_up, bias_gate, bias_up):
        out = gated_linear_op(a, b_gate, b_up, bias_gate, bias_up, activation)
    else:
        out = _gated_linear(a, b_gate, b_up, bias_gate, bias_up, activation, return_preact=return_preact)
    return tuple(out) if return_preact else out[0]


def gated_linear_backward(grad_output: Tensor, a: Tensor, b_gate: Tensor, b_up: Tensor, gate: Tensor, up: Tensor,
                          activation: str | None = "silu", has_bias: bool = False, need_a: bool = True,
                          need_b: bool = True):
    """(grad a, grad b_gate, grad b_up, grad bias_gate, grad bias_up) of
    ``gated_linear``; what is not asked for is None.  Both weight gradients
    have b_gate's memory order."""
    status, *grads = _binding().gated_linear_backward(grad_output, a, b_gate, b_up, gate, up, _activation(activation),
                                                      need_a, need_b, has_bias, _flags())
    _check(status, "glq_gated_linear_backward")
    return tuple(grads)


# ---------------------------------------------------------------- layer norm

def _layer_norm(x, weight, bias, eps, output=None, return_stats=False):
    status, y, mean, rstd = _binding().layer_norm(x, weight, bias, eps, output, return_stats, _flags())
    _check(status, "glq_layer_norm")
    return y, mean, rstd


def layer_norm_into(x: Tensor, output: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
                    eps: float = 1e-5) -> Tensor:
    """output = layer_norm(x).  Not differentiable."""
    return _layer_norm(x, weight, bias, eps, output)[0]


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
               return_stats: bool = False):
    """(x - mean) * rstd * weight + bias per row of x [M, N]; with return_stats,
    also the float32 mean and rstd (differentiable only through the first
    output)."""
    if _differentiable(x, weight, bias):
        out = layer_norm_op(x, weight, bias, eps)
    else:
        out = _layer_norm(x, weight, bias, eps, return_stats=return_stats)
    return tuple(out) if return_stats else out[0]


def layer_norm_backward(grad_output: Tensor, x: Tensor, mean: Tensor, rstd: Tensor, weight: Tensor | None = None,
                        has_bias: bool = False,
                        need_weight: bool = True) -> tuple[Tensor, Tensor | None, Tensor | None]:
    """(grad x, grad weight, grad bias) of ``layer_norm``; need_weight False
    leaves out the gradient of a weight that is not trained."""
    status, dx, dweight, dbias = _binding().layer_norm_backward(grad_output, x, mean, rstd, weight, has_bias,
                                                                need_weight, _flags())
    _check(status, "glq_layer_norm_backward")
    return dx, dweight, dbias


# ---------------------------------------------------------------- the block

def feed_forward(x: Tensor, b_gate: Tensor, b_up: Tensor, b_down: Tensor, norm_weight: Tensor | None = None,
                 norm_bias: Tensor | None = None, bias_gate: Tensor | None = None, bias_up: Tensor | None = None,
                 bias_down: Tensor | None = None, activation: str | None = "silu", eps: float = 1e-5) -> Tensor:
    """The pre-norm feed-forward block of a transformer layer:
    ``x + gated_linear(layer_norm(x)) @ b_down + bias_down``."""
    h = layer_norm(x, norm_weight, norm_bias, eps)
    h = gated_linear(h, b_gate, b_up, bias_gate, bias_up, activation)
    return fused_linear(h, b_down, bias_down, None, x)


# ---------------------------------------------------------------- torch custom ops

def _or_empty(t: Tensor | None, like: Tensor) -> Tensor:
    return like.new_empty(0) if t is None else t


def _weight_order(b: Tensor) -> Tensor:
    """An empty gradient of b [K, N] in b's memory order."""
    k, n = b.shape
    nk = b.stride(0) == 1 and not (b.stride(1) == 1 and k > 1 and n > 1)
    return b.new_empty((n, k)).t() if nk else b.new_empty((k, n))


@torch.library.custom_op("gemm_lab::fused_linear", mutates_args=())
def fused_linear_op(a: Tensor, b: Tensor, bias: Optional[Tensor], activation: Optional[str],
                    residual: Optional[Tensor], keep_preact: bool = False) -> tuple[Tensor, Tensor]:
    """(act(a @ b + bias) + residual, a @ b + bias); the latter is empty
    without an activation unless keep_preact asks for it."""
    y, z = _fused_linear(a, b, bias, activation, residual, return_preact=activation is not None or keep_preact)
    return y, _or_empty(z, a)


@fused_linear_op.register_fake
def _(a, b, bias, activation, residual, keep_preact=False):
    _activation(activation)
    if a.ndim != 2 or b.ndim != 2 or a.shape[1] != b.shape[0]:
        raise ValueError("incompatible matrix shapes")
    y = a.new_empty((a.shape[0], b.shape[1]))
    return y, (torch.empty_like(y) if activation is not None or keep_preact else a.new_empty(0))


@torch.library.custom_op("gemm_lab::fused_linear_backward", mutates_args=())
def fused_linear_backward_op(grad_output: Tensor, a: Tensor, b: Tensor, preact: Tensor, activation: Optional[str],
                             has_bias: bool, need_a: bool, need_b: bool) -> tuple[Tensor, Tensor, Tensor]:
    grads = fused_linear_backward(grad_output, a, b, preact if activation is not None else None, activation, has_bias,
                                  need_a, need_b)
    return tuple(_or_empty(g, a) for g in grads)


@fused_linear_backward_op.register_fake
def _(grad_output, a, b, preact, activation, has_bias, need_a, need_b):
    return (a.new_empty(a.shape) if need_a else a.new_empty(0), _weight_order(b) if need_b else a.new_empty(0),
            a.new_empty(b.shape[1]) if has_bias else a.new_empty(0))


def _fused_linear_setup(ctx, inputs, output):
    a, b, bias, activation, residual, _ = inputs
    ctx.save_for_backward(a, b, output[1] if activation is not None else None)
    ctx.activation, ctx.has_bias = activation, bias is not None
    ctx.mark_non_differentiable(output[1])


def _fused_linear_grad(ctx, grad_y, _):
    a, b, z = ctx.saved_tensors
    need = ctx.needs_input_grad
    want_bias = ctx.has_bias and need[2]
    da = db = dbias = None
    if need[0] or need[1] or want_bias:
        da, db, dbias = fused_linear_backward_op(grad_y, a, b, _or_empty(z, a), ctx.activation, want_bias, need[0],
                                                 need[1])
    return (da if need[0] else None, db if need[1] else None, dbias if want_bias else None, None,
            grad_y if need[4] else None, None)


fused_linear_op.register_autograd(_fused_linear_grad, setup_context=_fused_linear_setup)


@torch.library.custom_op("gemm_lab::gated_linear", mutates_args=())
def gated_linear_op(a: Tensor, b_gate: Tensor, b_up: Tensor, bias_gate: Optional[Tensor], bias_up: Optional[Tensor],
                    activation: Optional[str]) -> tuple[Tensor, Tensor, Tensor]:
    """(act(gate) * up, gate, up)."""
    return _gated_linear(a, b_gate, b_up, bias_gate, bias_up, activation, return_preact=True)


@gated_linear_op.register_fake
def _(a, b_gate, b_up, bias_gate, bias_up, activation):
    _activation(activation)
    if a.ndim != 2 or b_gate.ndim != 2 or a.shape[1] != b_gate.shape[0] or b_gate.shape != b_up.shape:
        raise ValueError("incompatible matrix shapes")
    y = a.new_empty((a.shape[0], b_gate.shape[1]))
    return y, torch.empty_like(y), torch.empty_like(y)


@torch.library.custom_op("gemm_lab::gated_linear_backward", mutates_args=())
def gated_linear_backward_op(grad_output: Tensor, a: Tensor, b_gate: Tensor, b_up: Tensor, gate: Tensor, up: Tensor,
                             activation: Optional[str], has_bias: bool, need_a: bool,
                             need_b: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    grads = gated_linear_backward(grad_output, a, b_gate, b_up, gate, up, activation, has_bias, need_a, need_b)
    return tuple(_or_empty(g, a) for g in grads)


@gated_linear_backward_op.register_fake
def _(grad_output, a, b_gate, b_up, gate, up, activation, has_bias, need_a, need_b):
    bias = [a.new_empty(b_gate.shape[1]) if has_bias else a.new_empty(0) for _ in range(2)]
    weights = [_weight_order(b_gate) if need_b else a.new_empty(0) for _ in range(2)]
    return (a.new_empty(a.shape) if need_a else a.new_empty(0), *weights, *bias)


def _gated_linear_setup(ctx, inputs, output):
    a, b_gate, b_up, bias_gate, bias_up, activation = inputs
    ctx.save_for_backward(a, b_gate, b_up, output[1], output[2])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1], output[2])


def _gated_linear_grad(ctx, grad_y, *_):
    a, b_gate, b_up, gate, up = ctx.saved_tensors
    need = ctx.needs_input_grad
    want_b, want_bias = need[1] or need[2], need[3] or need[4]
    grads = gated_linear_backward_op(grad_y, a, b_gate, b_up, gate, up, ctx.activation, want_bias, need[0], want_b)
    return (*(g if n else None for g, n in zip(grads, need)), None)


gated_linear_op.register_autograd(_gated_linear_grad, setup_context=_gated_linear_setup)


@torch.library.custom_op("gemm_lab::layer_norm", mutates_args=())
def layer_norm_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
                  eps: float) -> tuple[Tensor, Tensor, Tensor]:
    """(normalised rows, mean, rstd)."""
    return _layer_norm(x, weight, bias, eps, return_stats=True)


@layer_norm_op.register_fake
def _(x, weight, bias, eps):
    if x.ndim != 2:
        raise ValueError("layer_norm expects a rank-2 tensor")
    stats = x.new_empty(x.shape[0], dtype=torch.float32)
    return x.new_empty(x.shape), stats, torch.empty_like(stats)


@torch.library.custom_op("gemm_lab::layer_norm_backward", mutates_args=())
def layer_norm_backward_op(grad_output: Tensor, x: Tensor, mean: Tensor, rstd: Tensor, weight: Optional[Tensor],
                           has_bias: bool, need_weight: bool = True) -> tuple[Tensor, Tensor, Tensor]:
    return tuple(_or_empty(g, x) for g in layer_norm_backward(grad_output, x, mean, rstd, weight, has_bias, need_weight))


@layer_norm_backward_op.register_fake
def _(grad_output, x, mean, rstd, weight, has_bias, need_weight=True):
    n = x.shape[1]
    return (x.new_empty(x.shape), x.new_empty(n if weight is not None and need_weight else 0),
            x.new_empty(n if has_bias else 0))


def _layer_norm_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.mark_non_differentiable(output[1], output[2])


def _layer_norm_grad(ctx, grad_y, *_):
    x, weight, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dweight, dbias = layer_norm_backward_op(grad_y, x, mean, rstd, weight, need[2], need[1])
    return dx if need[0] else None, dweight if need[1] else None, dbias if need[2] else None, None


layer_norm_op.register_autograd(_layer_norm_grad, setup_context=_layer_norm_setup)
