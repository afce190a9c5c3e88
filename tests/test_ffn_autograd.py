"""What torch has to know about the feed-forward operators: tensors written in place, forward-mode tangents, what a
call keeps and computes for its backward pass, and ahead-of-time tracing."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from gemm_lab_qualification_b200 import ffn, kernels

F16 = torch.float16


# ---------------------------------------------------------------- forward mode

def dual(*shape):
    t = torch.zeros(*shape, dtype=F16)
    return fwd.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("call", [
    lambda x, p: ffn.fused_linear(x, p), lambda x, p: ffn.fused_linear(p, x.t()),
    lambda x, p: ffn.fused_linear(p, p, x[0]), lambda x, p: ffn.fused_linear(p, p, None, None, x),
    lambda x, p: ffn.fused_linear_into(x, p, torch.zeros_like(p)), lambda x, p: ffn.fused_linear_into(p, p, x),
    lambda x, p: ffn.fused_linear_backward(x, p, p),
    lambda x, p: ffn.gated_linear(p, p, x), lambda x, p: ffn.gated_linear_into(p, p, p, x),
    lambda x, p: ffn.gated_linear_backward(p, p, p, p, x, p),
    lambda x, p: ffn.layer_norm(x), lambda x, p: ffn.layer_norm(p, x[0]), lambda x, p: ffn.layer_norm_into(x, p),
    lambda x, p: ffn.layer_norm_backward(x, p, p[0].float(), p[0].float()),
    lambda x, p: ffn.feed_forward(x, p, p, p),
])
def test_forward_mode_tangents_are_refused(call):
    """An output without a tangent would be a derivative of zero."""
    with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        call(dual(8, 8), torch.zeros(8, 8, dtype=F16))


@pytest.mark.gpu
def test_forward_mode_of_trainable_tensors(cuda_device):
    x, w = (torch.randn(8, 8, device="cuda").half() for _ in range(2))
    with fwd.dual_level():
        for t in (x, x.clone().requires_grad_()):
            with pytest.raises(Exception):
                ffn.fused_linear(fwd.make_dual(t, torch.ones_like(x)), w)
    with pytest.raises(Exception):
        torch.func.jvp(lambda v: ffn.layer_norm(v), (x,), (torch.ones_like(x),))
    assert ffn.fused_linear(x, w).shape == (8, 8)


# ---------------------------------------------------------------- tensors written in place

def matrices(n, size=64):
    gen = torch.Generator().manual_seed(n)
    return [torch.randn(size, size, generator=gen).to(F16).cuda() for _ in range(n)]


def writers():
    """(name, call that writes its first argument from the others)"""
    return [
        ("fused_linear_into", lambda out, a, b, c: ffn.fused_linear_into(a, b, out, residual=out)),
        ("preact", lambda out, a, b, c: ffn.fused_linear_into(a, b, c, activation="silu", preact=out)),
        ("gated_linear_into", lambda out, a, b, c: ffn.gated_linear_into(a, b, b, out)),
        ("gate", lambda out, a, b, c: ffn.gated_linear_into(a, b, b, c, gate=out, up=torch.empty_like(c))),
        ("up", lambda out, a, b, c: ffn.gated_linear_into(a, b, b, c, gate=torch.empty_like(c), up=out)),
        ("layer_norm_into", lambda out, a, b, c: ffn.layer_norm_into(a, out)),
        ("triton_matmul_into", lambda out, a, b, c: kernels.triton_matmul_into(a, b, out)),
        ("triton_bias_silu_into", lambda out, a, b, c: kernels.triton_bias_silu_into(a, b, a[0], out)),
    ]


@pytest.mark.gpu
@pytest.mark.parametrize("name,write", writers(), ids=[w[0] for w in writers()])
def test_writes_raise_the_version(cuda_device, name, write):
    """A tensor that a pending backward pass has saved cannot be overwritten unseen."""
    x, a, b, c = matrices(4)
    weight = torch.ones(64, dtype=F16, device="cuda", requires_grad=True)
    y = ffn.layer_norm(x, weight)  # saves x
    before = x._version
    write(x, a, b, c)
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_inputs_and_inference_tensors_keep_their_version(cuda_device):
    x, a, b, c = matrices(4)
    for _, write in writers():
        write(x, a, b, c)
    assert a._version == 0 and b._version == 0
    with torch.inference_mode():
        frozen = torch.empty_like(x)
    for _, write in writers():
        write(frozen, a, b, c)  # (has no version to raise)


@pytest.mark.gpu
def test_outputs_that_autograd_follows_are_refused(cuda_device):
    """Writing a tensor that requires gradients would leave it the history, and the gradients, of what it held."""
    x, a, b, c = matrices(4)
    for out in (x.clone().requires_grad_(), x.clone().requires_grad_() * 1):
        was = out.detach().clone()
        for name, write in writers()[:6]:
            with pytest.raises(ValueError, match="requires gradients"):
                write(out, a, b, c)
        assert torch.equal(out.detach(), was)
    # An optimizer's or a decoder's writes are outside autograd.
    with torch.no_grad():
        for name, write in writers():
            write(out, a, b, c)
    # Inputs may require gradients: the call is documented as not differentiable.
    assert not ffn.fused_linear_into(a.requires_grad_(), b, c).requires_grad


# ---------------------------------------------------------------- what a call runs

class FakeBinding:
    """Counts the native calls, and answers them on the CPU."""

    def __init__(self):
        self.calls = []

    def fused_linear(self, a, b, bias, act, residual, output, preact, return_preact, flags):
        self.calls.append("fused_linear")
        z = a @ b if bias is None else a @ b + bias
        y = z.clone() if residual is None else z + residual
        return 0, y, z.clone() if return_preact else None

    def fused_linear_backward(self, dy, a, b, z, act, want_a, want_b, has_bias, flags):
        self.calls.append("fused_linear_backward")
        return (0, dy @ b.t() if want_a else None, a.t() @ dy if want_b else None, dy.sum(0) if has_bias else None)

    def layer_norm(self, x, weight, bias, eps, output, return_stats, flags):
        return 0, x.clone(), x.float().mean(1), torch.ones(x.shape[0])

    def layer_norm_backward(self, dy, x, mean, rstd, weight, has_bias, need_weight, flags):
        self.calls.append(("layer_norm_backward", has_bias, need_weight))
        return (0, dy.clone(), dy.sum(0) if weight is not None and need_weight else None,
                dy.sum(0) if has_bias else None)


@pytest.fixture
def native_calls(monkeypatch):
    fake = FakeBinding()
    monkeypatch.setattr(ffn, "_binding", lambda: fake)
    return fake.calls


@pytest.mark.parametrize("residual", [False, True])
def test_kept_preactivation_costs_no_second_product(native_calls, residual):
    """Without an activation the one product gives both results."""
    gen = torch.Generator().manual_seed(1)
    a, b, r = (torch.randn(4, 4, generator=gen, dtype=torch.float64).requires_grad_() for _ in range(3))
    y, z = ffn.fused_linear(a, b, None, None, r if residual else None, return_preact=True)
    assert native_calls == ["fused_linear"]
    assert torch.equal(z, (a @ b).detach()) and not z.requires_grad
    assert y.data_ptr() != z.data_ptr()
    y.backward(torch.ones_like(y))
    assert native_calls == ["fused_linear", "fused_linear_backward"]
    assert torch.equal(a.grad, torch.ones_like(y) @ b.detach().t())
    native_calls.clear()
    assert ffn.fused_linear(a, b).requires_grad and native_calls == ["fused_linear"]


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("activation", [None, "gelu"])
def test_kept_preactivation_is_the_same_with_gradients(cuda_device, m, activation):
    gen = torch.Generator().manual_seed(m)
    a, w = torch.randn(m, 72, generator=gen).to(F16).cuda(), torch.randn(136, 72, generator=gen).to(F16).cuda()
    r = torch.randn(m, 136, generator=gen).to(F16).cuda()
    for res in (None, r):
        want = ffn.fused_linear(a, w.t(), None, activation, res, return_preact=True)
        got = ffn.fused_linear(a.clone().requires_grad_(), w.t(), None, activation, res, return_preact=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert got[0].requires_grad and not got[1].requires_grad


@pytest.mark.parametrize("frozen", [True, False])
def test_frozen_norm_weights_cost_no_gradient(native_calls, frozen):
    x, weight = torch.randn(3, 4, requires_grad=True), torch.ones(4, requires_grad=not frozen)
    ffn.layer_norm(x, weight).sum().backward()
    assert native_calls == [("layer_norm_backward", False, not frozen)]
    assert (weight.grad is None) == frozen and x.grad is not None


@pytest.mark.gpu
def test_layer_norm_backward_without_the_weights_gradient(cuda_device):
    gen = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(40, 264, generator=gen).to(F16).cuda() for _ in range(2))
    w = torch.randn(264, generator=gen).to(F16).cuda()
    _, mean, rstd = ffn.layer_norm(x, w, return_stats=True)
    dx, dw, db = ffn.layer_norm_backward(dy, x, mean, rstd, w, has_bias=True)
    for has_bias in (True, False):
        got = ffn.layer_norm_backward(dy, x, mean, rstd, w, has_bias=has_bias, need_weight=False)
        assert torch.equal(got[0], dx) and got[1] is None
        assert torch.equal(got[2], db) if has_bias else got[2] is None


# ---------------------------------------------------------------- tracing

@pytest.mark.gpu
def test_custom_ops_trace_ahead_of_time(cuda_device):
    """Forward and backward graphs traced with symbolic sizes give what the eager calls give."""
    gen = torch.Generator().manual_seed(8)

    def leaf(*shape):
        return torch.randn(*shape, generator=gen).to(F16).cuda().requires_grad_()

    a, w, w2, bias, res, scale = leaf(12, 64), leaf(72, 64), leaf(64, 72), leaf(72), leaf(12, 72), leaf(64)
    ops = torch.ops.gemm_lab
    tests = ("test_aot_dispatch_dynamic",)
    for activation in ("silu", None):
        torch.library.opcheck(ops.fused_linear, (a, w.t(), bias, activation, res), test_utils=tests)
    torch.library.opcheck(ops.fused_linear, (a, w2, None, None, None, True), test_utils=tests)
    torch.library.opcheck(ops.gated_linear, (a, w.t(), w2, bias, bias, "gelu"), test_utils=tests)
    torch.library.opcheck(ops.layer_norm, (a, scale, scale, 1e-5), test_utils=tests)
    torch.library.opcheck(ops.layer_norm, (a, None, None, 1e-5), test_utils=tests)
