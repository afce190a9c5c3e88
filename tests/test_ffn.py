"""The feed-forward operators without a GPU: refusals, workspace sizes, tracing, and the test reference itself."""
from __future__ import annotations

import inspect

import pytest
import torch

import ffn_reference as ref
from gemm_lab_qualification_b200 import _native as native
from gemm_lab_qualification_b200 import ffn

OK, INVALID, SHAPE, WORKSPACE, LAYOUT, DEVICE = 0, 1, 2, 4, 5, 7
P = 1 << 20  # a 16-byte aligned address that no call here reaches


def fused(m=4, n=64, k=64, dtype=0, a=P, a_rs=64, a_cs=1, b=P, b_ks=1, b_ns=64, bias=None, act=0, res=None, res_rs=64,
          z=None, z_rs=64, y=P, y_rs=64, ws=None, ws_bytes=0, flags=0):
    return native.library().glq_fused_linear(dtype, a, a_rs, a_cs, b, b_ks, b_ns, bias, act, res, res_rs, z, z_rs, y,
                                             y_rs, m, n, k, ws, ws_bytes, None, flags)


def gated(m=4, n=64, k=64, dtype=0, a=P, bg=P, bu=P, b_ns=64, act=1, g=None, u=None, gu_rs=64, y=P, y_rs=64, ws=None,
          ws_bytes=0, flags=0):
    return native.library().glq_gated_linear(dtype, a, 64, 1, bg, 1, b_ns, bu, 1, b_ns, None, None, act, g, u, gu_rs,
                                             y, y_rs, m, n, k, ws, ws_bytes, None, flags)


def norm(m=4, n=64, dtype=0, x=P, x_rs=64, w=None, b=None, eps=1e-5, y=P, y_rs=64, mean=None, rstd=None, flags=0):
    return native.library().glq_layer_norm(dtype, x, x_rs, w, b, eps, y, y_rs, mean, rstd, m, n, None, flags)


needs_no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that pass every check would launch")


@needs_no_gpu
@pytest.mark.parametrize("call", [fused, gated, norm])
def test_valid_calls_reach_the_device(call):
    assert call() == DEVICE


@needs_no_gpu
@pytest.mark.parametrize("call,change,want", [
    (fused, dict(dtype=2), INVALID), (fused, dict(act=5), INVALID), (fused, dict(act=-1), INVALID),
    (fused, dict(flags=4), INVALID), (fused, dict(m=-1), SHAPE), (fused, dict(k=1 << 40), SHAPE),
    (fused, dict(n=1 << 23), SHAPE), (fused, dict(a=None), INVALID), (fused, dict(b=None), INVALID),
    (fused, dict(y=None), INVALID), (fused, dict(a=P + 1), INVALID), (fused, dict(b=P + 1), INVALID),
    (fused, dict(bias=P + 1), INVALID), (fused, dict(res=P + 1), INVALID), (fused, dict(z=P + 1), INVALID),
    (fused, dict(y=P + 1), INVALID), (fused, dict(y_rs=63), LAYOUT), (fused, dict(z=P, z_rs=63), LAYOUT),
    (fused, dict(res=P, res_rs=-1), SHAPE), (fused, dict(a=P + 2), WORKSPACE), (fused, dict(b_ns=65), WORKSPACE),
    (fused, dict(a=P + 2, ws=P, ws_bytes=16), WORKSPACE), (fused, dict(a=P + 2, ws=P + 16, ws_bytes=1 << 20), WORKSPACE),
    (fused, dict(a=P + 2, ws=P, ws_bytes=1 << 20), DEVICE), (fused, dict(m=0, y=None), OK), (fused, dict(n=0, y=None), OK),
    (fused, dict(k=0, a=None, b=None), DEVICE),
    (gated, dict(act=9), INVALID), (gated, dict(bg=None), INVALID), (gated, dict(bu=None), INVALID),
    (gated, dict(g=P), INVALID), (gated, dict(u=P), INVALID), (gated, dict(g=P, u=P, gu_rs=10), LAYOUT),
    (gated, dict(y_rs=3), LAYOUT), (gated, dict(bu=P + 1), INVALID), (gated, dict(bu=P + 2), WORKSPACE),
    (gated, dict(m=0), OK),
    (norm, dict(dtype=3), INVALID), (norm, dict(eps=-1.0), INVALID), (norm, dict(eps=float("nan")), INVALID),
    (norm, dict(mean=P), INVALID), (norm, dict(rstd=P), INVALID), (norm, dict(mean=P + 2, rstd=P), INVALID),
    (norm, dict(x=None), INVALID), (norm, dict(y=P + 1), INVALID), (norm, dict(y_rs=2), LAYOUT),
    (norm, dict(x_rs=-5), SHAPE), (norm, dict(m=-1), SHAPE), (norm, dict(m=0, x=None, y=None), OK),
])
def test_refusals(call, change, want):
    assert call(**change) == want


def fused_backward(m=4, n=64, k=64, dtype=0, dy=P, dy_rs=64, z=P, a=P, b=P, act=1, da=P, da_rs=64, db=P, db_ks=1,
                   db_ns=64, dbias=None, ws=P, ws_bytes=1 << 30, flags=0):
    return native.library().glq_fused_linear_backward(dtype, dy, dy_rs, z, 64, a, 64, 1, b, 1, 64, act, da, da_rs, db,
                                                      db_ks, db_ns, dbias, m, n, k, ws, ws_bytes, None, flags)


def gated_backward(m=4, n=64, k=64, dy=P, g=P, u=P, gu_rs=64, da=P, dbg=P, dbu=P, db_ks=1, db_ns=64, dbias_g=None,
                   dbias_u=None, act=1):
    return native.library().glq_gated_linear_backward(0, dy, 64, g, u, gu_rs, P, 64, 1, P, 1, 64, P, 1, 64, act, da, 64,
                                                      dbg, dbu, db_ks, db_ns, dbias_g, dbias_u, m, n, k, P, 1 << 30,
                                                      None, 0)


def norm_backward(m=4, n=64, dy=P, x=P, mean=P, rstd=P, dx=P, dx_rs=64, dw=None, db=None):
    return native.library().glq_layer_norm_backward(0, dy, 64, x, 64, None, mean, rstd, dx, dx_rs, dw, db, m, n, P,
                                                    1 << 30, None, 0)


@needs_no_gpu
@pytest.mark.parametrize("call,change,want", [
    (fused_backward, {}, DEVICE), (fused_backward, dict(dtype=7), INVALID), (fused_backward, dict(act=5), INVALID),
    (fused_backward, dict(dy=None), INVALID), (fused_backward, dict(z=None), INVALID),
    (fused_backward, dict(z=None, act=0), DEVICE), (fused_backward, dict(a=None), INVALID),
    (fused_backward, dict(a=None, db=None), DEVICE), (fused_backward, dict(b=None), INVALID),
    (fused_backward, dict(b=None, da=None), DEVICE), (fused_backward, dict(db_ks=2), LAYOUT),
    (fused_backward, dict(db_ns=60), LAYOUT), (fused_backward, dict(db_ks=64, db_ns=1), DEVICE),
    (fused_backward, dict(da_rs=60), LAYOUT), (fused_backward, dict(dy_rs=60), SHAPE),
    (fused_backward, dict(dy=P + 1), INVALID), (fused_backward, dict(dbias=P + 1), INVALID),
    (fused_backward, dict(flags=8), INVALID), (fused_backward, dict(m=-1), SHAPE),
    (gated_backward, {}, DEVICE), (gated_backward, dict(g=None), INVALID), (gated_backward, dict(u=None), INVALID),
    (gated_backward, dict(dbg=None), INVALID), (gated_backward, dict(dbias_g=P), INVALID),
    (gated_backward, dict(gu_rs=8), SHAPE), (gated_backward, dict(dbg=None, dbu=None), DEVICE),
    (norm_backward, {}, DEVICE), (norm_backward, dict(dx=None), INVALID), (norm_backward, dict(mean=None), INVALID),
    (norm_backward, dict(dx_rs=8), LAYOUT), (norm_backward, dict(rstd=P + 1), INVALID),
    (norm_backward, dict(dw=P + 1), INVALID),
])
def test_backward_refusals(call, change, want):
    assert call(**change) == want


def test_workspace_sizes():
    lib = native.library()
    aligned = lib.glq_fused_linear_workspace_bytes(0, P, 64, 1, P, 1, 64, 4, 64, 64)
    assert aligned == 0
    # A of 4 rows, W of 64 rows, 61 columns each in 64-element pitches, in 256-byte steps.
    assert lib.glq_fused_linear_workspace_bytes(0, P, 61, 1, P, 1, 61, 4, 64, 61) == 4 * 128 + 64 * 128
    assert lib.glq_fused_linear_workspace_bytes(0, P, 64, 1, P, 1, 61, 0, 64, 61) == 0
    # Rows at odd multiples of 16 bytes: the smaller operand is copied to whole sectors where that pays.
    whole, off = (lib.glq_fused_linear_workspace_bytes(0, P, ld, 1, P, 1, ld, 512, 8192, 4104) for ld in (4112, 4104))
    assert off - whole == 512 * 4112 * 2
    whole, off = (lib.glq_fused_linear_workspace_bytes(0, P, ld, 1, P, 1, ld, 512, 256, 136) for ld in (144, 136))
    assert off == whole
    # The gated pair copies an up weight of another order than the gate's.
    assert lib.glq_gated_linear_workspace_bytes(0, P, 64, 1, P, 1, 64, P, 64, 1, 4, 64, 64) == 64 * 128
    assert lib.glq_gated_linear_workspace_bytes(0, P, 64, 1, P, 64, 1, P, 64, 1, 4, 64, 64) == 0
    # dz, and dgate and dup; a linear layer without activation reads dy as it is.
    assert lib.glq_fused_linear_backward_workspace_bytes(0, P, 64, P, 64, 1, P, 1, 64, 1, 0, 4, 64, 64) == 4 * 128
    assert lib.glq_fused_linear_backward_workspace_bytes(0, P, 64, P, 64, 1, P, 1, 64, 0, 0, 4, 64, 64) == 0
    assert lib.glq_gated_linear_backward_workspace_bytes(0, P, 64, 1, P, 1, 64, P, 1, 64, 0, 4, 64, 64) == 2 * 4 * 128
    assert lib.glq_layer_norm_backward_workspace_bytes(0, 64) == 0
    assert lib.glq_layer_norm_backward_workspace_bytes(8, 64) > 0


def test_operands_copied_anyway_do_not_weigh_on_the_other():
    """A with rows that TMA cannot address is copied to whole sectors whatever the plan: B, off its sectors, then
    decides as beside an A in whole sectors."""
    lib = native.library()

    def copied(a, a_ld, b, b_ld, m, n, k):
        size = lib.glq_fused_linear_workspace_bytes(0, a, a_ld, 1, b, 1, b_ld, m, n, k)
        return size - lib.glq_fused_linear_workspace_bytes(0, P, k, 1, P, 1, k, m, n, k)

    m, n, k = 4096, 2048, 2048
    assert copied(P, k, P, k + 8, m, n, k) == 0  # (one operand off: not worth a copy)
    assert copied(P + 2, k + 1, P, k + 8, m, n, k) == m * k * 2
    assert copied(P, k + 8, P + 2, k + 1, n, m, k) == m * k * 2
    # The gated pair: an up weight of the other order is copied like that too.
    def gated_copies(a_ld, u_ks, u_ns):
        return lib.glq_gated_linear_workspace_bytes(0, P, a_ld, 1, P, 1, k, P, u_ks, u_ns, 8192, 1024, k)

    whole = gated_copies(k, 1, k)
    assert gated_copies(k + 8, 1, k) == whole
    assert gated_copies(k + 8, 1032, 1) - whole == 1024 * k * 2


@pytest.mark.parametrize("call", [
    lambda a, b: ffn.fused_linear(a, b), lambda a, b: ffn.gated_linear(a, b, b),
    lambda a, b: ffn.fused_linear_backward(a, a, b), lambda a, b: ffn.gated_linear_backward(a, a, b, b, a, a),
    lambda a, b: ffn.layer_norm(a), lambda a, b: ffn.layer_norm_backward(a, a, a[0], a[0]),
])
def test_python_refuses_cpu_tensors(call):
    a = torch.zeros(8, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="requires CUDA tensors"):
        call(a, a.t())


@pytest.mark.parametrize("call", [
    lambda: ffn.fused_linear(torch.zeros(2, 3), torch.zeros(4, 5)),
    lambda: ffn.fused_linear(torch.zeros(3), torch.zeros(3, 5)),
    lambda: ffn.fused_linear(torch.zeros(2, 3), torch.zeros(3, 5), activation="tanh"),
    lambda: ffn.fused_linear(torch.zeros(2, 3), torch.zeros(3, 5), activation=["silu"]),
    lambda: ffn.gated_linear(torch.zeros(2, 3), torch.zeros(3, 5), torch.zeros(2, 5)),
    lambda: ffn.layer_norm(torch.zeros(3)),
])
def test_python_refuses_shapes_and_names(call):
    with pytest.raises(ValueError):
        call()


def test_tracing_shapes():
    """The fake kernels give the shapes and memory orders of the real ones."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.gemm_lab
    with FakeTensorMode():
        a = torch.empty(6, 16, dtype=torch.float16)
        w, kn = torch.empty(24, 16, dtype=torch.float16).t(), torch.empty(16, 24, dtype=torch.float16)
        y, z = ops.fused_linear(a, w, None, "gelu", None)
        assert y.shape == z.shape == (6, 24)
        assert ops.fused_linear(a, w, None, None, None)[1].shape == (0,)
        da, db, dbias = ops.fused_linear_backward(y, a, w, z, "gelu", True, True, True)
        assert da.shape == a.shape and db.shape == w.shape and db.stride() == w.stride() and dbias.shape == (24,)
        assert ops.fused_linear_backward(y, a, kn, z, "gelu", True, True, True)[1].stride() == kn.stride()
        assert [t.shape for t in ops.gated_linear(a, w, kn, None, None, "silu")] == [(6, 24)] * 3
        assert [t.dtype for t in ops.layer_norm(a, None, None, 1e-5)] == [torch.float16, torch.float32, torch.float32]
        with pytest.raises(ValueError):
            ops.fused_linear(a, a, None, None, None)


def test_every_operator_is_documented_and_exported():
    for name in ffn.__all__:
        assert inspect.getdoc(getattr(ffn, name)), name


@pytest.mark.parametrize("name", [a for a in ref.ACTIVATIONS if a])
def test_reference_slopes_and_constants(name):
    z = torch.linspace(-12, 12, 4001, dtype=torch.float64)
    h = 1e-5
    slope = ref.act(z, name)[1]
    diff = (ref.act(z + h, name)[0] - ref.act(z - h, name)[0]) / (2 * h)
    away = z.abs() > 1e-3
    assert float((slope - diff)[away].abs().max()) < 1e-8
    assert float(slope.abs().max()) <= ref.SLOPE[name]
    if name != "relu":
        curve = (ref.act(z + h, name)[1] - ref.act(z - h, name)[1]) / (2 * h)
        assert float(curve.abs().max()) <= ref.CURVE[name]


def test_reference_gradients_against_autograd():
    gen = torch.Generator().manual_seed(0)

    def leaf(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64).requires_grad_()

    x, bg, bu, b0, b1, dy = leaf(5, 7), leaf(7, 6), leaf(7, 6), leaf(6), leaf(6), torch.randn(5, 6, generator=gen).double()
    for name in ref.ACTIVATIONS:
        h, g, u, *_ = ref.gated(x, bg, bu, b0, b1, name, torch.float16)
        want = torch.autograd.grad(h, (x, bg, bu, b0, b1), dy)
        da, db, dbias = ref.gated_backward(dy, x, bg, bu, g, u, name, torch.float16)
        for got, w in zip([da, *db, *dbias], want):
            assert torch.allclose(got[0], w, rtol=1e-12, atol=1e-12)
    w, b, dx = leaf(7), leaf(7), torch.randn(5, 7, generator=gen).double()
    y, mean, rstd, *_ = ref.layer_norm(x, w, b, 1e-5, torch.float16)
    want = torch.autograd.grad(y, (x, w, b), dx)
    for got, v in zip(ref.layer_norm_backward(dx, x, mean, rstd, w, torch.float16), want):
        assert torch.allclose(got[0], v, rtol=1e-12, atol=1e-12)
