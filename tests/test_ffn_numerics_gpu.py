"""The feed-forward operators where their arithmetic is hardest: tails of the activations, huge and infinite values,
rows far off centre, empty rows, and the large products' dealt schedules with every epilogue."""
from __future__ import annotations

import math

import pytest
import torch

import ffn_reference as ref
from gemm_lab_qualification_b200 import _native as native
from gemm_lab_qualification_b200 import ffn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    native.device_error(clear=True)
    yield
    torch.cuda.synchronize()
    assert native.device_error(clear=True) == 0


def make(gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def d(t):
    return None if t is None else t.double()


def slope_of(z, name):
    """act'(z) as the bias gradient of one row whose output gradient is 1."""
    a, b = torch.ones((1, 8), dtype=z.dtype, device="cuda"), torch.ones((z.numel(), 8), dtype=z.dtype, device="cuda").t()
    return ffn.fused_linear_backward(torch.ones_like(z)[None], a, b, z[None], name, has_bias=True, need_a=False,
                                     need_b=False)[2]


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_slopes_of_huge_inputs(name):
    """1 and 0 up to the largest finite values, whose squares and cubes overflow 32 bits."""
    huge = torch.tensor([30.0, 1e4, 1e10, 1e13, 1e18, 1.8e19, 1.9e19, 1e25, 3e38], dtype=torch.float64)
    z = torch.cat([huge, -huge]).to(BF16).cuda()
    want = (z > 0).double()
    # One half-step, and 2^-19 for the 32-bit functions; the slopes' own distance from 1 and 0 at 30 is below 1e-11.
    bound = ref.unit(BF16) * want + 2.0 ** -19
    ref.within(slope_of(z, name), want, bound, name)
    a, b = torch.ones((1, 8), dtype=BF16, device="cuda"), torch.ones((z.numel(), 8), dtype=BF16, device="cuda").t()
    one = torch.ones_like(z)[None]
    dbias = ffn.gated_linear_backward(one, a, b, b, z[None], one, name, has_bias=True, need_a=False, need_b=False)[3]
    ref.within(dbias, want, bound, name)


# Relative error of the 32-bit exact GELU's tail: its polynomial (2^-19 with its evaluation), the reciprocal and three
# products (2^-21 together), and the exponential of -z^2/2, documented as 2 + 1.173 z^2 / 2 units of 2^-23, with the
# rounding of z^2: below 2^-18 + 2^-23 z^2; twice the second term is allowed.
def tail_error(z):
    return 2.0 ** -18 + 2.0 ** -22 * z * z


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("m", [1, 20, 300])
def test_exact_gelu_tail(m, dtype):
    """Negative inputs, where the value is far smaller than its argument: bounds relative to the value.  The products
    are exact (one term each), so the argument is the 16-bit z itself."""
    z = torch.linspace(-13, -0.5, 2048, dtype=torch.float64).to(dtype).cuda()
    a, w = torch.zeros((m, 8), dtype=dtype, device="cuda"), torch.zeros((z.numel(), 8), dtype=dtype, device="cuda")
    a[:, 0] = 1.0
    w[:, 0] = z
    ones = torch.zeros_like(w)
    ones[:, 0] = 1.0
    zz = z.double()
    want = ref.act(zz, "gelu")[0]
    bound = (ref.unit(dtype) + tail_error(zz) * (1 + ref.unit(dtype))) * want.abs() + ref.tiny(dtype)
    for y in (ffn.fused_linear(a, w.t(), activation="gelu"), ffn.gated_linear(a, w.t(), ones.t(), activation="gelu")):
        ref.within(y, want.expand(m, -1), bound.expand(m, -1), "gelu")


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_exact_gelu_slope_tail(dtype):
    z = torch.linspace(-13, -0.5, 2048, dtype=torch.float64).to(dtype).cuda()
    zz = z.double()
    parts = 0.5 * torch.erfc(-zz / math.sqrt(2)) + zz.abs() * torch.exp(-zz * zz / 2) / math.sqrt(2 * math.pi)
    want = ref.act(zz, "gelu")[1]
    bound = ref.unit(dtype) * want.abs() + tail_error(zz) * (1 + ref.unit(dtype)) * parts + ref.tiny(dtype)
    ref.within(slope_of(z, "gelu"), want, bound, "slope")
    # In the gated backward pass, the value goes into the up projection's gradient.
    a, b = torch.ones((1, 8), dtype=dtype, device="cuda"), torch.ones((z.numel(), 8), dtype=dtype, device="cuda").t()
    one = torch.ones_like(z)[None]
    dup = ffn.gated_linear_backward(one, a, b, b, z[None], one, "gelu", has_bias=True, need_a=False, need_b=False)[4]
    value = ref.act(zz, "gelu")[0]
    ref.within(dup, value, (ref.unit(dtype) + tail_error(zz) * (1 + ref.unit(dtype))) * value.abs() + ref.tiny(dtype),
               "value")


@pytest.mark.parametrize("name", [a for a in ref.ACTIVATIONS if a])
@pytest.mark.parametrize("m", [1, 20, 300])
def test_activations_of_the_largest_values(m, name):
    """Infinity, the largest finite values and NaN (exact products of one term)."""
    big = float(torch.finfo(BF16).max)
    z = torch.tensor([math.inf, big, 2.0 ** 100, -big, -(2.0 ** 100), math.nan], dtype=BF16, device="cuda")
    a, w = torch.zeros((m, 8), dtype=BF16, device="cuda"), torch.zeros((z.numel(), 8), dtype=BF16, device="cuda")
    a[:, 0] = 1.0
    w[:, 0] = z
    y = ffn.fused_linear(a, w.t(), activation=name)
    assert torch.equal(y[:, :3], z[:3].expand(m, 3)) and float(y[:, 3:5].abs().max()) == 0.0
    assert bool(torch.isnan(y[:, 5]).all())


@pytest.mark.parametrize("m,n", [(5, 256), (9, 1000), (40, 1001), (300, 4096), (40, 4095), (6, 8200), (4, 16384),
                                 (3, 16392), (2, 20001)])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_layer_norm_backward_far_off_centre(m, n, dtype):
    """Rows whose mean is hundreds of deviations (constant rows: any number) away from zero.  x - mean has one
    rounding, so the bound is the one of the centred row."""
    gen = torch.Generator().manual_seed(m + n)
    step = 1000 * torch.finfo(dtype).eps
    x = (1000 + torch.randint(-2, 3, (m, n), generator=gen) * step).to(dtype)
    x[0] = 1000.0
    x = x.cuda()
    w, dy = make(gen, dtype, n, scale=0.2) + 1, make(gen, dtype, m, n)
    mean = x.double().mean(1)
    rstd = (x.double().var(1, unbiased=False) + 1e-5).rsqrt()
    mean, rstd = mean.float(), rstd.float()
    got = ffn.layer_norm_backward(dy, x, mean, rstd, w, has_bias=True)
    want = ref.layer_norm_backward(d(dy), d(x) - d(mean)[:, None], torch.zeros_like(d(mean)), d(rstd), d(w), dtype)
    for g, (v, bound), what in zip(got, want, ("dx", "dw", "db")):
        ref.within(g, v, bound, what)


@pytest.mark.parametrize("n", [100, 251, 513, 1001, 2047, 4095, 8190, 12001, 20001])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_layer_norm_of_constant_rows(n, dtype):
    """Every partial sum of rows of 1000 or 7 is exact, and so is their quotient by n: deviations are exactly zero
    (one last bit of the mean would come out as 1000 * 2^-24 * 316, far above the bias)."""
    x = torch.tensor([[1000.0], [7.0], [-1000.0]], dtype=dtype, device="cuda").expand(3, n).contiguous()
    bias = torch.linspace(-1, 1, n).to(dtype).cuda()
    y, mean, rstd = ffn.layer_norm(x, None, bias, 1e-5, return_stats=True)
    assert torch.equal(mean, x[:, 0].float())
    assert torch.equal(y, bias.expand(3, n))
    assert float((rstd.double() * math.sqrt(1e-5) - 1).abs().max()) <= 2.0 ** -21


@pytest.mark.parametrize("n", [264, 4095, 20001])
def test_statistics_of_infinite_rows(n):
    x = torch.zeros((3, n), dtype=BF16, device="cuda")
    x[0, 5], x[1, 6], x[2, 7] = math.inf, -math.inf, math.nan
    y, mean, _ = ffn.layer_norm(x, return_stats=True)
    assert float(mean[0]) == math.inf and float(mean[1]) == -math.inf and math.isnan(float(mean[2]))
    assert not bool(torch.isfinite(y).any())


def test_statistics_of_empty_rows():
    """The mean of no values is 0 / 0, and so is their variance: not what the memory held before."""
    torch.full((3,), 7.0, device="cuda")  # the block that the statistics will take
    torch.full((3,), 7.0, device="cuda")
    y, mean, rstd = ffn.layer_norm(torch.empty((3, 0), dtype=F16, device="cuda"), return_stats=True)
    assert y.shape == (3, 0) and bool(torch.isnan(mean).all()) and bool(torch.isnan(rstd).all())


SLOT = 2 * 128 * 256 * 4 + 2 * 8 * 8  # workspace of a dealt run: a pair's partial tile and its flags


def runs_of(op, a, bs, n):
    """Dealt runs of a forward call on aligned operands in whole sectors: what its workspace is for."""
    m, k = a.shape
    args = [int(a.dtype == BF16), a.data_ptr(), k, 1]
    for b in bs:
        args += [b.data_ptr(), b.stride(0), b.stride(1)]
    size = getattr(native.library(), f"glq_{op}_workspace_bytes")(*args, m, n, k)
    runs = size // SLOT
    assert size == (runs * SLOT + 255) // 256 * 256
    return runs


@pytest.mark.parametrize("m,n,k,act,order,dtype", [
    (500, 10240, 8192, "gelu", "nk", BF16),  # 80 tiles: 74 whole, the blocks of 6 dealt
    (700, 6500, 8192, "silu", "nk", F16),    # rows off 16 bytes: stored element by element
    (300, 9808, 8192, None, "kn", BF16),
])
def test_dealt_remainder_of_a_linear_layer(m, n, k, act, order, dtype):
    """Whole tiles first, then runs joined through the workspace, with bias, activation, residual and kept z."""
    gen = torch.Generator().manual_seed(n)
    a, bias, res = make(gen, dtype, m, k), make(gen, dtype, n), make(gen, dtype, m, n)
    b = make(gen, dtype, n, k, scale=k ** -0.5).t() if order == "nk" else make(gen, dtype, k, n, scale=k ** -0.5)
    assert runs_of("fused_linear", a, (b,), n) > 0
    y, z = ffn.fused_linear(a, b, bias, act, res, return_preact=True)
    wy, wz, ey, ez = ref.linear(d(a), d(b), d(bias), act, d(res), dtype)
    ref.within(y, wy, ey, "y")
    ref.within(z, wz, ez, "z")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ffn.fused_linear(a, b, bias, act, res)
    for _ in range(3):
        again.zero_()
        graph.replay()
        assert torch.equal(again, y)


@pytest.mark.parametrize("m,n,k,dtype", [
    (500, 8192, 11008, BF16),  # 128 tiles: 74 whole, 54 dealt to every pair
    (300, 5004, 8192, F16),    # few pairs have a run; rows off 16 bytes
])
def test_dealt_remainder_of_a_gated_pair(m, n, k, dtype):
    gen = torch.Generator().manual_seed(n)
    a, bias_g, bias_u = make(gen, dtype, m, k), make(gen, dtype, n), make(gen, dtype, n)
    bg, bu = (make(gen, dtype, n, k, scale=k ** -0.5).t() for _ in range(2))
    assert runs_of("gated_linear", a, (bg, bu), n) > 0
    h, g, u = ffn.gated_linear(a, bg, bu, bias_g, bias_u, "gelu_tanh", return_preact=True)
    wh, wg, wu, eh, eg, eu = ref.gated(d(a), d(bg), d(bu), d(bias_g), d(bias_u), "gelu_tanh", dtype)
    for got, want, bound in ((h, wh, eh), (g, wg, eg), (u, wu, eu)):
        ref.within(got, want, bound, "gated")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ffn.gated_linear(a, bg, bu, bias_g, bias_u, "gelu_tanh")
    for _ in range(3):
        again.zero_()
        graph.replay()
        assert torch.equal(again, h)


@pytest.mark.parametrize("m", [20, 300])
def test_non_finite_gradients_stay_in_their_rows(m):
    gen = torch.Generator().manual_seed(3)
    n, k = 136, 200
    a, z, u, dy = make(gen, F16, m, k), make(gen, F16, m, n), make(gen, F16, m, n), make(gen, F16, m, n)
    b, b2 = (make(gen, F16, n, k, scale=k ** -0.5).t() for _ in range(2))
    _, mean, rstd = ffn.layer_norm(z, return_stats=True)

    def input_gradients(dy):
        return [ffn.fused_linear_backward(dy, a, b, z, "silu")[0], ffn.gated_linear_backward(dy, a, b, b2, z, u, "gelu")[0],
                ffn.layer_norm_backward(dy, z, mean, rstd)[0]]

    clean = input_gradients(dy)
    dy[7, 3], dy[11, 5] = float("nan"), float("inf")
    keep = [i for i in range(m) if i not in (7, 11)]
    for got, was in zip(input_gradients(dy), clean):
        assert bool(torch.isnan(got[7]).all()) and not bool(torch.isfinite(got[11]).all())
        assert torch.equal(got[keep], was[keep])
    # A column's sum sees what is in its column alone.
    dbias = ffn.fused_linear_backward(dy, a, b, z, "silu", has_bias=True, need_a=False, need_b=False)[2]
    assert [i for i in range(n) if not math.isfinite(float(dbias[i]))] == [3, 5]


@pytest.mark.parametrize("n", [264, 1001])
def test_layer_norm_near_the_largest_float16(n):
    gen = torch.Generator().manual_seed(n)
    x = (torch.randint(0, 2, (6, n), generator=gen) * 2.0 - 1.0).mul(65504.0).to(F16).cuda()
    x[1] = 65504.0
    x[2] = 2.0 ** -24
    w, b, dy = make(gen, F16, n, scale=0.2) + 1, make(gen, F16, n), make(gen, F16, 6, n)
    y, mean, rstd = ffn.layer_norm(x, w, b, 1e-5, return_stats=True)
    wy, wm, wr, ey, em, er = ref.layer_norm(d(x), d(w), d(b), 1e-5, F16)
    ref.within(mean, wm, em, "mean")
    ref.within(rstd, wr, er, "rstd")
    ref.within(y, wy, ey, "y")
    got = ffn.layer_norm_backward(dy, x, mean, rstd, w, has_bias=True)
    for g, (v, bound) in zip(got, ref.layer_norm_backward(d(dy), d(x), d(mean), d(rstd), d(w), F16)):
        ref.within(g, v, bound, "gradient")
