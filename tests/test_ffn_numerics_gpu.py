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
