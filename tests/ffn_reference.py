"""64-bit definitions of the feed-forward operators and the error bounds their tests hold the kernels to.

Every bound is a sum of what the kernels round: one half-step `unit` (2^-8 bfloat16, 2^-11 float16) per stored
16-bit value, and the 32-bit sums.  A sum of k products carries at most k + 1 roundings of a 32-bit accumulator
that may truncate (2^-23 each, of the sum of magnitudes); the activations add a few units of the 32-bit functions
they use (2^-19 of their argument's or value's size, far above exp's and the divide's documented errors).
"""
from __future__ import annotations

import math

import torch

ACTIVATIONS = [None, "silu", "gelu", "gelu_tanh", "relu"]
# Largest |act'| of each, rounded up.
SLOPE = {None: 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13, "relu": 1.0}
# Largest |act''|, rounded up (relu's slope is exact in the 16-bit argument).
CURVE = {None: 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.81, "relu": 0.0}


def unit(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half a step of the smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def act(z: torch.Tensor, name: str | None) -> tuple[torch.Tensor, torch.Tensor]:
    """(act(z), act'(z)), z float64."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def dot_error(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Bound on the 32-bit accumulation error of x @ y."""
    return (x.shape[1] + 1) * 2.0 ** -23 * (x.abs() @ y.abs())


def linear(a, b, bias, name, residual, dtype):
    """(y, z, bound of y, bound of z); operands float64."""
    z = a @ b
    err = dot_error(a, b)
    if bias is not None:
        z = z + bias
        err = err + 2.0 ** -23 * z.abs()
    v, _ = act(z, name)
    y = v if residual is None else v + residual
    u = unit(dtype)
    err_z = u * z.abs() + err * (1 + u) + tiny(dtype)
    err_v = SLOPE[name] * err + (0 if name is None else 2.0 ** -19 * (z.abs() + v.abs())) + 2.0 ** -23 * y.abs()
    return y, z, u * y.abs() + err_v * (1 + u) + tiny(dtype), err_z


def gated(a, bg, bu, bias_g, bias_u, name, dtype):
    """(h, gate, up, bounds of the three)."""
    _, g, _, eg = linear(a, bg, bias_g, None, None, dtype)
    _, v, _, ev = linear(a, bu, bias_u, None, None, dtype)
    value, _ = act(g, name)
    # 32-bit errors of the two sums (what linear() adds to the rounding).
    rg = dot_error(a, bg) + 2.0 ** -23 * g.abs()
    rv = dot_error(a, bu) + 2.0 ** -23 * v.abs()
    ra = SLOPE[name] * rg + (0 if name is None else 2.0 ** -19 * (g.abs() + value.abs()))
    h = value * v
    u = unit(dtype)
    err = ra * v.abs() + rv * value.abs() + ra * rv + 2.0 ** -23 * h.abs()
    return h, g, v, u * h.abs() + err * (1 + u) + tiny(dtype), eg, ev


def products_backward(dz_pairs, a, b_pairs, dtype):
    """(dA, [dB], [dbias]) and their bounds, from [(dz, 32-bit error of dz)]."""
    u = unit(dtype)
    da, ea = 0, 0
    db, eb, dbias, ebias = [], [], [], []
    for (dz, edz), b in zip(dz_pairs, b_pairs):
        e16 = u * dz.abs() + edz * (1 + u) + tiny(dtype)  # the rounded operand of the products
        da = da + dz @ b.t()
        ea = ea + e16 @ b.abs().t() + dot_error(dz.abs() + e16, b.t())
        w = a.t() @ dz
        ew = a.abs().t() @ e16 + dot_error(a.t(), dz.abs() + e16)
        db.append(w)
        eb.append(u * w.abs() + ew * (1 + u) + tiny(dtype))
        s = dz.sum(0)
        es = edz.sum(0) + (dz.shape[0] + 1) * 2.0 ** -23 * dz.abs().sum(0)
        dbias.append(s)
        ebias.append(u * s.abs() + es * (1 + u) + tiny(dtype))
    return (da, u * da.abs() + ea * (1 + u) + tiny(dtype)), list(zip(db, eb)), list(zip(dbias, ebias))


def linear_backward(dy, a, b, z, name, dtype):
    if name is None:
        dz, edz = dy, torch.zeros_like(dy)
    else:
        dz = dy * act(z, name)[1]
        edz = 2.0 ** -19 * dy.abs() * (2 + CURVE[name] * z.abs()) if name != "relu" else torch.zeros_like(dy)
    return products_backward([(dz, edz)], a, [b], dtype)


def gated_backward(dy, a, bg, bu, g, v, name, dtype):
    value, slope = act(g, name)
    dg, du = dy * v * slope, dy * value
    rel = 2.0 ** -19
    eg = rel * (dy * v).abs() * (2 + CURVE[name] * g.abs())
    eu = rel * dy.abs() * (value.abs() + g.abs())
    return products_backward([(dg, eg), (du, eu)], a, [bg, bu], dtype)


def layer_norm(x, w, b, eps, dtype):
    """(y, mean, rstd, bound of y, of mean, of rstd)."""
    n = x.shape[1]
    mean, var = x.mean(1, keepdim=True), x.var(1, unbiased=False, keepdim=True)
    rstd = (var + eps) ** -0.5
    xhat = (x - mean) * rstd
    # A row's 32-bit sums are trees of at most 64 sequential terms per thread and a few joins.
    steps = 2.0 ** -24 * 128
    e_mean = steps * x.abs().mean(1, keepdim=True)
    e_rstd = rstd * (steps + (e_mean * rstd) ** 2 + 2.0 ** -21)
    e_hat = e_mean * rstd + xhat.abs() * (e_rstd / rstd) + 2.0 ** -22 * (xhat.abs() + x.abs() * rstd)
    y = xhat if w is None else xhat * w
    e = e_hat if w is None else e_hat * w.abs()
    if b is not None:
        y = y + b
    e = e + 2.0 ** -22 * (y.abs() + xhat.abs() * (1 if w is None else w.abs()))
    u = unit(dtype)
    return y, mean[:, 0], rstd[:, 0], u * y.abs() + e * (1 + u) + tiny(dtype), e_mean[:, 0] + 1e-45, e_rstd[:, 0]


def layer_norm_backward(dy, x, mean, rstd, w, dtype):
    """((dx, bound), (dw, bound), (db, bound)); mean and rstd as given."""
    m, n = x.shape
    xhat = (x - mean[:, None]) * rstd[:, None]
    g = dy if w is None else dy * w
    c1, c2 = (g * xhat).mean(1, keepdim=True), g.mean(1, keepdim=True)
    dx = rstd[:, None] * (g - c2 - xhat * c1)
    steps = 2.0 ** -24 * 128
    e_hat = 2.0 ** -22 * (xhat.abs() + x.abs() * rstd[:, None])
    e1 = steps * (g * xhat).abs().mean(1, keepdim=True) + (g.abs() * e_hat).mean(1, keepdim=True)
    e2 = steps * g.abs().mean(1, keepdim=True)
    e = rstd[:, None] * (e2 + e_hat * c1.abs() + xhat.abs() * e1
                         + 2.0 ** -21 * (g.abs() + c2.abs() + (xhat * c1).abs()))
    u = unit(dtype)
    out = [(dx, u * dx.abs() + e * (1 + u) + tiny(dtype))]
    rows = (m + 1) * 2.0 ** -24
    for s, mag, extra in ((dy * xhat, (dy * xhat).abs(), dy.abs() * e_hat), (dy, dy.abs(), None)):
        total = s.sum(0)
        es = rows * mag.sum(0) + (0 if extra is None else extra.sum(0))
        out.append((total, u * total.abs() + es * (1 + u) + tiny(dtype)))
    return out


def within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    if not got.numel():
        return
    off = (got.double() - want).abs()
    bad = ~(off <= bound)  # NaN counts as bad
    if bad.any():
        i = int(torch.argmax(torch.where(torch.isnan(off), torch.full_like(off, math.inf), off / bound)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds; worst at flat index {i}: "
                             f"{float(got.reshape(-1)[i])} for {float(want.reshape(-1)[i])} "
                             f"+- {float(bound.reshape(-1)[i])}")
