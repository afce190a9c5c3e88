"""Timed cases of the feed-forward operators: the linear layer with bias, activation and residual, the gated
linear pair and layer norm, each forward and backward.

`own` False runs the plain forms (32-bit elementary torch operations); `own` True makes the calls that a user of
`gemm_lab_qualification_b200.ffn` makes.  Weights are W [N, K] (layout "nk", handed over as W.t()) or the lab's
B [K, N] (layout "kn").
"""
import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # One token through a square layer with bias, SiLU and residual: latency counts.
        dict(name="linear_m1", op="linear", m=1, n=4096, k=4096, dtype="float16", act="silu", bias=True,
             residual=True, layout="nk"),
        # The down-projection of a decode batch, added to the residual stream.
        dict(name="linear_m32_down", op="linear", m=32, n=4096, k=11008, dtype="bfloat16", act="none", bias=False,
             residual=True, layout="nk"),
        # The same down-projection over a prompt.
        dict(name="linear_m4096_down", op="linear", m=4096, n=4096, k=11008, dtype="bfloat16", act="none",
             bias=False, residual=True, layout="nk"),
        # A small training batch through a biased GELU layer; ragged tokens and output columns.
        dict(name="linear_bwd_ragged", op="linear_bwd", m=999, n=4100, k=1032, dtype="float16", act="gelu",
             bias=True, residual=False, layout="nk"),
        # One token through the gated pair.
        dict(name="gated_m1", op="gated", m=1, n=11008, k=4096, dtype="float16", act="silu", bias=False,
             layout="nk"),
        # A decode batch through the widest gated pair.
        dict(name="gated_m32_wide", op="gated", m=32, n=28672, k=8192, dtype="bfloat16", act="silu", bias=False,
             layout="nk"),
        # A short prompt through an odd-sized biased GEGLU pair stored as the lab's B [K, N].
        dict(name="gated_ragged_kn", op="gated", m=131, n=2736, k=1000, dtype="float16", act="gelu", bias=True,
             layout="kn"),
        # Training forward of the gated pair: the pre-activations are kept for the backward pass.
        dict(name="gated_train", op="gated_train", m=4096, n=11008, k=4096, dtype="bfloat16", act="silu",
             bias=False, layout="nk"),
        # Its backward pass: gradients of the input and of both weights.
        dict(name="gated_bwd", op="gated_bwd", m=4096, n=11008, k=4096, dtype="bfloat16", act="silu", bias=False,
             layout="nk"),
        # The norm in front of a decode step.
        dict(name="norm_m32", op="norm", m=32, n=4096, dtype="float16", affine=True),
        # The norm over a long batch, with the statistics that training keeps.
        dict(name="norm_train", op="norm_train", m=16384, n=8192, dtype="bfloat16", affine=True),
        # Its backward pass with the gradients of weight and bias.
        dict(name="norm_bwd", op="norm_bwd", m=8192, n=4096, dtype="bfloat16", affine=True),
    ]


def _log_size(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_bwd", "gated", "gated", "gated_train", "gated_bwd", "norm",
                     "norm_train", "norm_bwd"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op.startswith("norm"):
        n = _log_size(rng, 64, 16384)
        if rng.random() < 0.7:
            n = max(8, n // 8 * 8)
        m = _log_size(rng, 1, min(16384, (1 << 27) // n))
        return dict(op=op, m=m, n=n, dtype=dtype, affine=rng.random() < 0.85)
    gated = op.startswith("gated")
    n, k = _log_size(rng, 256, 28672), _log_size(rng, 256, 11008)
    kind = rng.random()
    if kind < 0.55:
        n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
    elif kind < 0.85:
        n, k = n // 8 * 8, k // 8 * 8
    limit = 1.0e12 / (n * k * (2 if not op.endswith("bwd") else 4) * (2 if gated else 1))
    m = _log_size(rng, 1, max(1, min(4096, limit)))
    case = dict(op=op, m=m, n=n, k=k, dtype=dtype, act=rng.choice(["silu", "gelu", "gelu_tanh", "relu"]),
                bias=rng.random() < 0.5, layout=rng.choice(["nk", "nk", "nk", "kn"]))
    if not gated:
        case["residual"] = op == "linear" and rng.random() < 0.6
        if rng.random() < 0.3:
            case["act"] = "none"
    return case


def work(case):
    m, n = case["m"], case["n"]
    op = case["op"]
    if op.startswith("norm"):
        vectors = 2 * n * (3 if op == "norm_bwd" else 2) if case["affine"] else 0
        tensors = {"norm": 4, "norm_train": 4, "norm_bwd": 6}[op] * m * n
        stats = 0 if op == "norm" else 8 * m
        return {"bytes": tensors + vectors + stats, "flops": (8 if op != "norm_bwd" else 16) * m * n}
    k = case["k"]
    pair = 2 if op.startswith("gated") else 1
    bias = 2 * n * pair if case["bias"] else 0
    if op.endswith("bwd"):
        # dy, the kept pre-activations, A and the weights in; dA, the weights' and biases' gradients out.
        kept = pair * m * n if case["act"] != "none" or pair == 2 else 0
        elements = m * n + kept + m * k + pair * n * k + m * k + pair * n * k
        return {"bytes": 2 * elements + bias, "flops": 4 * pair * m * n * k}
    outs = 3 if op == "gated_train" else 1
    elements = m * k + pair * n * k + outs * m * n + (m * n if case.get("residual") else 0)
    return {"bytes": 2 * elements + bias, "flops": 2 * pair * m * n * k}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0, shift=0.0):
        v = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
        return v if scale == 1.0 and shift == 0.0 else v.mul_(scale).add_(shift)

    m, n, op = case["m"], case["n"], case["op"]
    state = {"case": case}
    if op.startswith("norm"):
        # A residual stream: unit scale, off centre.
        state["x"] = normal(m, n, scale=1.3, shift=0.4)
        if case["affine"]:
            state["weight"] = normal(n, scale=0.1, shift=1.0)
            state["bias"] = normal(n, scale=0.1)
        if op == "norm_bwd":
            state["dy"] = normal(m, n)
            x = state["x"].double()
            state["mean"] = x.mean(1).float()
            state["rstd"] = (x.var(1, unbiased=False) + EPS).rsqrt().float()
        return state
    k = case["k"]

    def weight():
        w = normal(n, k, scale=k ** -0.5) if case["layout"] == "nk" else normal(k, n, scale=k ** -0.5)
        return w.t() if case["layout"] == "nk" else w

    state["x"] = normal(m, k)
    state["b"] = weight()
    if op.startswith("gated"):
        state["b_up"] = weight()
    if case["bias"]:
        state["bias"] = normal(n, scale=0.2)
        if op.startswith("gated"):
            state["bias_up"] = normal(n, scale=0.2)
    if case.get("residual"):
        state["residual"] = normal(m, n)
    if op.endswith("bwd"):
        state["dy"] = normal(m, n)
        if op == "gated_bwd":
            state["gate"], state["up"] = normal(m, n), normal(m, n)
        elif case["act"] != "none":
            state["z"] = normal(m, n)
    return state


# ---------------------------------------------------------------- plain forms (32 bits)

def _act(z, name):
    if name == "none":
        return z
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    if name == "gelu_tanh":
        return z / (1.0 + torch.exp(-1.5957691216057308 * (z + 0.044715 * z * z * z)))
    return torch.where(z > 0, z, torch.zeros_like(z))


def _act_grad(z, name):
    if name == "none":
        return torch.ones_like(z)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        return (0.5 * (1.0 + torch.erf(z * 0.7071067811865476))
                + z * 0.3989422804014327 * torch.exp(-0.5 * z * z))
    if name == "gelu_tanh":
        s = 1.0 / (1.0 + torch.exp(-1.5957691216057308 * (z + 0.044715 * z * z * z)))
        return s + z * s * (1.0 - s) * 1.5957691216057308 * (1.0 + 0.134145 * z * z)
    return (z > 0).to(z.dtype)


def _plain(state):
    case = state["case"]
    op, act = case["op"], case.get("act")
    x = state["x"].float()
    dtype = state["x"].dtype
    if op in ("norm", "norm_train"):
        mean = x.sum(1, keepdim=True) / x.shape[1]
        centred = x - mean
        rstd = 1.0 / torch.sqrt((centred * centred).sum(1, keepdim=True) / x.shape[1] + EPS)
        y = centred * rstd
        if case["affine"]:
            y = y * state["weight"].float() + state["bias"].float()
        y = y.to(dtype)
        return [y] if op == "norm" else [y, mean[:, 0], rstd[:, 0]]
    if op == "norm_bwd":
        dy = state["dy"].float()
        rstd = state["rstd"][:, None]
        xhat = (x - state["mean"][:, None]) * rstd
        wdy = dy * state["weight"].float() if case["affine"] else dy
        c1 = (wdy * xhat).sum(1, keepdim=True) / x.shape[1]
        c2 = wdy.sum(1, keepdim=True) / x.shape[1]
        dx = ((wdy - c2 - xhat * c1) * rstd).to(dtype)
        return [dx, (dy * xhat).sum(0).to(dtype), dy.sum(0).to(dtype)] if case["affine"] else [dx]
    b = state["b"].float()
    if op == "linear":
        z = x @ b
        if case["bias"]:
            z = z + state["bias"].float()
        y = _act(z, act)
        if case["residual"]:
            y = y + state["residual"].float()
        return [y.to(dtype)]
    if op == "linear_bwd":
        dz = state["dy"].float()
        if act != "none":
            dz = dz * _act_grad(state["z"].float(), act)
        out = [(dz @ b.t()).to(dtype), (x.t() @ dz).to(dtype)]
        return out + [dz.sum(0).to(dtype)] if case["bias"] else out
    b_up = state["b_up"].float()
    if op in ("gated", "gated_train"):
        gate, up = x @ b, x @ b_up
        if case["bias"]:
            gate, up = gate + state["bias"].float(), up + state["bias_up"].float()
        h = (_act(gate, act) * up).to(dtype)
        return [h] if op == "gated" else [h, gate.to(dtype), up.to(dtype)]
    dy, gate, up = state["dy"].float(), state["gate"].float(), state["up"].float()
    dgate, dup = dy * up * _act_grad(gate, act), dy * _act(gate, act)
    out = [(dgate @ b.t() + dup @ b_up.t()).to(dtype), (x.t() @ dgate).to(dtype), (x.t() @ dup).to(dtype)]
    return out + [dgate.sum(0).to(dtype), dup.sum(0).to(dtype)] if case["bias"] else out


# ---------------------------------------------------------------- the framework's calls

def _own(state):
    from gemm_lab_qualification_b200 import ffn

    case = state["case"]
    op, x = case["op"], state["x"]
    if op == "norm":
        return [ffn.layer_norm(x, state.get("weight"), state.get("bias"), EPS)]
    if op == "norm_train":
        return list(ffn.layer_norm(x, state.get("weight"), state.get("bias"), EPS, return_stats=True))
    if op == "norm_bwd":
        out = ffn.layer_norm_backward(state["dy"], x, state["mean"], state["rstd"], state.get("weight"),
                                      has_bias=case["affine"])
        return [v for v in out if v is not None]
    act = None if case["act"] == "none" else case["act"]
    if op == "linear":
        return [ffn.fused_linear(x, state["b"], state.get("bias"), act, state.get("residual"))]
    if op == "linear_bwd":
        out = ffn.fused_linear_backward(state["dy"], x, state["b"], state.get("z"), act, has_bias=case["bias"])
        return [v for v in out if v is not None]
    if op in ("gated", "gated_train"):
        out = ffn.gated_linear(x, state["b"], state["b_up"], state.get("bias"), state.get("bias_up"), act,
                               return_preact=op == "gated_train")
        return [out] if op == "gated" else list(out)
    out = ffn.gated_linear_backward(state["dy"], x, state["b"], state["b_up"], state["gate"], state["up"], act,
                                    has_bias=case["bias"])
    return [v for v in out if v is not None]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _act64(z, name):
    """(act(z), act'(z)) from the textbook definitions."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def exact(case, seed):
    state = {key: v.double() if isinstance(v, torch.Tensor) else v for key, v in prepare(case, seed).items()}
    op, x = case["op"], state["x"]
    if op.startswith("norm"):
        weight = state.get("weight", torch.ones(case["n"], dtype=torch.float64, device=x.device))
        if op == "norm_bwd":
            dy, rstd = state["dy"], state["rstd"].unsqueeze(1)
            xhat = (x - state["mean"].unsqueeze(1)) * rstd
            t = dy * weight
            dx = rstd * (t - t.mean(1, True) - xhat * (t * xhat).mean(1, True))
            if not case["affine"]:
                return [dx]
            return [dx, torch.einsum("mn,mn->n", dy, xhat), dy.sum(0)]
        mean, var = x.mean(1), x.var(1, unbiased=False)
        rstd = (var + EPS) ** -0.5
        y = (x - mean.unsqueeze(1)) * rstd.unsqueeze(1) * weight
        if case["affine"]:
            y = y + state["bias"]
        return [y] if op == "norm" else [y, mean, rstd]
    b = state["b"]
    if op == "linear":
        y = _act64(torch.mm(x, b) + state.get("bias", 0.0), case["act"])[0]
        return [y + state.get("residual", 0.0)]
    if op == "linear_bwd":
        dz = state["dy"] * _act64(state["z"], case["act"])[1] if case["act"] != "none" else state["dy"]
        out = [torch.mm(dz, b.t()), torch.mm(x.t(), dz)]
        return out + [dz.sum(0)] if case["bias"] else out
    if op in ("gated", "gated_train"):
        gate = torch.mm(x, b) + state.get("bias", 0.0)
        up = torch.mm(x, state["b_up"]) + state.get("bias_up", 0.0)
        h = _act64(gate, case["act"])[0] * up
        return [h] if op == "gated" else [h, gate, up]
    act, slope = _act64(state["gate"], case["act"])
    dgate, dup = state["dy"] * state["up"] * slope, state["dy"] * act
    out = [torch.mm(dgate, b.t()) + torch.mm(dup, state["b_up"].t()), torch.mm(x.t(), dgate), torch.mm(x.t(), dup)]
    return out + [dgate.sum(0), dup.sum(0)] if case["bias"] else out
