"""The feed-forward operators on a B200 against their 64-bit definitions.

Bounds come from ffn_reference (one half-step per stored 16-bit value plus the 32-bit sums).  Integer-valued
operands small enough that every sum is exact are compared bit for bit, and give exact differences for the
gradients of the (bi)linear forms.
"""
from __future__ import annotations

import pytest
import torch

import ffn_reference as ref
from gemm_lab_qualification_b200 import _native as native
from gemm_lab_qualification_b200 import ffn, kernels

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


def weight(gen, dtype, k, n, layout):
    """A [K, N] operand: W.t(), row-major [K, N], either in padded rows, or neither dimension contiguous."""
    s = k ** -0.5 if k else 1.0
    if layout == "nk":
        return make(gen, dtype, n, k, scale=s).t()
    if layout == "kn":
        return make(gen, dtype, k, n, scale=s)
    if layout == "nk_padded":
        return make(gen, dtype, n, (k + 7) // 8 * 8 + 16, scale=s)[:, :k].t()
    if layout == "kn_padded":
        return make(gen, dtype, k, (n + 7) // 8 * 8 + 8, scale=s)[:, :n]
    if layout == "nk_offset":  # base two bytes off
        return make(gen, dtype, n * k + 1, scale=s)[1:].view(n, k).t()
    if layout == "strided":
        return make(gen, dtype, n, 2 * k, scale=s)[:, ::2].t()
    raise ValueError(layout)


def rows(gen, dtype, m, n, layout="plain"):
    if layout == "plain":
        return make(gen, dtype, m, n)
    if layout == "padded":
        return make(gen, dtype, m, (n + 7) // 8 * 8 + 8)[:, :n]
    if layout == "odd":  # rows off 16 bytes
        return make(gen, dtype, m, n + 3)[:, 1:n + 1]
    if layout == "transposed":
        return make(gen, dtype, n, m).t()
    raise ValueError(layout)


def d(t):
    return None if t is None else t.double()


# Sizes: one token, every token tile and one past it, ragged and odd columns and contractions, several row tiles of
# the pair kernel, more K blocks than its ring, split contractions.
SIZES = [(1, 64, 64), (1, 1000, 4096), (2, 31, 13), (3, 72, 40), (8, 136, 200), (16, 200, 1032), (17, 257, 131),
         (32, 1032, 520), (33, 40, 2056), (64, 128, 320), (65, 300, 72), (100, 8, 1), (127, 1, 64), (128, 520, 264),
         (129, 257, 65), (200, 384, 512), (256, 256, 64), (257, 136, 136), (300, 1000, 1000), (513, 264, 1544),
         (600, 2056, 128), (1025, 65, 520), (160, 1000, 520), (192, 264, 1032), (193, 72, 200)]
W_LAYOUTS = ["nk", "kn", "nk_padded", "kn_padded", "nk_offset", "strided"]
A_LAYOUTS = ["plain", "padded", "odd", "transposed"]


def variants():
    """Sizes with the other choices dealt round, so every choice meets small and large sizes."""
    out = []
    for i, size in enumerate(SIZES):
        out.append((size, BF16 if i % 2 else F16, ref.ACTIVATIONS[i % 5], W_LAYOUTS[i % 6], A_LAYOUTS[(i // 2) % 4]))
        j = i + 2
        out.append((size, F16 if i % 2 else BF16, ref.ACTIVATIONS[(i + 2) % 5], W_LAYOUTS[j % 2], "plain"))
    return out


IDS = [f"m{s[0]}-n{s[1]}-k{s[2]}-{str(t)[6:]}-{a}-{w}-{x}" for s, t, a, w, x in variants()]


@pytest.mark.parametrize("case", variants(), ids=IDS)
def test_fused_linear(case):
    (m, n, k), dtype, act, wl, al = case
    gen = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    a, b = rows(gen, dtype, m, k, al), weight(gen, dtype, k, n, wl)
    bias, res = make(gen, dtype, n, scale=0.3), rows(gen, dtype, m, n, "odd" if m % 2 else "plain")
    for bi, r in ((bias, res), (None, None), (bias, None), (None, res)):
        y, z = ffn.fused_linear(a, b, bi, act, r, return_preact=True)
        wy, wz, ey, ez = ref.linear(d(a), d(b), d(bi), act, d(r), dtype)
        ref.within(y, wy, ey, "y")
        ref.within(z, wz, ez, "z")
        assert torch.equal(y, ffn.fused_linear(a, b, bi, act, r))  # the same bits without z


@pytest.mark.parametrize("case", variants(), ids=IDS)
def test_gated_linear(case):
    (m, n, k), dtype, act, wl, al = case
    gen = torch.Generator().manual_seed(m + n * 5 + k * 11)
    a, bg = rows(gen, dtype, m, k, al), weight(gen, dtype, k, n, wl)
    bu = weight(gen, dtype, k, n, "kn" if m % 3 == 0 else wl)  # sometimes of another order
    bias_g, bias_u = make(gen, dtype, n, scale=0.3), make(gen, dtype, n, scale=0.3)
    for b0, b1 in ((bias_g, bias_u), (None, None), (None, bias_u)):
        h, g, u = ffn.gated_linear(a, bg, bu, b0, b1, act, return_preact=True)
        wh, wg, wu, eh, eg, eu = ref.gated(d(a), d(bg), d(bu), d(b0), d(b1), act, dtype)
        ref.within(g, wg, eg, "gate")
        ref.within(u, wu, eu, "up")
        ref.within(h, wh, eh, "h")
        assert torch.equal(h, ffn.gated_linear(a, bg, bu, b0, b1, act))


@pytest.mark.parametrize("case", variants(), ids=IDS)
def test_fused_linear_backward(case):
    (m, n, k), dtype, act, wl, al = case
    gen = torch.Generator().manual_seed(m * 3 + n + k * 13)
    a, b = rows(gen, dtype, m, k, al), weight(gen, dtype, k, n, wl)
    dy, z = rows(gen, dtype, m, n, "odd" if n % 3 == 0 else "plain"), rows(gen, dtype, m, n)
    da, db, dbias = ffn.fused_linear_backward(dy, a, b, z if act else None, act, has_bias=True)
    wa, (wb,), (wbias,) = ref.linear_backward(d(dy), d(a), d(b), d(z), act, dtype)
    ref.within(da, *wa, "da")
    ref.within(db, *wb, "db")
    ref.within(dbias, *wbias, "dbias")
    if wl in ("nk", "kn"):
        assert db.stride() == b.stride()
    only = ffn.fused_linear_backward(dy, a, b, z if act else None, act, need_b=False)
    # (the cut of the sums, and so their last bits, depend on what is asked for together)
    ref.within(only[0], *wa, "da alone")
    assert only[1] is None and only[2] is None
    only = ffn.fused_linear_backward(dy, a, b, z if act else None, act, need_a=False)
    ref.within(only[1], *wb, "db alone")
    assert only[0] is None


@pytest.mark.parametrize("case", variants(), ids=IDS)
def test_gated_linear_backward(case):
    (m, n, k), dtype, act, wl, al = case
    gen = torch.Generator().manual_seed(m * 5 + n * 2 + k)
    a, bg = rows(gen, dtype, m, k, al), weight(gen, dtype, k, n, wl)
    bu = weight(gen, dtype, k, n, "kn" if m % 3 == 0 else wl)
    dy, g, u = rows(gen, dtype, m, n), rows(gen, dtype, m, n), rows(gen, dtype, m, n, "odd" if n % 3 == 0 else "plain")
    da, dbg, dbu, dbias_g, dbias_u = ffn.gated_linear_backward(dy, a, bg, bu, g, u, act, has_bias=True)
    wa, wb, wbias = ref.gated_backward(d(dy), d(a), d(bg), d(bu), d(g), d(u), act, dtype)
    ref.within(da, *wa, "da")
    for got, want in zip((dbg, dbu, dbias_g, dbias_u), wb + wbias):
        ref.within(got, *want, "weight or bias gradient")


def integers(gen, dtype, *shape, high=3):
    return torch.randint(-high, high + 1, shape, generator=gen).to(dtype).cuda()


@pytest.mark.parametrize("m,n,k", [(5, 72, 104), (40, 136, 72), (300, 200, 136)])
@pytest.mark.parametrize("layout", ["nk", "kn"])
def test_exact_integers_and_differences(m, n, k, layout):
    """Sums below 2^11 are exact in float16: values bit for bit, and the gradients of the (bi)linear forms equal
    exact differences of the forward kernels."""
    gen = torch.Generator().manual_seed(m + n)
    a, e = integers(gen, F16, m, k), integers(gen, F16, m, k, high=1)

    def w():
        return integers(gen, F16, n, k, high=1).t() if layout == "nk" else integers(gen, F16, k, n, high=1)

    b, b2, f = w(), w(), w()
    dy = integers(gen, F16, m, n, high=1)
    y0 = ffn.fused_linear(a, b)
    assert torch.equal(y0.double(), a.double() @ b.double())
    da, db, _ = ffn.fused_linear_backward(dy, a, b)
    step_a = ffn.fused_linear(a + e, b).double() - y0.double()
    assert float((step_a * dy.double()).sum()) == float((da.double() * e.double()).sum())
    step_b = ffn.fused_linear(a, b + f).double() - y0.double()
    assert float((step_b * dy.double()).sum()) == float((db.double() * f.double()).sum())
    # gate * up without an activation: the central difference of a product is exact.
    lo = integers(gen, F16, m, 8, high=1)
    bg, bu = b[:8], b2[:8]
    g, u = ffn.fused_linear(lo, bg), ffn.fused_linear(lo, bu)
    h = ffn.gated_linear(lo, bg, bu, activation=None)
    assert torch.equal(h, g * u)
    el = integers(gen, F16, m, 8, high=1)
    da, dbg, dbu, _, _ = ffn.gated_linear_backward(dy, lo, bg, bu, g, u, activation=None)
    up = ffn.gated_linear(lo + el, bg, bu, activation=None).double()
    down = ffn.gated_linear(lo - el, bg, bu, activation=None).double()
    assert float(((up - down) * dy.double()).sum()) / 2 == float((da.double() * el.double()).sum())


@pytest.mark.parametrize("name", [a for a in ref.ACTIVATIONS if a not in (None, "relu")])
def test_activation_slope_against_differences(name):
    """dbias of one row is act'(z) dy: against the 64-bit central difference of act."""
    z = torch.linspace(-9, 9, 1024).to(F16).cuda()[None]
    dy = torch.ones_like(z)
    a, b = torch.ones((1, 8), dtype=F16, device="cuda"), torch.ones((1024, 8), dtype=F16, device="cuda").t()
    dbias = ffn.fused_linear_backward(dy, a, b, z, name, has_bias=True)[2]
    h = 1e-5
    zz = z[0].double()
    slope = (ref.act(zz + h, name)[0] - ref.act(zz - h, name)[0]) / (2 * h)
    # one half-step, 2^-19 of the parts the slope is made of, and the difference's own h^2 and 64-bit noise
    bound = ref.unit(F16) * slope.abs() + 2.0 ** -19 * (2 + zz.abs()) + ref.tiny(F16) + 1e-9
    ref.within(dbias, slope, bound, name)


@pytest.mark.parametrize("m,n,k", [(0, 64, 64), (5, 0, 64), (5, 64, 0), (300, 72, 0), (0, 0, 0), (0, 64, 0)])
@pytest.mark.parametrize("layout", ["nk", "kn"])
def test_empty(m, n, k, layout):
    gen = torch.Generator().manual_seed(1)
    a, b, b2 = make(gen, F16, m, k), weight(gen, F16, k, n, layout), weight(gen, F16, k, n, layout)
    bias, res, dy, z = make(gen, F16, n), make(gen, F16, m, n), make(gen, F16, m, n), make(gen, F16, m, n)
    y = ffn.fused_linear(a, b, bias, "silu", res)
    wy, _, ey, _ = ref.linear(d(a), d(b), d(bias), "silu", d(res), F16)
    ref.within(y, wy, ey, "y")
    h = ffn.gated_linear(a, b, b2, bias, bias)
    wh, _, _, eh, _, _ = ref.gated(d(a), d(b), d(b2), d(bias), d(bias), "silu", F16)
    ref.within(h, wh, eh, "h")
    da, db, dbias = ffn.fused_linear_backward(dy, a, b, z, "gelu", has_bias=True)
    wa, (wb,), (wbias,) = ref.linear_backward(d(dy), d(a), d(b), d(z), "gelu", F16)
    for got, want in ((da, wa), (db, wb), (dbias, wbias)):
        ref.within(got, *want, "gradient")
    grads = ffn.gated_linear_backward(dy, a, b, b2, z, z, has_bias=True)
    wa, wb, wbias = ref.gated_backward(d(dy), d(a), d(b), d(b2), d(z), d(z), "silu", F16)
    for got, want in zip(grads, [wa, *wb, *wbias]):
        ref.within(got, *want, "gradient")


@pytest.mark.parametrize("m", [3, 130])
@pytest.mark.parametrize("n,pad,off", [(200, 8, 0), (200, 3, 1), (77, 0, 0)])
def test_outputs_touch_nothing_else(m, n, pad, off):
    """Outputs in a wider buffer, aligned and not: everything around them keeps its bits."""
    gen = torch.Generator().manual_seed(m)
    k = 136
    a, b, b2 = make(gen, F16, m, k), weight(gen, F16, k, n, "nk"), weight(gen, F16, k, n, "nk")

    def guarded():
        buf = torch.full((m + 2, n + pad + 8), 123.0, dtype=F16, device="cuda")
        return buf, buf[1:m + 1, off:off + n]

    bufs = [guarded() for _ in range(5)]
    (y, z, h, g, u) = (v for _, v in bufs)
    ffn.fused_linear_into(a, b, y, None, "gelu", None, z)
    ffn.gated_linear_into(a, b, b2, h, None, None, "gelu", g, u)
    nbuf, nv = guarded()
    ffn.layer_norm_into(z, nv)
    assert torch.equal(y, ffn.fused_linear(a, b, None, "gelu"))
    want = ffn.gated_linear(a, b, b2, None, None, "gelu", return_preact=True)
    assert all(torch.equal(x, w) for x, w in zip((h, g, u), want))
    # z and gate are the same sums, cut up for different kernels: each within its own bound.
    _, wz, _, ez = ref.linear(d(a), d(b), None, "gelu", None, F16)
    ref.within(z, wz, ez, "z")
    assert torch.equal(nv, ffn.layer_norm(z))
    for buf, v in bufs + [(nbuf, nv)]:
        v.fill_(123.0)
        assert bool((buf == 123.0).all())


@pytest.mark.parametrize("off", [(True, True), (True, False), (False, True)], ids=["both", "a", "b"])
def test_rows_off_whole_sectors(off):
    # Rows at odd multiples of 16 bytes (copied where that pays) hold what rows of whole sectors hold.
    gen = torch.Generator().manual_seed(6)
    m, n, k = 512, 8200, 4104
    a, b, b2 = make(gen, BF16, m, k), weight(gen, BF16, k, n, "nk"), weight(gen, BF16, k, n, "nk")
    dy = make(gen, BF16, m, n)

    def padded(x, on):
        return torch.nn.functional.pad(x, (0, 8))[:, :k] if on else x

    def all_of(a, b, b2):
        h, g, u = ffn.gated_linear(a, b, b2, return_preact=True)
        return [ffn.fused_linear(a, b, activation="silu"), h, g, u,
                *ffn.gated_linear_backward(dy, a, b, b2, g, u, has_bias=True)]

    want = all_of(padded(a, True), padded(b.t(), True).t(), padded(b2.t(), True).t())
    got = all_of(padded(a, not off[0]), padded(b.t(), not off[1]).t(), padded(b2.t(), not off[1]).t())
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # Two roundings of y and one of z (slope of SiLU at most 1.1): 2^-8 each, of values that 2^-6 covers.
    torch.testing.assert_close(want[0], torch.nn.functional.silu(a @ b), rtol=2.0 ** -6, atol=2.0 ** -6)


def test_broadcast_residual_and_gradient():
    gen = torch.Generator().manual_seed(2)
    a, b = make(gen, BF16, 70, 64), weight(gen, BF16, 64, 96, "nk")
    r = make(gen, BF16, 1, 96)
    assert torch.equal(ffn.fused_linear(a, b, residual=r.expand(70, 96)),
                       ffn.fused_linear(a, b, residual=r.expand(70, 96).contiguous()))
    one = torch.ones((), dtype=BF16, device="cuda").expand(70, 96)
    got = ffn.fused_linear_backward(one, a, b, has_bias=True)
    want = ffn.fused_linear_backward(one.contiguous(), a, b, has_bias=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("m", [20, 300])
def test_non_finite_rows_stay_in_their_rows(m):
    gen = torch.Generator().manual_seed(3)
    a, b, b2 = make(gen, F16, m, 200), weight(gen, F16, 200, 136, "nk"), weight(gen, F16, 200, 136, "nk")
    clean = ffn.fused_linear(a, b), ffn.gated_linear(a, b, b2), ffn.layer_norm(a)
    a[7, 3], a[11, 5] = float("nan"), float("inf")
    for got, was in zip((ffn.fused_linear(a, b), ffn.gated_linear(a, b, b2), ffn.layer_norm(a)), clean):
        assert bool(torch.isnan(got[7]).all()) and not bool(torch.isfinite(got[11]).any())
        keep = [i for i in range(m) if i not in (7, 11)]
        assert torch.equal(got[keep], was[keep])


NORM_SIZES = [(1, 1), (1, 8), (3, 33), (5, 256), (9, 264), (4, 512), (130, 520), (7, 1024), (6, 1032), (300, 2048),
              (33, 2050), (1, 4096), (700, 4096), (5, 4104), (150, 8192), (6, 8200), (300, 16384), (3, 16392), (2, 20001),
              (958, 111), (40, 257), (7, 513), (300, 1001), (9, 1030), (1200, 2047), (40, 4095), (160, 8190), (5, 12001),
              (4, 16383)]


@pytest.mark.parametrize("i,size", list(enumerate(NORM_SIZES)), ids=[f"m{m}-n{n}" for m, n in NORM_SIZES])
def test_layer_norm(i, size):
    m, n = size
    dtype = BF16 if i % 2 else F16
    gen = torch.Generator().manual_seed(m + n)
    for layout in ("plain", "odd"):
        x = rows(gen, dtype, m, n, layout) * 1.5 + 0.5 if layout == "plain" else rows(gen, dtype, m, n, layout)
        w, b = make(gen, dtype, n, scale=0.2) + 1, make(gen, dtype, n, scale=0.2)
        dy = rows(gen, dtype, m, n, layout)
        for ww, bb in ((w, b), (None, None), (w, None), (None, b)):
            y, mean, rstd = ffn.layer_norm(x, ww, bb, 1e-5, return_stats=True)
            wy, wm, wr, ey, em, er = ref.layer_norm(d(x), d(ww), d(bb), 1e-5, dtype)
            ref.within(mean, wm, em, "mean")
            ref.within(rstd, wr, er, "rstd")
            ref.within(y, wy, ey, "y")
            assert torch.equal(y, ffn.layer_norm(x, ww, bb, 1e-5))
            got = ffn.layer_norm_backward(dy, x, mean, rstd, ww, has_bias=bb is not None)
            want = ref.layer_norm_backward(d(dy), d(x), d(mean), d(rstd), d(ww), dtype)
            assert (got[1] is None) == (ww is None) and (got[2] is None) == (bb is None)
            for g, (wv, we) in zip(got, want):
                if g is not None:
                    ref.within(g, wv, we, "gradient")


def test_layer_norm_of_constant_and_empty_rows():
    x = torch.full((4, 100), 7.0, dtype=F16, device="cuda")
    y, mean, rstd = ffn.layer_norm(x, eps=1e-5, return_stats=True)
    # 7 * 100 and its mean are exact up to the reciprocal of 100: deviations of 2^-23 * 7 times rstd.
    assert float(y.abs().max()) <= 7 * 2.0 ** -22 * (1e-5) ** -0.5
    assert float((mean - 7).abs().max()) <= 7 * 2.0 ** -22
    empty = torch.empty((0, 100), dtype=F16, device="cuda")
    assert ffn.layer_norm(empty).shape == (0, 100)
    w = torch.ones(100, dtype=F16, device="cuda")
    stats = torch.empty(0, device="cuda")
    _, dw, db = ffn.layer_norm_backward(empty, empty, stats, stats, w, has_bias=True)
    assert float(dw.abs().sum()) == 0.0 and float(db.abs().sum()) == 0.0
    assert ffn.layer_norm(torch.empty((5, 0), dtype=F16, device="cuda")).shape == (5, 0)


def test_same_bits_on_every_run():
    gen = torch.Generator().manual_seed(5)
    for m in (7, 128, 700):
        a, b, b2 = make(gen, BF16, m, 1000), weight(gen, BF16, 1000, 520, "nk"), weight(gen, BF16, 1000, 520, "nk")
        dy = make(gen, BF16, m, 520)

        def everything():
            h, g, u = ffn.gated_linear(a, b, b2, return_preact=True)
            y, mean, rstd = ffn.layer_norm(a, return_stats=True)
            return [h, y, *(t for t in ffn.gated_linear_backward(dy, a, b, b2, g, u, has_bias=True)),
                    *(t for t in ffn.layer_norm_backward(a, a, mean, rstd, a[0], has_bias=True))]

        first = everything()
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(first, everything()))


@pytest.mark.parametrize("m", [9, 300])
def test_block_runs_and_trains(m):
    """layer_norm -> gated_linear -> fused_linear with the residual, as one differentiable block."""
    gen = torch.Generator().manual_seed(6)
    dim, hidden, dtype = 136, 328, BF16
    x = make(gen, dtype, m, dim)
    nw, nb = make(gen, dtype, dim, scale=0.1) + 1, make(gen, dtype, dim, scale=0.1)
    wg, wu, wd = make(gen, dtype, hidden, dim, scale=dim ** -0.5), make(gen, dtype, hidden, dim, scale=dim ** -0.5), \
        make(gen, dtype, dim, hidden, scale=hidden ** -0.5)
    bg, bu, bd = (make(gen, dtype, s, scale=0.1) for s in (hidden, hidden, dim))
    leaves = [x, wg, wu, wd, nw, nb, bg, bu, bd]

    def block(f, x, wg, wu, wd, nw, nb, bg, bu, bd):
        return f(x, wg.t(), wu.t(), wd.t(), nw, nb, bg, bu, bd, "silu")

    plain = block(ffn.feed_forward, *leaves)
    params = [t.clone().requires_grad_() for t in leaves]
    y = block(ffn.feed_forward, *params)
    assert torch.equal(y, plain)
    dy = make(gen, dtype, m, dim)
    y.backward(dy)

    def reference(x, bg_, bu_, bd_, nw, nb, b0, b1, b2, act):
        h = torch.nn.functional.layer_norm(x, (x.shape[1],), nw, nb, 1e-5)
        return x + (ref.act(h @ bg_ + b0, act)[0] * (h @ bu_ + b1)) @ bd_ + b2

    doubles = [t.double().requires_grad_() for t in leaves]
    want = block(reference, *doubles)
    want.backward(dy.double())
    want = want.detach()
    # Four 16-bit roundings lie on the path of y (norm, h, and y itself; gate and up stay in 32 bits), up to eight
    # on a gradient's; each is half a step at most of values of the result's own size, so in the 2-norm their sum
    # stays below their number times the unit.
    u = ref.unit(dtype)
    assert float((y.detach().double() - want).norm() / want.norm()) <= 4 * u
    for p, q in zip(params, doubles):
        assert p.grad.dtype == dtype and p.grad.shape == q.grad.shape
        assert float((p.grad.double() - q.grad).norm() / q.grad.norm()) <= 8 * u


def test_partial_gradients():
    gen = torch.Generator().manual_seed(7)
    a, w, bias, res = make(gen, F16, 40, 64), make(gen, F16, 72, 64, scale=0.1), make(gen, F16, 72), make(gen, F16, 40, 72)
    full = [t.clone().requires_grad_() for t in (a, w, bias, res)]
    dy = make(gen, F16, 40, 72)
    y, z = ffn.fused_linear(full[0], full[1].t(), full[2], "gelu", full[3], return_preact=True)
    y.backward(dy)
    wa, (wb,), (wbias,) = ref.linear_backward(d(dy), d(a), d(w.t()), d(z.detach()), "gelu", F16)
    want = [wa, (wb[0].t(), wb[1].t()), wbias, (d(dy), torch.zeros_like(d(dy)))]
    for t, v in zip(full, want):
        ref.within(t.grad, *v, "gradient")
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((a, w, bias, res))]
        ffn.fused_linear(some[0], some[1].t(), some[2], "gelu", some[3]).backward(dy)
        for j, t in enumerate(some):
            assert (t.grad is None) == (j != i)
        ref.within(some[i].grad, *want[i], "gradient alone")


def test_custom_ops_check():
    gen = torch.Generator().manual_seed(8)
    a, b, b2 = make(gen, F16, 12, 64), weight(gen, F16, 64, 72, "nk"), weight(gen, F16, 64, 72, "kn")
    bias = make(gen, F16, 72)
    ops = torch.ops.gemm_lab
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(ops.fused_linear, (a, b, bias, "silu", None), test_utils=tests)
    torch.library.opcheck(ops.gated_linear, (a, b, b2, None, None, "silu"), test_utils=tests)
    torch.library.opcheck(ops.layer_norm, (a, None, None, 1e-5), test_utils=tests)


def test_another_stream():
    gen = torch.Generator().manual_seed(9)
    a, b, b2 = make(gen, F16, 300, 512), weight(gen, F16, 512, 1032, "nk"), weight(gen, F16, 512, 1032, "nk")
    dy = make(gen, F16, 300, 1032)
    h, g, u = ffn.gated_linear(a, b, b2, return_preact=True)
    want = [h, *ffn.gated_linear_backward(dy, a, b, b2, g, u, has_bias=True)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                h, g, u = ffn.gated_linear(a, b, b2, return_preact=True)
                out = [h, *ffn.gated_linear_backward(dy, a, b, b2, g, u, has_bias=True)]
            got.append(out)
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("m", [4, 300])
@pytest.mark.parametrize("pdl", [True, False])
def test_captured_graphs(m, pdl):
    """Two graphs of the same operators, replayed in turn and on new inputs; odd sizes take workspaces."""
    gen = torch.Generator().manual_seed(10)
    k, n = 131, 264
    w = [weight(gen, F16, k, n, "nk") for _ in range(2)]
    down = weight(gen, F16, n, k, "nk")

    def step(x, dy):
        hn, mean, rstd = ffn.layer_norm(x, return_stats=True)
        h, g, u = ffn.gated_linear(hn, *w, return_preact=True)
        y = ffn.fused_linear(h, down, residual=x)
        dh, ddown, _ = ffn.fused_linear_backward(dy, h, down)
        grads = ffn.gated_linear_backward(dh, hn, *w, g, u, has_bias=True)
        return [y, ddown, *grads, ffn.layer_norm_backward(grads[0], x, mean, rstd)[0]]

    with kernels.launch_options(pdl=pdl):
        xs = [make(gen, F16, m, k) for _ in range(2)]
        dys = [make(gen, F16, m, k) for _ in range(2)]
        step(xs[0], dys[0])  # set-up before capture
        torch.cuda.synchronize()
        graphs, outs = [], []
        for x, dy in zip(xs, dys):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(step(x, dy))
            graphs.append(graph)
        for turn in range(3):
            for x, dy in zip(xs, dys):
                x.copy_(make(gen, F16, m, k))
                dy.copy_(make(gen, F16, m, k))
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for x, dy, out in zip(xs, dys, outs):
                assert all(torch.equal(p, q) for p, q in zip(out, step(x, dy)))


def test_dealt_runs_replay():
    """A backward pass whose K blocks are dealt over the pairs: joins through the workspace, replayed and on two
    streams at once."""
    gen = torch.Generator().manual_seed(12)
    m, n, k = 999, 1032, 520
    lib = native.library()
    a, b = make(gen, BF16, m, k), weight(gen, BF16, k, n, "nk")
    dy = make(gen, BF16, m, n)
    # Aligned operands and no activation: what the workspace is for is the runs.
    assert lib.glq_fused_linear_backward_workspace_bytes(
        1, dy.data_ptr(), n, a.data_ptr(), k, 1, b.data_ptr(), 1, k, 0, 0, m, n, k) > 0
    want = ffn.fused_linear_backward(dy, a, b)
    wa, (wb,), _ = ref.linear_backward(d(dy), d(a), d(b), None, None, BF16)
    ref.within(want[0], *wa, "da")
    ref.within(want[1], *wb, "db")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ffn.fused_linear_backward(dy, a, b)
        again = ffn.fused_linear_backward(dy, a, b)
    side = torch.cuda.Stream()
    for _ in range(5):
        for t in (*got[:2], *again[:2]):
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            other = ffn.fused_linear_backward(dy, a, b)
        torch.cuda.synchronize()
        for out in (got, again, other):
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_large_products():
    """Whole waves and a dealt remainder; two outputs, concatenated contraction; against matmul in 64 bits."""
    gen = torch.Generator().manual_seed(13)
    m, n, k = 2100, 2600, 1032
    a, bg, bu = make(gen, F16, m, k), weight(gen, F16, k, n, "nk"), weight(gen, F16, k, n, "nk")
    dy = make(gen, F16, m, n)
    h, g, u = ffn.gated_linear(a, bg, bu, return_preact=True)
    wh, wg, wu, eh, eg, eu = ref.gated(d(a), d(bg), d(bu), None, None, "silu", F16)
    for got, want, bound in ((h, wh, eh), (g, wg, eg), (u, wu, eu)):
        ref.within(got, want, bound, "gated")
    grads = ffn.gated_linear_backward(dy, a, bg, bu, g, u, has_bias=True)
    wa, wb, wbias = ref.gated_backward(d(dy), d(a), d(bg), d(bu), d(g), d(u), "silu", F16)
    for got, want in zip(grads, [wa, *wb, *wbias]):
        ref.within(got, *want, "gradient")


def test_a_fresh_thread():
    """The first CUDA work of a thread may be one of these calls (an autograd thread's, for one)."""
    import threading

    gen = torch.Generator().manual_seed(15)
    a, b, dy = make(gen, F16, 24, 64), weight(gen, F16, 64, 72, "nk"), make(gen, F16, 24, 72)
    calls = [lambda: ffn.fused_linear_backward(dy, a, b)[:2], lambda: (ffn.gated_linear(a, b, b),),
             lambda: (ffn.layer_norm(a),), lambda: (kernels.triton_matmul(a, b),)]
    for call in calls:
        want, got, errors = call(), [], []

        def work():
            try:
                got.extend(call())
                torch.cuda.synchronize()
            except Exception as e:  # noqa: BLE001 -- reported below
                errors.append(e)

        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        assert not errors, errors
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("m,layout", [(1, "nk"), (5, "kn"), (128, "nk"), (300, "nk")])
def test_output_may_be_the_residual(m, layout):
    gen = torch.Generator().manual_seed(14)
    a, b, r = make(gen, F16, m, 264), weight(gen, F16, 264, 520, layout), make(gen, F16, m, 520)
    want = ffn.fused_linear(a, b, activation="relu", residual=r)
    assert ffn.fused_linear_into(a, b, r, activation="relu", residual=r) is r
    assert torch.equal(r, want)


def test_static_weights_flag():
    gen = torch.Generator().manual_seed(11)
    a, b, b2 = make(gen, F16, 5, 520), weight(gen, F16, 520, 264, "nk"), weight(gen, F16, 520, 264, "nk")
    want = ffn.gated_linear(a, b, b2), ffn.fused_linear(a, b)
    with kernels.launch_options(static_weights=True):
        for _ in range(3):
            a2 = a * 1  # a kernel that writes A just before
            got = ffn.gated_linear(a2, b, b2), ffn.fused_linear(a2, b)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
