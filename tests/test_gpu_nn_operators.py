"""The gated feed-forward block's operators (libsdfnn.so) against plain fp64 implementations on the GPU's own inputs.

Tolerances are counted in roundings: half a step of the result's type is `finfo(t).eps / 2` relative to the value (fp32 2^-24, bf16 2^-8,
fp16 2^-11).  A sum of n products in fp32 is allowed n-independent 2^-19 of sum |a b| (its blocks of 16 - 64 terms and their tree stay far
below n 2^-24 for n <= 2^16 in the typical case; 2^-19 is 32 steps)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
SUM = 2.0 ** -19


def half(t):
    return torch.finfo(t).eps / 2


def close(name, got, want, atol, rtol):
    """|got - want| <= atol + rtol |want| element-wise; atol may be a tensor.  A relative half step holds for normal numbers: fp16's end at
    2^-14, and below that its values lie 2^-24 apart, so rounding to it is off by up to 2^-25 there (bf16 and fp32 reach down to 2^-126)."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got, want = got.detach(), want.detach()
    err = (got.double() - want).abs()
    bound = rtol * want.abs() + atol + (2.0 ** -25 if got.dtype == F16 else 0.0)
    bad = ~(err <= bound)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - bound).max()):.3e} beyond, err {float(err.max()):.3e}"


def rnd(*shape, t=F32, std=1.0, dev="cuda"):
    return (torch.randn(*shape, device=dev) * std).to(t)


# ------------------------------------------------------------------------------------------------ norm
def norm_ref(x, r, w, eps=1e-6):
    h = x.double() + (r.double() if r is not None else 0.0)
    inv = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h, inv, h * inv * w.double()


NORM_SHAPES = [(1, 1), (1, 7), (3, 8), (5, 63), (64, 256), (130, 513), (33, 1000), (9, 1025), (7, 2049), (3, 4097), (2, 8200), (2, 33001)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_forward_backward(device, t, rows, dim, residual):
    from sdfstudio_amd.field_components.normalization import rms_norm

    x, w = rnd(rows, dim, t=t), (1 + rnd(dim, std=0.2)).to(t)
    r = rnd(rows, dim, t=t) if residual else None
    dy, dh = rnd(rows, dim, t=t), rnd(rows, dim, t=t)
    leaves = [v.requires_grad_(True) for v in (x, w, r) if v is not None]
    out = rms_norm(x, w, residual=r)
    y, h = out if residual else (out, None)
    grads = torch.autograd.grad((y, h) if residual else y, leaves, (dy, dh) if residual else dy)
    hr, inv, yr = norm_ref(x.detach(), r.detach() if residual else None, w.detach())
    close("y", y, yr, 1e-30, half(t) + 2.0 ** -21)  # the statistic, two products and the rounding: 8 steps of fp32
    if residual:
        close("h", h, hr, 0.0, half(t) + 2.0 ** -23)
    n, u = hr * inv, dy.double() * w.detach().double()
    mean = (u * n).mean(-1, keepdim=True)
    dx = inv * (u - n * mean) + (dh.double() if residual else 0.0)
    # terms of dx cancel: allow the steps of its largest term
    room = 2.0 ** -20 * (inv * (u.abs() + n.abs() * (u * n).abs().mean(-1, keepdim=True)) + (dh.double().abs() if residual else 0.0))
    close("dx", grads[0], dx, room, half(t))
    if residual:
        assert torch.equal(grads[0], grads[2])
    close("dw", grads[1], (dy.double() * n).sum(0), SUM * (dy.double() * n).abs().sum(0), half(t))


def test_rms_norm_partial_gradients_and_strides(device):
    from sdfstudio_amd.field_components.normalization import rms_norm

    base = rnd(6, 5, 100)
    x = base[:, 1:4, 10:90]  # rows that are not adjacent
    w = rnd(80)
    y = rms_norm(x, w)
    close("strided", y, norm_ref(x, None, w)[2], 1e-30, 2.0 ** -21)
    xt = rnd(80, 12).t()  # a transposed view: elements of a row are not adjacent
    close("transposed", rms_norm(xt, w), norm_ref(xt, None, w)[2], 1e-30, 2.0 ** -21)
    xe = rnd(1, 80).expand(9, 80).requires_grad_(True)  # a broadcast input: the gradients of its copies add up
    (g,) = torch.autograd.grad(rms_norm(xe, w).sum(), xe)
    assert g.shape == (9, 80)
    for use in ("y", "h"):  # only one of the outputs has a gradient
        xl, rl, wl = rnd(4, 80).requires_grad_(True), rnd(4, 80).requires_grad_(True), rnd(80).requires_grad_(True)
        y, h = rms_norm(xl, wl, residual=rl)
        got = torch.autograd.grad((y if use == "y" else h).sum(), (xl, rl, wl), allow_unused=True)
        xd, rd, wd = (v.detach().double().requires_grad_(True) for v in (xl, rl, wl))
        hd, _, yd = norm_ref(xd, rd, wd)
        want = torch.autograd.grad((yd if use == "y" else hd).sum(), (xd, rd, wd), allow_unused=True)
        for a, b in zip(got, want):
            b = torch.zeros_like(a).double() if b is None else b
            close(use, a, b, 1e-5, 1e-5)


# ------------------------------------------------------------------------------------------------ 8 bits
def codes_ref(v):
    top = v.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * v / top), torch.zeros_like(v)), top / 127


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_quantized(device, t, rows, dim, residual):
    from sdfstudio_amd.field_components.normalization import rms_norm_quantized

    x, w = rnd(rows, dim, t=t), (1 + rnd(dim, std=0.2)).to(t)
    r = rnd(rows, dim, t=t) if residual else None
    out = rms_norm_quantized(x, w, residual=r)
    hr, inv, _ = norm_ref(x, r, w)
    q, step = codes_ref(hr * w.double())
    assert out[0].dtype == torch.int8 and torch.equal(out[0].double(), q)
    close("scales", out[1], (step * inv).squeeze(-1), 0.0, 2.0 ** -21)
    if residual:
        close("h", out[2], hr, 0.0, half(t) + 2.0 ** -23)


@pytest.mark.parametrize("t", TYPES)
def test_quantize_rows_values(device, t):
    from sdfstudio_amd.field_components.quantization import quantize_rows

    x = rnd(257, 129, t=t)
    x[3] = 0
    x[4] = torch.arange(129, device="cuda").to(t) - 64  # |max| 64: exact ties
    x[5, 0], x[5, 1:] = 127, (torch.arange(128, device="cuda") - 63.5).to(t)  # step 1: every second value is a tie, half to even
    q, s = quantize_rows(x)
    want, step = codes_ref(x.double())
    assert torch.equal(q.double(), want)
    close("scales", s, step.squeeze(-1), 0.0, 2.0 ** -24)
    assert s[3] == 0 and not q[3].any()
    x[6, 7] = float("nan")
    x[7, 7] = float("inf")
    q, s = quantize_rows(x)
    assert not torch.isfinite(s[6:8]).any() and torch.isfinite(s[:6]).all() and torch.isfinite(s[8:]).all()
    assert torch.isnan(q[6:8] * s[6:8, None]).all()
    tiny = (torch.randn(3, 64, device="cuda") * (1e-37 if t != F16 else 1e-7)).to(t)
    q, s = quantize_rows(tiny)
    assert torch.equal(q.double(), codes_ref(tiny.double())[0])


def int8_ref(q, s, w, sw, b=None):
    y = (q.double() @ w.double().t()) * s.double()[..., None] * sw.double()
    return y if b is None else y + b.double()


def codes(rows, k):
    q = torch.randint(-127, 128, (rows, k), device="cuda", dtype=torch.int8)
    return q, torch.rand(rows, device="cuda") * 0.01


INT8_SHAPES = [(1, 1, 1), (1, 16, 64), (2, 17, 100), (16, 64, 256), (17, 33, 31), (32, 129, 1000), (33, 64, 128), (100, 70, 1001), (128, 128, 2048),
               (257, 300, 144), (1000, 513, 640), (40, 24, 16384)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n,k", INT8_SHAPES)
def test_int8_linear(device, t, rows, n, k):
    from sdfstudio_amd.field_components.quantization import int8_linear

    q, s = codes(rows, k)
    w, sw = codes(n, k)
    b = rnd(n)
    for bias in (None, b):
        y = int8_linear(q, s, w, sw, bias=bias, out_dtype=t)
        # sum exact; its conversion, two products and the bias' addition: 4 half steps of fp32 of the larger term, then the type's own
        prod = int8_ref(q, s, w, sw)
        close("y", y, int8_ref(q, s, w, sw, bias), 2.0 ** -22 * prod.abs() + (2.0 ** -24 if t == F16 else 0), half(t) + 2.0 ** -23)


@pytest.mark.parametrize("k", [131072])
@pytest.mark.parametrize("rows", [3, 40])
def test_int8_linear_extreme_sums(device, k, rows):
    from sdfstudio_amd.field_components.quantization import int8_linear

    q = torch.full((rows, k), 127, device="cuda", dtype=torch.int8)
    w = torch.full((5, k), -127, device="cuda", dtype=torch.int8)
    w[1] = 127
    one = torch.ones
    y = int8_linear(q, one(rows, device="cuda"), w, one(5, device="cuda"))
    want = torch.full((rows, 5), -127.0 * 127.0 * k, device="cuda")
    want[:, 1] *= -1
    assert torch.equal(y, want)


ACTS = {"silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: z * 0.5 * torch.erfc(-z / math.sqrt(2)), "relu": torch.relu}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,n,k", [(1, 16, 64), (5, 65, 200), (24, 130, 513), (70, 33, 96), (300, 257, 384), (40, 16, 8192)])
def test_int8_gated_linear(device, t, act, rows, n, k):
    from sdfstudio_amd.field_components.quantization import int8_gated_linear

    q, s = codes(rows, k)
    (g, sg), (u, su) = codes(n, k), codes(n, k)
    s = s / k ** 0.5 * 0.2
    y = int8_gated_linear(q, s, g, sg, u, su, activation=act, out_dtype=t)
    gate, up = int8_ref(q, s, g, sg), int8_ref(q, s, u, su)
    # gate to 4 half steps, its activation's slope (<= 1.13), the activation itself to 8 half steps of its argument, the product
    want = ACTS[act](gate) * up
    close("y", y, want, 2.0 ** -20 * (gate * up).abs() + (2.0 ** -24 if t == F16 else 0), half(t) + 2.0 ** -20)


# ------------------------------------------------------------------------------------------------ gated MLP
def gated_ref(x, wg, wu, wd, dy, act):
    """y, gradients and, for the tolerance, sums of magnitudes of each, in fp64."""
    x, wg, wu, wd, dy = (v.detach().double() for v in (x, wg, wu, wd, dy))
    g, u = x @ wg.t(), x @ wu.t()
    gl = g.clone().requires_grad_(True)
    a = ACTS[act](gl)
    (slope,) = torch.autograd.grad(a.sum(), gl)
    a = a.detach()
    h = a * u
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    out = [h @ wd.t(), dg @ wg + du @ wu, dg.t().contiguous() @ x, du.t().contiguous() @ x, dy.t().contiguous() @ h]
    # magnitudes: an error of relative size e in every intermediate (g, u, dh carry e of THEIR magnitudes) moves the results by about e mag
    gm, um, dhm = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t(), dy.abs() @ wd.abs()
    hm = 1.2 * (gm * u.abs() + g.abs() * um) + h.abs()
    dgm = dhm * (u.abs() * slope.abs()) + dh.abs() * (1.2 * um + u.abs() * gm) + dg.abs()
    dum = dhm * a.abs() + dh.abs() * 1.2 * gm + du.abs()
    mag = [hm @ wd.abs().t(), dgm @ wg.abs() + dum @ wu.abs(), dgm.t().contiguous() @ x.abs(), dum.t().contiguous() @ x.abs(), dy.abs().t().contiguous() @ hm]
    # roundings to the type of g, u (backward), h, dg, du: relative to these values themselves
    r = 3 * (dg.abs()), 3 * (du.abs())
    rg = r[0] + (dh * u).abs() * g.abs()  # the slope at a rounded g (|act''| < 1.2)
    rmag = [h.abs() @ wd.abs().t(), rg @ wg.abs() + (r[1] + (dh * g).abs()) @ wu.abs(), rg.t().contiguous() @ x.abs(),
            (r[1] + (dh * g).abs()).t().contiguous() @ x.abs(), dy.abs().t().contiguous() @ h.abs()]
    return out, mag, rmag


GATED_SHAPES = [(1, 1, 1, 1), (1, 64, 128, 64), (2, 7, 13, 5), (16, 100, 40, 36), (17, 64, 64, 64), (32, 33, 65, 31), (33, 64, 128, 64), (49, 100, 70, 52), (64, 31, 129, 65), (65, 63, 127, 61),
                (5, 700, 33, 900), (40, 90, 1500, 1003), (64, 513, 300, 257),
                (128, 128, 256, 128), (200, 72, 136, 40), (300, 256, 512, 264), (515, 40, 24, 8), (1025, 200, 72, 300)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,d,f,o", GATED_SHAPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_mlp_forward_backward(device, t, m, d, f, o, act):
    from sdfstudio_amd.field_components.mlp import gated_mlp

    x, dy = rnd(m, d, t=t), rnd(m, o, t=t)
    ws = [rnd(f, d, t=t, std=d ** -0.5), rnd(f, d, t=t, std=d ** -0.5), rnd(o, f, t=t, std=f ** -0.5)]
    leaves = [v.requires_grad_(True) for v in (x, *ws)]
    y = gated_mlp(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        y2 = gated_mlp(*leaves, activation=act)
    assert torch.equal(y, y2), "training and inference forward"
    out, mag, rmag = gated_ref(*leaves, dy, act)
    tiny = 2.0 ** -24 if t == F16 else 0.0  # half a step of fp16's smallest values
    for name, got, want, am, rm in zip(("y", "dx", "dwg", "dwu", "dwd"), (y, *grads), out, mag, rmag):
        # few-row forward and every sum: 2^-19 of the magnitudes; roundings of the intermediates: half a step each
        room = 2.0 ** -20 * am + (half(t) * rm if t != F32 else 0.0) + tiny * (1 + am.amax())
        close(f"{name} {t}", got, want, room, half(t) + 2.0 ** -20)


def test_gated_mlp_relu(device):
    """max(z, 0): inputs of halves and integers, so that every gate is an exact sum and the kink (slope 0 at 0) is decided alike."""
    from sdfstudio_amd.field_components.mlp import gated_mlp

    def halves(*shape):
        return torch.randint(-3, 4, shape, device="cuda").float() / 2

    x, ws, dy = halves(150, 32), [halves(48, 32), halves(48, 32), halves(16, 48)], halves(150, 16)
    leaves = [v.requires_grad_(True) for v in (x, *ws)]
    y = gated_mlp(*leaves, activation="relu")
    grads = torch.autograd.grad(y, leaves, dy)
    out, _, _ = gated_ref(*leaves, dy, "relu")
    for got, want in zip((y, *grads), out):
        assert torch.equal(got.double(), want)  # sums of eighths far below 2^24: exact
