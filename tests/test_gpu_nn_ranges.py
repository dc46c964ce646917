"""The gated block's operators (libsdfnn.so) at the ends of their ranges.

Tolerances are counted in roundings as in test_gpu_nn_operators.py, whose references are used here."""
import pytest
import torch

from test_gpu_nn_operators import ACTS, BF16, F16, F32, close, gated_ref, half, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 15, 16])
@pytest.mark.parametrize("d,f,o", [(64, 128, 64), (100, 513, 77), (256, 4096, 130)])
def test_few_rows_keep_their_hidden_values(device, t, rows, d, f, o):
    """Up to 16 rows of a 16-bit type the hidden row goes into the second product as two numbers of that type: what is left out is half a step of half a
    step of it, where one number alone would be off by half a step."""
    from sdfstudio_amd.field_components.mlp import gated_mlp

    x = rnd(rows, d, t=t)
    ws = [rnd(f, d, t=t, std=d ** -0.5), rnd(f, d, t=t, std=d ** -0.5), rnd(o, f, t=t, std=f ** -0.5)]
    for act in ("silu", "gelu"):
        y = gated_mlp(x, *ws, activation=act)
        out, mag, _ = gated_ref(x, *ws, torch.zeros_like(y), act)
        xd, wg, wu, wd = (v.double() for v in (x, *ws))
        h = (ACTS[act](xd @ wg.t()) * (xd @ wu.t())).abs()
        # sums and activations as in test_gated_mlp_forward_backward; the second number's rounding, fp16's not below 2^-25; the result's own
        room = 2.0 ** -20 * mag[0] + half(t) ** 2 * (h @ wd.abs().t()) + (2.0 ** -25 * wd.abs().sum(-1) if t == F16 else 0.0)
        close(f"{act} {t}", y, out[0], room, half(t) + 2.0 ** -20)
        leaves = [v.clone().requires_grad_(True) for v in (x, *ws)]
        assert torch.equal(gated_mlp(*leaves, activation=act), y)


Z = [0.0, 1.0, -1.0, 9.5, -9.5, 20.0, -20.0, -60.0, -86.0, -87.5, -88.0, -89.0, -100.0, -110.0, -129.0, -1e4, -1e20, -1e36, -1e38, 89.0, 129.0, 1e4, 1e20, 1e36]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [24, 240])
def test_fp32_activations_far_from_zero(device, act, rows):
    """act(z) and act'(z) in fp32 where the exponential leaves the normal numbers: values and slopes end in 0 on the left, in z and 1 on the right."""
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.quantization import int8_gated_linear

    z = torch.tensor(Z, device="cuda").repeat(rows // len(Z))
    x = torch.stack([z, torch.ones_like(z)], 1).requires_grad_(True)
    ws = [torch.tensor([v], device="cuda") for v in ([1.0, 0.0], [0.0, 1.0], [1.0])]
    y = gated_mlp(x, *ws, activation=act)
    (dx,) = torch.autograd.grad(y.sum(), x)
    zd = z.double().requires_grad_(True)
    a = ACTS[act](zd)
    (slope,) = torch.autograd.grad(a.sum(), zd)
    a = a.detach()
    slope = torch.where(zd.detach().abs() > 1e3, (zd.detach() > 0).double(), slope)  # (the formula's inf * 0)
    # 2^-19 as everywhere; the exponent z^2 / 2 of the normal distribution is rounded once: half a step of it; what lies below the normal numbers
    # of fp32 may be 0, times |z| < 2^8
    rel = 2.0 ** -19 + (2.0 ** -24 * (z.double().square() / 2).clamp_max(128.0) if act == "gelu" else 0.0)
    close("y", y[:, 0], a, 2.0 ** -126 * 256, rel)
    close("slope", dx[:, 0], slope, 2.0 ** -126 * 256 + 2.0 ** -21, rel)  # (the slope's two terms cancel near its zero at z = -1.28 / -0.75)
    close("gate", dx[:, 1], a, 2.0 ** -126 * 256, rel)
    keep = z < 1e30  # (their products with `up` stay finite)
    z, a, rel = (v[keep] if isinstance(v, torch.Tensor) else v for v in (z, a, rel))
    q = torch.where(z < 0, -1, 1)[:, None].to(torch.int8)
    one = torch.ones(1, 1, device="cuda", dtype=torch.int8)
    s = z.abs() / 2.0 ** 20
    y = int8_gated_linear(q, s, one, torch.full((1,), 2.0 ** 20, device="cuda"), one, torch.full((1,), 2.0 ** -20, device="cuda"), activation=act)
    close("8 bits", y[:, 0], a * (z.double() * 2.0 ** -40), 2.0 ** -126 * 256, rel + 2.0 ** -20)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("rows", [30, 8192])
def test_16_bit_gelu_holds_its_relative_accuracy(device, t, rows):
    """gelu of values far left of zero, where it is small but not nothing: z Phi(z) to the type's own step."""
    from sdfstudio_amd.field_components.quantization import int8_gated_linear

    x = torch.linspace(0.0, 12.5, rows, device="cuda")
    q = torch.full((rows, 1), -1, device="cuda", dtype=torch.int8)
    one = torch.ones(1, 1, device="cuda", dtype=torch.int8)
    su = 1.0 if t == BF16 else 4096.0
    y = int8_gated_linear(q, x, one, torch.ones(1, device="cuda"), one, torch.full((1,), su, device="cuda"), activation="gelu", out_dtype=t)
    z = -x.double()
    # 2^-12 for log2 of the tail's polynomial (1.3e-4), its exponent of up to 113 rounded twice (1e-5) and the exponential (2^-23)
    close("gelu", y[:, 0], ACTS["gelu"](z) * (z * su), 2.0 ** -126 * 256, half(t) + 2.0 ** -12)


@pytest.mark.parametrize("rows", [20, 40])
def test_rows_of_long_strides(device, rows):
    """The last token of every sequence of a batch: rows 8 MiB apart and more give what their copies give, forward and backward."""
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm
    from sdfstudio_amd.field_components.quantization import int8_gated_linear, int8_linear, quantize_rows

    base = torch.empty(rows, 1025, 4096, device="cuda", dtype=BF16)
    x = base[:, -1]
    x.copy_(torch.randn(rows, 4096, device="cuda"))
    c = x.contiguous()
    ws = [torch.randn(72, 4096, device="cuda").div_(64).to(BF16), torch.randn(72, 4096, device="cuda").div_(64).to(BF16), torch.randn(4096, 72, device="cuda").to(BF16)]
    dy = base[:, 1]  # as far apart
    dy.copy_(torch.randn(rows, 4096, device="cuda"))
    got, want = [], []
    for a, d, out in ((x, dy, got), (c, dy.contiguous(), want)):
        leaves = [v.detach().requires_grad_(True) for v in (a, *ws)]
        y = gated_mlp(*leaves)
        out += [y, *torch.autograd.grad(y, leaves, d), rms_norm(a, ws[0][0]), *quantize_rows(a)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del base, x, dy
    base = torch.empty(rows, 2050, 4096, device="cuda", dtype=torch.int8)
    q, s = base[:, -1], torch.rand(rows, device="cuda")
    q.copy_(torch.randint(-127, 128, (rows, 4096), device="cuda"))
    w, sw = torch.randint(-127, 128, (40, 4096), device="cuda", dtype=torch.int8), torch.rand(40, device="cuda")
    assert torch.equal(int8_linear(q, s, w, sw), int8_linear(q.contiguous(), s, w, sw))
    assert torch.equal(int8_gated_linear(q, s, w, sw, w, sw), int8_gated_linear(q.contiguous(), s, w, sw, w, sw))
    few = base[:3, -1]  # as weights
    assert torch.equal(int8_linear(w, sw, few, s[:3]), int8_linear(w, sw, few.contiguous(), s[:3]))


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows", [5, 20, 50, 70, 3000])
def test_rows_that_are_not_finite_have_no_finite_result(device, t, act, rows):
    """An infinity or a NaN among a row's inputs, on every kernel: no result of that row is a number; fp32 beyond 64 rows gives NaN alone."""
    from sdfstudio_amd.field_components.mlp import gated_mlp

    x = rnd(rows, 64, t=t)
    ws = [rnd(96, 64, t=t), rnd(96, 64, t=t), rnd(64, 96, t=t)]
    x[0, 3], x[2, 60], x[4, 0] = float("inf"), float("-inf"), float("nan")
    y = gated_mlp(x, *ws, activation=act)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[0, 2, 4]] = True
    assert not torch.isfinite(y[bad]).any() and torch.isfinite(y[~bad]).all()
    if t == F32 and rows > 64:
        assert torch.isnan(y[bad]).all()
