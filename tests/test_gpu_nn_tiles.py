"""The gated block's products (libsdfnn.so) on their 256 x 256 tiles, split along k and not, at ragged sizes; norms whose backward pass takes more than one
turn; codes at the ends of their type.

Tolerances are counted in roundings as in test_gpu_nn_operators.py, whose references are used here."""
import ctypes

import pytest
import torch

from test_gpu_nn_operators import BF16, F16, F32, SUM, ACTS, close, codes, gated_ref, half, int8_ref, norm_ref, rnd

# rows, dim, hidden, out: together they take each product of a pass (0 gate and up, 1 down, 2 gradients of g and u, 3 dx, 4 dw_down, 5 dw_gate and dw_up)
# through 256 x 256 tiles, whole along k and split (test_cpu_nn_calls.py holds the library's choice to this)
TILES_F32 = [(700, 264, 2100, 4100), (6001, 264, 1030, 4100), (4099, 3100, 300, 520), (16387, 264, 600, 4100), (700, 4104, 1030, 264)]
TILES_16 = [(8195, 264, 1030, 4100), (4099, 2056, 300, 264), (2100, 264, 5000, 2057), (6001, 264, 6008, 4100), (700, 2056, 6008, 2057), (700, 4104, 1030, 264)]
TILES_INT8 = [(4099, 2000, 8192, 2), (700, 2000, 32768, 2), (1030, 1000, 40001, 2), (4099, 2001, 8200, 1), (2000, 1001, 60000, 1)]  # rows, n, k, projections


def chosen(dtype, shape):
    """[(tile, k is split)] of the six products"""
    from sdfstudio_amd import _nn

    out, splits = [], ctypes.c_int32(0)
    for backward, count in ((0, 2), (1, 4)):
        for i in range(count):
            out.append((_nn.load().sdfnn_gated_product(dtype, *shape, backward, i, ctypes.byref(splits)), splits.value > 1))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("t,shape", [(F32, s) for s in TILES_F32] + [(t, s) for t in (BF16, F16) for s in TILES_16])
def test_gated_mlp_on_large_tiles(device, t, shape):
    from sdfstudio_amd.field_components.mlp import gated_mlp

    m, d, f, o = shape
    act = "gelu" if d == 264 else "silu"
    x, dy = rnd(m, d, t=t), rnd(m, o, t=t)
    ws = [rnd(f, d, t=t, std=d ** -0.5), rnd(f, d, t=t, std=d ** -0.5), rnd(o, f, t=t, std=f ** -0.5)]
    leaves = [v.requires_grad_(True) for v in (x, *ws)]
    y = gated_mlp(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(y, gated_mlp(*leaves, activation=act))
    out, mag, rmag = gated_ref(*leaves, dy, act)
    tiny = 2.0 ** -24 if t == F16 else 0.0
    for name, got, want, am, rm in zip(("y", "dx", "dwg", "dwu", "dwd"), (y, *grads), out, mag, rmag):
        # as test_gated_mlp_forward_backward: 2^-20 of the magnitudes for every sum, half a step of the type for every rounding between the products
        room = 2.0 ** -20 * am + (half(t) * rm if t != F32 else 0.0) + tiny * (1 + am.amax())
        close(f"{name} {t}", got, want, room, half(t) + 2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("shape", TILES_INT8)
def test_8_bit_products_on_large_tiles(device, t, shape):
    """Codes far from uniform, so that a column, row or step taken from another place shows; results as in test_int8_linear / test_int8_gated_linear."""
    from sdfstudio_amd.field_components.quantization import int8_gated_linear, int8_linear

    rows, n, k, projections = shape
    q, s = codes(rows, k)
    w, sw = codes(n, k)
    sw = sw / k ** 0.5
    if projections == 1:
        b = rnd(n)
        prod = int8_ref(q, s, w, sw)
        y = int8_linear(q, s, w, sw, bias=b, out_dtype=t)
        close("y", y, prod + b.double(), 2.0 ** -22 * prod.abs(), half(t) + 2.0 ** -23)
        return
    u, su = codes(n, k)
    su = su / k ** 0.5
    gate, up = int8_ref(q, s, w, sw), int8_ref(q, s, u, su)
    y = int8_gated_linear(q, s, w, sw, u, su, activation="gelu", out_dtype=t)
    close("y", y, ACTS["gelu"](gate) * up, 2.0 ** -20 * (gate * up).abs(), half(t) + 2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("k,rows", [(131071, 3), (131071, 40), (64, 300), (50, 20)])
def test_codes_of_minus_128(device, k, rows):
    """The lowest code, which no quantisation here makes but the products take: sums up to 2^14 k < 2^31."""
    from sdfstudio_amd.field_components.quantization import int8_linear

    q = torch.full((rows, k), -128, device="cuda", dtype=torch.int8)
    w = torch.full((5, k), -128, device="cuda", dtype=torch.int8)
    w[1] = 127
    y = int8_linear(q, torch.ones(rows, device="cuda"), w, torch.ones(5, device="cuda"))
    want = torch.full((rows, 5), 128.0 * 128.0 * k, device="cuda", dtype=torch.float64)
    want[:, 1] = -128.0 * 127.0 * k
    assert torch.equal(y, want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,dim", [(700, 8200), (257, 8193), (600, 20001)])
def test_wide_norms_of_many_rows(device, t, rows, dim):
    """Rows beyond 8192 columns, more of them than the weight's gradient takes in one turn (256)."""
    from sdfstudio_amd.field_components.normalization import rms_norm

    x, w, r = rnd(rows, dim, t=t), (1 + rnd(dim, std=0.2)).to(t), rnd(rows, dim, t=t)
    dy, dh = rnd(rows, dim, t=t), rnd(rows, dim, t=t)
    leaves = [v.requires_grad_(True) for v in (x, w, r)]
    y, h = rms_norm(x, w, residual=r)
    dx, dw, dr = torch.autograd.grad((y, h), leaves, (dy, dh))
    hr, inv, yr = norm_ref(x.detach(), r.detach(), w.detach())
    close("y", y, yr, 1e-30, half(t) + 2.0 ** -21)
    close("h", h, hr, 0.0, half(t) + 2.0 ** -23)
    n, u = hr * inv, dy.double() * w.detach().double()
    mean = (u * n).mean(-1, keepdim=True)
    room = 2.0 ** -20 * (inv * (u.abs() + n.abs() * (u * n).abs().mean(-1, keepdim=True)) + dh.double().abs())
    close("dx", dx, inv * (u - n * mean) + dh.double(), room, half(t))
    assert torch.equal(dx, dr)
    close("dw", dw, (dy.double() * n).sum(0), SUM * (dy.double() * n).abs().sum(0), half(t))
