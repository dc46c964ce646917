"""The gated block's operators (libsdfnn.so) at the ends of their ranges: few rows in 16 bits, activations far from zero, rows of long strides.

Tolerances are counted in roundings as in test_gpu_nn_operators.py, whose references are used here."""
import pytest
import torch

from test_gpu_nn_operators import ACTS, BF16, F16, close, gated_ref, half, rnd

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

