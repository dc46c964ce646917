"""8-bit serving form of a field's linear layers: rows quantised symmetrically (one scale a token / point, one a channel of the weights),
products on the integer matrix cores with exact 32-bit sums.  Runs on libsdfnn.so (include/sdfnn.h); no CPU path, no gradients.
"""
from typing import Optional, Tuple

import torch
from torch import nn

from sdfstudio_amd import _nn
from sdfstudio_amd.field_components.normalization import _check, _quantize

_CODE, _SCALE = torch.int8, torch.float32
MAX_K = 131072  # 127 * 127 * k stays below 2^31


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., dim] -> (codes int8 [..., dim] in [-127, 127], scales float32 [...]): code = round(127 x / max|x|) half to even, scale =
    max|x| / 127 of its row (a row of zeros: scale 0).  Serves activations (a scale a token) and weights [out, in] (a scale a channel).  Both results
    are constants to autograd, as rounded values are."""
    _check("quantize_rows", x, None, None)
    return _quantize("quantize_rows", x, None, None, 0.0)


def _check_operand(what: str, name: str, q: torch.Tensor, scales: torch.Tensor, k: Optional[int] = None) -> None:
    if q.dtype != torch.int8 or q.dim() < 1:
        raise TypeError(f"{what}: {name} {tuple(q.shape)} {q.dtype}: int8 rows expected")
    if k is not None and (q.dim() != 2 or q.shape[1] != k):
        raise ValueError(f"{what}: {name} {tuple(q.shape)} does not fit k = {k}")
    if scales.dtype != torch.float32 or scales.shape != q.shape[:-1]:
        raise ValueError(f"{what}: scales {tuple(scales.shape)} {scales.dtype} of {name} {tuple(q.shape)}: one float32 a row")


def _prepare(what, q, scales, weights, out_dtype):
    shape = q.shape
    k = shape[-1] if shape else 0
    if not (q.dtype is _CODE and scales.dtype is _SCALE and len(shape) == 2 and scales.shape == (shape[0],)):  # (as nearly always)
        _check_operand(what, "q", q, scales)
    for name, w, s in weights:
        shape = w.shape
        if not (w.dtype is _CODE and s.dtype is _SCALE and len(shape) == 2 and shape[1] == k and s.shape == (shape[0],)):
            _check_operand(what, name, w, s, k)
    if not 1 <= k <= MAX_K:
        raise ValueError(f"{what}: k = {k}: the 32-bit sum is exact for 1 .. {MAX_K}")
    if out_dtype not in _nn.DTYPES:
        raise TypeError(f"{what}: out_dtype {out_dtype} (float32, bfloat16, float16)")


def int8_linear(q: torch.Tensor, scales: torch.Tensor, weight_q: torch.Tensor, weight_scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y[..., n] = (sum_k q[..., k] weight_q[n, k]) scales[...] weight_scales[n] + bias[n] in out_dtype.  q int8 [..., k] with scales
    float32 [...], weight_q int8 [n, k] with weight_scales float32 [n], bias float32 [n].  No gradients: scales or a bias that would need one are refused."""
    what = "int8_linear"
    _prepare(what, q, scales, (("weight_q", weight_q, weight_scales),), out_dtype)
    _nn.check_modes(what, scales, weight_scales, bias)
    _nn.check_no_gradient(what, scales, weight_scales, bias)
    n = weight_q.shape[0]
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (n,)):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} {bias.dtype} for {n} channels: float32")
    lib, dev = _nn.load(), _nn.on_device(what, q, scales, weight_q, weight_scales, bias)
    with _nn.on(dev) as cur:
        q2, pq, rows, ldq = _nn.rows_of(q, align=True)
        w2, pw, _, ldw = _nn.rows_of(weight_q, align=True)
        sq, sw = scales.contiguous(), weight_scales.contiguous()
        b = bias.contiguous() if bias is not None else None
        k = q.shape[-1]
        y = torch.empty((rows, n) if q.dim() == 2 else (*q.shape[:-1], n), dtype=out_dtype, device=dev)
        if rows and n:
            size = _nn.size("sdfnn_int8_linear_workspace_size", rows, n, k, 1)
            ws = _nn.workspace(size, dev) if size else None
            _nn.check(lib.sdfnn_int8_linear(pq, ldq, sq.data_ptr(), pw, ldw, sw.data_ptr(), _nn.ptr(b), _nn.DTYPES[out_dtype], rows, n, k,
                                            y.data_ptr(), _nn.ptr(ws), size, cur.stream), "sdfnn_int8_linear")
    return y


def int8_gated_linear(q: torch.Tensor, scales: torch.Tensor, gate_q: torch.Tensor, gate_scales: torch.Tensor, up_q: torch.Tensor,
                      up_scales: torch.Tensor, activation: str = "silu", out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """activation(gate) * up of two int8_linear products of the same rows, in one kernel: neither product is written out."""
    what = "int8_gated_linear"
    _prepare(what, q, scales, (("gate_q", gate_q, gate_scales), ("up_q", up_q, up_scales)), out_dtype)
    _nn.check_modes(what, scales, gate_scales, up_scales)
    _nn.check_no_gradient(what, scales, gate_scales, up_scales)
    if gate_q.shape != up_q.shape:
        raise ValueError(f"{what}: gate_q {tuple(gate_q.shape)} and up_q {tuple(up_q.shape)}")
    act = _nn.activation_code(activation, what)
    n = gate_q.shape[0]
    lib, dev = _nn.load(), _nn.on_device(what, q, scales, gate_q, gate_scales, up_q, up_scales)
    with _nn.on(dev) as cur:
        q2, pq, rows, ldq = _nn.rows_of(q, align=True)
        g2, pg, _, ldg = _nn.rows_of(gate_q, align=True)
        u2, pu, _, ldu = _nn.rows_of(up_q, align=True)
        sq, sg, su = scales.contiguous(), gate_scales.contiguous(), up_scales.contiguous()
        k = q.shape[-1]
        y = torch.empty((rows, n) if q.dim() == 2 else (*q.shape[:-1], n), dtype=out_dtype, device=dev)
        if rows and n:
            size = _nn.size("sdfnn_int8_linear_workspace_size", rows, n, k, 2)
            ws = _nn.workspace(size, dev) if size else None
            _nn.check(lib.sdfnn_int8_gated_linear(pq, ldq, sq.data_ptr(), pg, ldg, sg.data_ptr(), pu, ldu, su.data_ptr(), act,
                                                  _nn.DTYPES[out_dtype], rows, n, k, y.data_ptr(), _nn.ptr(ws), size, cur.stream),
                      "sdfnn_int8_gated_linear")
    return y


class Int8Linear(nn.Module):
    """A trained linear layer in 8 bits: its weight quantised once, by channel; takes the codes and scales of its input."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> None:
        super().__init__()
        codes, scales = quantize_rows(weight.detach())
        self.register_buffer("weight_q", codes)
        self.register_buffer("weight_scales", scales)
        self.register_buffer("bias", bias.detach().float().clone() if bias is not None else None)

    def forward(self, q: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return int8_linear(q, scales, self.weight_q, self.weight_scales, self.bias, out_dtype)
