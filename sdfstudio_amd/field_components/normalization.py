"""Root-mean-square norm with the residual's addition, as the pre-norm blocks of field_components/mlp.py use it: training form with its
gradients, and a form whose output is the 8-bit codes that field_components/quantization.py multiplies.

Beside the weight norm of the SDF field's layers (csrc/theta_kernels.h), this is the framework's norm over FEATURES.  Runs on libsdfnn.so
(include/sdfnn.h); no CPU path.
"""
from typing import Optional, Tuple, Union

import torch
from torch import nn

from sdfstudio_amd import _nn


def _check(what: str, x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor]) -> None:
    shape, dtype = x.shape, x.dtype
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: x {tuple(x.shape)} has no features")
    if weight is not None and (weight.shape != (shape[-1],) or weight.dtype is not dtype):
        raise ValueError(f"{what}: weight {tuple(weight.shape)} {weight.dtype} for x {tuple(x.shape)} {x.dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype):
        raise ValueError(f"{what}: residual {tuple(residual.shape)} {residual.dtype} for x {tuple(x.shape)} {x.dtype}")


def _forward(x, weight, residual, eps, save):
    """y, h (None without a residual) and, with `save`, inv (else None)."""
    lib, code = _nn.load(), _nn.dtype_code(x, "rms_norm")
    dev = _nn.on_device("rms_norm", x, weight, residual)
    with _nn.on(dev) as cur:
        x2, px, rows, ldx = _nn.rows_of(x)
        r2, pr, _, ldr = _nn.rows_of(residual) if residual is not None else (None, None, 0, 0)
        w = weight.contiguous()
        y = _nn.like(x)
        h = _nn.like(x) if residual is not None else None
        inv = torch.empty(rows, dtype=torch.float32, device=dev) if save else None
        if rows:
            _nn.check(lib.sdfnn_rms_norm_forward(px, ldx, pr, ldr, w.data_ptr(), code, rows, x.shape[-1], eps, y.data_ptr(), _nn.ptr(h),
                                                 _nn.ptr(inv), cur.stream), "sdfnn_rms_norm_forward")
    return y, h, inv


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, inv = _forward(x, weight, residual, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, residual, inv)
        return y if residual is None else (y, h)

    @staticmethod
    @_nn.once
    def backward(ctx, dy, dh=None):
        x, weight, residual, inv = ctx.saved_tensors
        if dy is None and dh is None:
            return None, None, None, None
        lib, code, dev = _nn.load(), _nn.dtype_code(x, "rms_norm"), x.device
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
        need_w = ctx.needs_input_grad[1]
        dim = x.shape[-1]
        with _nn.on(dev) as cur:
            x2, px, rows, ldx = _nn.rows_of(x)
            r2, pr, _, ldr = _nn.rows_of(residual) if residual is not None else (None, None, 0, 0)
            w = weight.contiguous()
            g2, pg, _, ldg = _nn.rows_of(dy) if dy is not None else (None, None, 0, 0)
            k2, pk, _, ldk = _nn.rows_of(dh) if dh is not None else (None, None, 0, 0)
            dx = _nn.like(x) if need_x else None
            dw = _nn.like(weight) if need_w else None
            if rows == 0:
                return dx, dw.zero_() if need_w else None, dx if residual is not None else None, None
            size = _nn.size("sdfnn_rms_norm_backward_workspace_size", rows, dim) if need_w else 0
            ws = _nn.workspace(size, dev) if need_w else None
            _nn.check(lib.sdfnn_rms_norm_backward(px, ldx, pr, ldr, w.data_ptr(), inv.data_ptr(), pg, ldg, pk, ldk, code, rows, dim, _nn.ptr(dx),
                                                  _nn.ptr(dw), _nn.ptr(ws), size, cur.stream), "sdfnn_rms_norm_backward")
        return dx, dw, dx if residual is not None else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension with h = x + residual, the statistic in fp32 from the unrounded sum (values
    beyond 1e19 overflow their squares there).  Returns y, with a residual (y, h).  x [..., dim] in float32 / bfloat16 / float16, weight [dim] and residual of the same type; gradients
    for x, weight and residual (one pass; not differentiable twice)."""
    _check("rms_norm", x, weight, residual)
    _nn.check_modes("rms_norm", x, weight, residual, function=True)
    if not _nn.differentiated(x, weight, residual) and not _nn.traced():
        y, h, _ = _forward(x, weight, residual, float(eps), False)
        return y if residual is None else (y, h)
    return _RMSNorm.apply(x, weight, residual, float(eps))


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """rms_norm with its output in 8 bits: codes int8 [..., dim] in [-127, 127] and scales float32 [...], codes * scales = y to half a step
    of max|y| / 127 a row.  Returns (codes, scales), with a residual (codes, scales, h).  For serving: it has no gradients, and a call that would
    need them is refused."""
    _check("rms_norm_quantized", x, weight, residual)
    _nn.check_no_gradient("rms_norm_quantized", x, weight, residual)
    return _quantize("rms_norm_quantized", x, weight, residual, float(eps))


def _quantize(what: str, x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor], eps: float):
    _nn.check_modes(what, x, weight, residual)
    lib, code = _nn.load(), _nn.dtype_code(x, what)
    dev = _nn.on_device(what, x, weight, residual)
    with _nn.on(dev) as cur:
        x2, px, rows, ldx = _nn.rows_of(x)
        r2, pr, _, ldr = _nn.rows_of(residual) if residual is not None else (None, None, 0, 0)
        w = weight.contiguous() if weight is not None else None
        q = _nn.like(x, torch.int8)
        scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
        h = _nn.like(x) if residual is not None else None
        if rows:
            _nn.check(lib.sdfnn_rms_norm_quantize(px, ldx, pr, ldr, _nn.ptr(w), code, rows, x.shape[-1], eps, q.data_ptr(), scales.data_ptr(),
                                                  _nn.ptr(h), cur.stream), "sdfnn_rms_norm_quantize")
    return (q, scales) if residual is None else (q, scales, h)


class RMSNorm(nn.Module):
    """The norm as a module: weight [dim], ones at the start."""

    def __init__(self, dim: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, residual, self.eps)

    def quantized(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm_quantized(x, self.weight, residual, self.eps)
