"""ctypes binding of libsdfnn.so (the C ABI declared in include/sdfnn.h): the gated feed-forward block's operators.

No fallback, as _lib.py: a missing library or a failing call raises.  PyTorch provides device memory and the stream.
"""
import ctypes
import functools
import os
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("SDFNN_LIB", os.path.join(_HERE, "libsdfnn.so"))

_p, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
_SIGNATURES = {
    "sdfnn_version": (ctypes.c_int, []),
    "sdfnn_last_error": (ctypes.c_char_p, []),
    "sdfnn_rms_norm_forward": (ctypes.c_int, [_p, _i64, _p, _i64, _p, _i32, _i64, _i64, _f32, _p, _p, _p, _p]),
    "sdfnn_rms_norm_backward_workspace_size": (_i64, [_i64, _i64]),
    "sdfnn_rms_norm_backward": (ctypes.c_int, [_p, _i64, _p, _i64, _p, _p, _p, _i64, _p, _i64, _i32, _i64, _i64, _p, _p, _p, _i64, _p]),
    "sdfnn_rms_norm_quantize": (ctypes.c_int, [_p, _i64, _p, _i64, _p, _i32, _i64, _i64, _f32, _p, _p, _p, _p]),
    "sdfnn_int8_linear_workspace_size": (_i64, [_i64, _i64, _i64, _i32]),
    "sdfnn_int8_product": (_i32, [_i64, _i64, _i64, _i32, _p]),
    "sdfnn_int8_linear": (ctypes.c_int, [_p, _i64, _p, _p, _i64, _p, _p, _i32, _i64, _i64, _i64, _p, _p, _i64, _p]),
    "sdfnn_int8_gated_linear": (ctypes.c_int, [_p, _i64, _p, _p, _i64, _p, _p, _i64, _p, _i32, _i32, _i64, _i64, _i64, _p, _p, _i64, _p]),
    "sdfnn_gated_saved_size": (_i64, [_i32, _i64, _i64, _i64]),
    "sdfnn_gated_workspace_size": (_i64, [_i32, _i64, _i64, _i64, _i64, _i32]),
    "sdfnn_gated_product": (_i32, [_i32, _i64, _i64, _i64, _i64, _i32, _i32, _p]),
    "sdfnn_gated_forward": (ctypes.c_int, [_p, _i64, _p, _p, _p, _i32, _i32, _i64, _i64, _i64, _i64, _p, _p, _p, _i64, _p]),
    "sdfnn_gated_backward": (ctypes.c_int, [_p, _i64, _p, _p, _p, _p, _p, _i64, _i32, _i64, _i64, _i64, _i64, _p, _p, _p, _p, _p, _i64, _p]),
}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
ROW_REACH = 1 << 23  # bytes between rows from which the products do not read them in place
_lib: Optional[ctypes.CDLL] = None


class SdfNnError(RuntimeError):
    pass


def load() -> ctypes.CDLL:
    """Load libsdfnn.so; raises if it has not been built (python -m sdfstudio_amd.build / __graft_entry__.build())."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise SdfNnError(f"{LIB_PATH} is missing: build the HIP extensions first (python -m sdfstudio_amd.build). "
                         "There is no CPU fallback for the gated block.")
    lib = ctypes.CDLL(LIB_PATH)
    for name, (restype, argtypes) in _SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError if the symbol is not exported
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = lib
    return lib


def last_error() -> str:
    return (load().sdfnn_last_error() or b"").decode(errors="replace")


def check(rc: int, what: str):
    if rc != 0:
        raise SdfNnError(f"{what} failed ({rc}): {last_error()}")


def dtype_code(t: torch.Tensor, what: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: {t.dtype} is not supported (float32, bfloat16, float16)")
    return code


def activation_code(name: str, what: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"{what}: activation {name!r}: one of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def on_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """The one HIP device that every tensor of a call lives on."""
    if not first.is_cuda:
        raise SdfNnError(f"{what} runs on the sdfnn kernels: HIP device tensors required (no CPU fallback)")
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")
    return first.device


def rows_of(t: torch.Tensor, align: bool = False) -> Tuple[torch.Tensor, int, int, int]:
    """t [..., dim] as rows the kernels can walk: (tensor to keep alive, its address, rows, row stride in elements).  The tensor itself or a
    view wherever that is possible; a copy for rows that are not adjacent in memory, overlap, or - with `align`, for the products - do not start at
    16-byte boundaries although their width would allow it or are 8 MiB and more apart."""
    dim = t.shape[-1]
    whole = align and dim * t.element_size() % 16 == 0
    if t.is_contiguous():
        at = t.data_ptr()
        if not (whole and at % 16):
            return t, at, t.numel() // dim, dim
    rows = t.numel() // dim
    t2 = t.reshape(rows, dim)
    stride = t2.stride(0) if rows > 1 else dim
    if (dim > 1 and t2.stride(1) != 1) or stride < dim or (align and stride * t2.element_size() >= ROW_REACH) or \
            (whole and (t2.data_ptr() % 16 or stride * t2.element_size() % 16)):
        t2, stride = t2.clone(memory_format=torch.contiguous_format), dim
    return t2, t2.data_ptr(), rows, stride


def aligned(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor that starts at a 16-byte boundary where the kernels read it in place (16-bit types; a slice of a flat parameter
    buffer may not)."""
    t = t.contiguous()
    return t if t.element_size() == 4 or t.data_ptr() % 16 == 0 else t.clone()


def ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def like(t: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A contiguous uninitialised tensor of t's shape (empty_like, half the host time of empty, where it makes one)."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device)


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Scratch memory of one call, from the caching allocator: it goes back when the call has been issued, in stream order, and inside a
    graph capture it belongs to that graph's pool - no two calls or graphs share one."""
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


# the stream's handle without the Stream object around it (1 us of a call's host time)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def differentiated(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a call on these is recorded for a backward pass.  (Inside an autograd function it cannot be told: its needs_input_grad does not
    know about torch.no_grad().)"""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# whether torch.jit.trace is recording: it keeps autograd functions as calls, nothing else of these operators
traced = getattr(torch._C, "_is_tracing", None) or torch.jit.is_tracing
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None) or (lambda: 1)


def check_modes(what: str, *tensors: Optional[torch.Tensor], function: bool = False) -> None:
    """Refuses what torch would take further without knowing that a kernel was there: tangents of forward-mode differentiation, which the result
    would have lost, and graphs recorded tensor operation by tensor operation (make_fx; torch.jit.trace, unless the call is an autograd `function`),
    which would hold the allocation of the outputs alone."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")
    if _modes():
        from torch.fx.experimental.proxy_tensor import get_proxy_mode  # (takes a second; here it has been imported)

        if get_proxy_mode() is not None:
            raise SdfNnError(f"{what} runs on the sdfnn kernels, which a graph of torch operations (make_fx) cannot hold")
    if not function and traced():
        raise SdfNnError(f"{what} runs on the sdfnn kernels, which torch.jit.trace cannot record")


def check_no_gradient(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses a call that would be recorded for a backward pass, by an operator that has none."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise SdfNnError(f"{what} has no gradient: call it under torch.no_grad() or on tensors that require none")


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _NotTwice(torch.autograd.Function):
    """The gradients of a backward pass whose graph is recorded, tied to what they depend on: differentiating them is an error, not zero."""

    @staticmethod
    def forward(ctx, count, *tensors):
        return tuple(t.detach() for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("sdfnn operators cannot be differentiated twice: their backward pass has no derivative of its own")


def once(backward):
    """A backward whose results cannot be differentiated again.  torch's once_differentiable lets them pass as constants where the incoming
    gradient is one, and costs 20 us of host time in every call; here the graph, where one is recorded, leads to an error."""

    @functools.wraps(backward)
    def call(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        there = [t for t in out if t is not None]
        depends = [t for t in (*ctx.saved_tensors, *grads) if isinstance(t, torch.Tensor) and t.requires_grad]
        guarded = iter(_NotTwice.apply(len(there), *there, *depends))
        return tuple(None if t is None else next(guarded) for t in out)

    return call


class on:
    """The call's device as the current one for the length of a `with` block (nothing is touched where it is already); `.stream` is its
    current stream."""

    __slots__ = ("device", "stream", "before")

    def __init__(self, device: torch.device) -> None:
        self.device = device

    def __enter__(self) -> "on":
        index = self.device.index
        before = _current_device()
        self.before = before if before != index else None
        if self.before is not None:
            torch.cuda.set_device(index)
        self.stream = _raw_stream(index)
        return self

    def __exit__(self, *exc) -> None:
        if self.before is not None:
            torch.cuda.set_device(self.before)


@functools.lru_cache(maxsize=4096)
def size(query: str, *args: int) -> int:
    """A size query of the library (a function of sizes alone)."""
    n = getattr(load(), query)(*args)
    if n < 0:
        raise SdfNnError(f"{query}{args}: refused")
    return n
