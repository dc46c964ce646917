"""libsdfnn.so without a GPU: the C ABI's declarations, the binding, sizes, and every refusal (arguments are checked before anything is launched,
so a call that is refused needs no device)."""
import ctypes
import os
import re

import pytest
import torch

from sdfstudio_amd import _nn
from sdfstudio_amd.field_components.mlp import GatedMLP, GatedStack, gated_mlp
from sdfstudio_amd.field_components.normalization import RMSNorm, rms_norm, rms_norm_quantized
from sdfstudio_amd.field_components.quantization import int8_gated_linear, int8_linear, quantize_rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # a non-null, 16-byte aligned address nobody reads


def test_header_binding_and_library_agree():
    src = open(os.path.join(ROOT, "include", "sdfnn.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    declared = dict(re.findall(r"(sdfnn_\w+)\s*\(([^;]*)\)\s*;", src))
    assert set(declared) == set(_nn._SIGNATURES)
    lib = ctypes.CDLL(_nn.LIB_PATH)
    for name, args in declared.items():
        assert hasattr(lib, name), name
        n = 0 if args.strip() == "void" else len(args.split(","))
        assert n == len(_nn._SIGNATURES[name][1]), name
    assert _nn.load().sdfnn_version() >= 100


def refused(rc, *words):
    assert rc != 0
    msg = _nn.last_error()
    assert all(w in msg for w in words), msg


def test_c_abi_refuses_bad_calls():
    lib = _nn.load()
    norm = lib.sdfnn_rms_norm_forward
    ok = [P, 8, None, 0, P, 0, 4, 8, 1e-6, P, None, None, None]

    def call(fn, base, **change):
        a = list(base)
        for k, v in change.items():
            a[int(k[1:])] = v
        return fn(*a)

    refused(call(norm, ok, _0=None), "null")
    refused(call(norm, ok, _4=None), "null")
    refused(call(norm, ok, _1=7), "stride")
    refused(call(norm, ok, _2=P, _3=7), "stride")
    refused(call(norm, ok, _5=3), "dtype")
    refused(call(norm, ok, _6=-1), "rows")
    refused(call(norm, ok, _7=0), "elements")
    refused(call(norm, ok, _8=-1.0), "eps")
    refused(call(norm, ok, _8=float("nan")), "eps")
    assert call(norm, ok, _6=0) == 0  # nothing to do
    bwd = lib.sdfnn_rms_norm_backward
    ok = [P, 8, None, 0, P, P, P, 8, None, 0, 0, 4, 8, P, P, P, 1 << 20, None]
    refused(call(bwd, ok, _6=None), "neither")
    refused(call(bwd, ok, _16=3), "workspace")
    refused(call(bwd, ok, _15=None), "workspace")
    refused(call(bwd, ok, _7=5), "stride")
    assert call(bwd, ok, _13=None, _14=None) == 0
    q = lib.sdfnn_rms_norm_quantize
    refused(q(P, 8, None, 0, None, 0, 4, 8, 0.0, None, P, None, None), "null")
    lin = lib.sdfnn_int8_linear
    ok = [P, 64, P, P, 64, P, None, 1, 40, 16, 64, P, P, 1 << 30, None]
    refused(call(lin, ok, _10=131073, _1=131073, _4=131073), "131072")
    refused(call(lin, ok, _10=0), "k = 0")
    refused(call(lin, ok, _9=0), "channels")
    refused(call(lin, ok, _1=63), "stride")
    refused(call(lin, ok, _0=P + 1), "16-byte")
    refused(call(lin, ok, _1=72), "16-byte")
    refused(call(lin, ok, _7=5), "dtype")
    refused(call(lin, ok, _8=200, _9=64, _10=8192, _1=8192, _4=8192, _13=16), "workspace")
    gl = lib.sdfnn_int8_gated_linear
    ok = [P, 64, P, P, 64, P, P, 64, P, 0, 1, 40, 16, 64, P, P, 1 << 30, None]
    refused(call(gl, ok, _9=7), "activation")
    refused(call(gl, ok, _6=None), "null")
    fwd = lib.sdfnn_gated_forward
    ok = [P, 64, P, P, P, 1, 0, 40, 64, 128, 64, None, P, P, 1 << 30, None]
    refused(call(fwd, ok, _6=9), "activation")
    refused(call(fwd, ok, _8=0), "widths")
    refused(call(fwd, ok, _9=(1 << 20) + 1), "widths")
    refused(call(fwd, ok, _1=63), "stride")
    refused(call(fwd, ok, _0=P + 2), "16-byte")
    refused(call(fwd, ok, _4=P + 2), "16-byte")
    refused(call(fwd, ok, _11=P + 4), "saved")
    refused(call(fwd, ok, _14=64), "workspace")
    refused(call(fwd, ok, _13=P + 8), "workspace")
    gb = lib.sdfnn_gated_backward
    ok = [P, 64, P, P, P, P, P, 64, 1, 40, 64, 128, 64, P, P, P, P, P, 1 << 30, None]
    refused(call(gb, ok, _14=None), "together")
    refused(call(gb, ok, _7=63), "stride")
    refused(call(gb, ok, _6=P + 2), "16-byte")
    refused(call(gb, ok, _18=64), "workspace")
    assert lib.sdfnn_gated_workspace_size(1, -1, 64, 64, 64, 0) == -1 and lib.sdfnn_gated_saved_size(7, 1, 1, 1) == -1
    assert lib.sdfnn_int8_linear_workspace_size(1, 1, 131073, 1) == -1 and lib.sdfnn_rms_norm_backward_workspace_size(1, 0) == -1


def test_workspaces_are_sized_by_the_call():
    """Few rows need no copies; a product that is read where it lies needs no workspace; copies and split sums are accounted for."""
    lib = _nn.load()
    assert lib.sdfnn_int8_linear_workspace_size(32, 4096, 4096, 2) == 0
    assert lib.sdfnn_int8_linear_workspace_size(1 << 20, 4096, 4096, 1) == 0
    assert lib.sdfnn_int8_linear_workspace_size(1 << 16, 512, 1000, 1) >= (1 << 16) * 1024 + 512 * 1024
    for dt, es in ((0, 4), (1, 2), (2, 2)):
        a = lib.sdfnn_gated_workspace_size(dt, 1000, 64, 100, 64, 0)
        assert a >= 1000 * 128 * es
        assert lib.sdfnn_gated_workspace_size(dt, 1000, 64, 100, 64, 1) >= 1000 * 256 * es
        assert lib.sdfnn_gated_saved_size(dt, 1000, 60, 100) == 1000 * 128 * (8 + (6 if dt == 0 else 2)) + (1000 * 64 * 6 if dt == 0 else 0)
        assert lib.sdfnn_gated_saved_size(dt, 20, 60, 100) == 20 * 128 * (8 + es)


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.ones(8)
    for call in (lambda: rms_norm(x, w), lambda: rms_norm_quantized(x, w), lambda: quantize_rows(x), lambda: RMSNorm(8)(x),
                 lambda: gated_mlp(x, torch.randn(6, 8), torch.randn(6, 8), torch.randn(8, 6)), lambda: GatedMLP(8, 6)(x),
                 lambda: GatedStack(8, 6, 2)(x), lambda: GatedStack(8, 6, 2).quantize(),
                 lambda: int8_linear(x.to(torch.int8), torch.ones(4), x.to(torch.int8), torch.ones(4))):
        with pytest.raises(_nn.SdfNnError, match="no CPU"):
            call()


def test_shapes_and_types_are_refused():
    x, w = torch.randn(4, 8), torch.ones(8)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    for err, call in [
        (ValueError, lambda: rms_norm(x, torch.ones(7))),
        (ValueError, lambda: rms_norm(x, w.half())),
        (ValueError, lambda: rms_norm(x, w, residual=x[:2])),
        (ValueError, lambda: rms_norm(x, w, residual=x.half())),
        (ValueError, lambda: rms_norm(torch.zeros(3, 0), torch.zeros(0))),
        (ValueError, lambda: quantize_rows(torch.zeros(()))),
        (TypeError, lambda: rms_norm(x.double(), w.double())),
        (TypeError, lambda: quantize_rows(q)),
        (TypeError, lambda: int8_linear(x, s, q, s)),
        (ValueError, lambda: int8_linear(q, s[:3], q, s)),
        (ValueError, lambda: int8_linear(q, s.half(), q, s)),
        (ValueError, lambda: int8_linear(q, s, q[:, :7], s)),
        (ValueError, lambda: int8_linear(q, s, q, s, bias=torch.ones(5))),
        (ValueError, lambda: int8_linear(q, s, q, s, bias=torch.ones(4).half())),
        (TypeError, lambda: int8_linear(q, s, q, s, out_dtype=torch.float64)),
        (ValueError, lambda: int8_linear(q.new_zeros(4, 131073), s, q.new_zeros(2, 131073), s[:2])),
        (ValueError, lambda: int8_gated_linear(q, s, q, s, q[:3], s[:3])),
        (ValueError, lambda: int8_gated_linear(q, s, q, s, q, s, activation="tanh")),
        (ValueError, lambda: gated_mlp(x, torch.randn(6, 7), torch.randn(6, 7), torch.randn(8, 6))),
        (ValueError, lambda: gated_mlp(x, torch.randn(6, 8), torch.randn(5, 8), torch.randn(8, 6))),
        (ValueError, lambda: gated_mlp(x, torch.randn(6, 8), torch.randn(6, 8), torch.randn(8, 5))),
        (ValueError, lambda: gated_mlp(x, torch.randn(0, 8), torch.randn(0, 8), torch.randn(8, 0))),
        (TypeError, lambda: gated_mlp(x.half(), torch.randn(6, 8), torch.randn(6, 8), torch.randn(8, 6))),
        (ValueError, lambda: gated_mlp(x, torch.randn(6, 8), torch.randn(6, 8), torch.randn(8, 6), activation="tanh")),
        (ValueError, lambda: GatedMLP(8, 6, activation="tanh")),
        (ValueError, lambda: GatedStack(8, 6, 0)),
    ]:
        with pytest.raises(err):
            call()


def test_stack_and_field_parameters():
    """The stack's state_dict holds its parameters alone, and the background field has one only when it is asked for."""
    from sdfstudio_amd.fields.vanilla_nerf_field import NeRFEncoding, NeRFField

    stack = GatedStack(8, 12, 2)
    assert {k: tuple(v.shape) for k, v in stack.state_dict().items()} == {
        "norms.0.weight": (8,), "norms.1.weight": (8,), "norms.2.weight": (8,),
        "mlps.0.w_gate": (12, 8), "mlps.0.w_up": (12, 8), "mlps.0.w_down": (8, 12),
        "mlps.1.w_gate": (12, 8), "mlps.1.w_up": (12, 8), "mlps.1.w_down": (8, 12)}

    def field(**kw):
        return NeRFField(position_encoding=NeRFEncoding(3, 10, 0.0, 9.0, include_input=True),
                         direction_encoding=NeRFEncoding(3, 4, 0.0, 3.0, include_input=True), **kw)

    plain, with_blocks = field(), field(feature_blocks=2)
    extra = set(with_blocks.state_dict()) - set(plain.state_dict())
    assert extra == {"feature_blocks." + k for k in GatedStack(128, 256, 2).state_dict()}
    assert set(plain.state_dict()) <= set(with_blocks.state_dict())
    from sdfstudio_amd.models.neus_facto import NeuSFactoModelConfig

    assert NeuSFactoModelConfig().background_feature_blocks == 0
