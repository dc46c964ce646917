"""What the gated block's operators (libsdfnn.so) refuse, copy or look at before they launch anything: no GPU needed."""
import pytest
import torch

from sdfstudio_amd import _nn

P = 4096  # a non-null, 16-byte aligned address nobody reads


def apart(rows, dim, stride, t):
    """rows x dim with `stride` elements between rows (memory that is never touched)."""
    return torch.empty((rows - 1) * stride + dim, dtype=t).as_strided((rows, dim), (stride, 1))


def test_rows_far_apart_are_copied_for_the_products():
    for t, es in ((torch.bfloat16, 2), (torch.float32, 4), (torch.int8, 1)):
        near, far = (1 << 23) // es - 16, (1 << 23) // es
        for stride, copied in ((near, False), (far, True), (far + 16, True)):
            x = apart(3, 32, stride, t)
            x.copy_(torch.arange(96).view(3, 32) % 50)
            kept, at, rows, ld = _nn.rows_of(x, align=True)
            assert rows == 3 and (ld == 32) == copied and (at == x.data_ptr()) == (not copied)
            assert torch.equal(kept, x)
            assert _nn.rows_of(x)[3] == stride  # the norms walk any stride


def test_c_abi_refuses_rows_far_apart_before_it_launches():
    """Also where operands would be copied first (hidden widths that are no multiple of 8)."""
    lib = _nn.load()

    def refused(rc):
        assert rc == -1 and "8 MiB" in _nn.last_error(), (rc, _nn.last_error())

    far16, far8, big = 1 << 22, 1 << 23, 1 << 40
    refused(lib.sdfnn_int8_linear(P, far8, P, P, 64, P, None, 1, 40, 16, 64, P, P, big, None))
    refused(lib.sdfnn_int8_linear(P, 64, P, P, far8, P, None, 1, 40, 16, 64, P, P, big, None))
    refused(lib.sdfnn_int8_gated_linear(P, 64, P, P, 64, P, P, far8, P, 0, 1, 40, 16, 64, P, P, big, None))
    for hidden in (72, 75):
        refused(lib.sdfnn_gated_forward(P, far16, P, P, P, 1, 0, 40, 64, hidden, 64, None, P, P, big, None))
        for rows in (4, 40):
            refused(lib.sdfnn_gated_backward(P, far16, P, P, P, P, P, 64, 1, rows, 64, hidden, 64, P, P, P, P, P, big, None))
            refused(lib.sdfnn_gated_backward(P, 64, P, P, P, P, P, far16, 1, rows, 64, hidden, 64, P, P, P, P, P, big, None))


def every_operator():
    """name -> (call, its floating tensors), on the CPU: what is refused here is refused before the device is looked at."""
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm, rms_norm_quantized
    from sdfstudio_amd.field_components.quantization import int8_gated_linear, int8_linear, quantize_rows

    x, w, r = torch.randn(4, 8), torch.ones(8), torch.randn(4, 8)
    q, s, sw, b = torch.ones(4, 8, dtype=torch.int8), torch.ones(4), torch.ones(4), torch.ones(4)
    return {
        "rms_norm": (lambda x, w, r: rms_norm(x, w, residual=r), (x, w, r)),
        "rms_norm_quantized": (lambda x, w, r: rms_norm_quantized(x, w, residual=r), (x, w, r)),
        "quantize_rows": (quantize_rows, (x,)),
        "int8_linear": (lambda s, sw, b: int8_linear(q, s, q, sw, bias=b), (s, sw, b)),
        "int8_gated_linear": (lambda s, sg, su: int8_gated_linear(q, s, q, sg, q, su), (s, sw, sw.clone())),
        "gated_mlp": (lambda x, g, u, d: gated_mlp(x, g, u, d), (x, torch.randn(6, 8), torch.randn(6, 8), torch.randn(5, 6))),
    }


@pytest.mark.parametrize("name", list(every_operator()))
def test_forward_mode_is_refused(name):
    """A tangent of any input: there is no forward-mode derivative, and a result without a tangent would be a constant to what follows."""
    from torch.autograd import forward_ad

    call, tensors = every_operator()[name]
    for i in range(len(tensors)):
        with forward_ad.dual_level():
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(tensors)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(*args)
    with forward_ad.dual_level(), pytest.raises(_nn.SdfNnError, match="no CPU"):
        call(*tensors)  # no tangent: as ever


@pytest.mark.parametrize("name", list(every_operator()))
def test_graphs_of_operations_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    call, tensors = every_operator()[name]
    with pytest.raises(_nn.SdfNnError, match="make_fx"):
        make_fx(call)(*tensors)
    with FlopCounterMode(display=False), pytest.raises(_nn.SdfNnError, match="no CPU"):  # other modes see the call as ever
        call(*tensors)


@pytest.mark.parametrize("name", ["rms_norm_quantized", "quantize_rows", "int8_linear", "int8_gated_linear"])
def test_traces_of_8_bit_calls_are_refused(name):
    call, tensors = every_operator()[name]
    with torch.no_grad(), pytest.raises(_nn.SdfNnError, match="jit.trace"):
        torch.jit.trace(call, tensors, check_trace=False)


def test_traces_keep_the_calls(monkeypatch):
    """torch.jit.trace keeps rms_norm and gated_mlp as calls, also under torch.no_grad(): a replay on other values computes theirs.  The kernels are
    replaced by their formulas here."""
    from sdfstudio_amd.field_components import mlp, normalization

    def norm(x, weight, residual, eps, save):
        h = x.detach().numpy() + residual.detach().numpy()  # (numpy: as invisible to a trace as a kernel)
        y = torch.from_numpy(h * weight.detach().numpy())
        return y, torch.from_numpy(h), torch.ones(len(h)) if save else None

    def gated(x, w_gate, w_up, w_down, act, save):
        n = [t.detach().numpy() for t in (x, w_gate, w_up, w_down)]
        return torch.from_numpy(((n[0] @ n[1].T) * (n[0] @ n[2].T)) @ n[3].T), torch.ones(1) if save else None

    monkeypatch.setattr(normalization, "_forward", norm)
    monkeypatch.setattr(mlp, "_forward", gated)
    for name in ("rms_norm", "gated_mlp"):
        call, tensors = every_operator()[name]
        with torch.no_grad():
            graph = torch.jit.trace(call, tensors, check_trace=False)
            other = [torch.randn_like(t) for t in tensors]
            got, want = graph(*other), call(*other)
            for a, b in zip(got if isinstance(got, tuple) else [got], want if isinstance(want, tuple) else [want]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["rms_norm_quantized", "int8_linear", "int8_gated_linear"])
def test_calls_without_a_backward_refuse_what_needs_one(name):
    """Each floating input in turn requires a gradient: refused, and served under torch.no_grad() (up to the device)."""
    call, tensors = every_operator()[name]
    for i in range(len(tensors)):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate(tensors)]
        with pytest.raises(_nn.SdfNnError, match="no gradient"):
            call(*args)
        with torch.no_grad(), pytest.raises(_nn.SdfNnError, match="no CPU"):
            call(*args)
    from sdfstudio_amd.field_components.normalization import RMSNorm

    with pytest.raises(_nn.SdfNnError, match="no gradient"):
        RMSNorm(8).quantized(torch.randn(4, 8))  # its weight is a parameter


def test_a_served_form_knows_its_weights(monkeypatch):
    """After an optimiser's step, a load or a move the 8-bit form of a stack is refused until it is made again; training calls, copies and pickles are
    unaffected.  (Kernels left out: the blocks are the identity.)"""
    import copy
    import pickle

    from sdfstudio_amd.engine.optimizers import FlatParameters
    from sdfstudio_amd.field_components import mlp

    monkeypatch.setattr(mlp, "Int8GatedMLP", IdentityBlock)
    monkeypatch.setattr(mlp.RMSNorm, "quantized", lambda self, x, r=None: (x, None) if r is None else (x, None, x))
    monkeypatch.setattr(mlp.RMSNorm, "forward", lambda self, x, r=None: (x, x))
    stack, x = mlp.GatedStack(8, 6, 2), torch.randn(3, 8)

    def serve(s=stack):
        with torch.no_grad():
            return s(x)

    def stale(s=stack):
        with pytest.raises(_nn.SdfNnError, match="since quantize"):
            serve(s)

    stack.quantize()
    serve(), serve()
    for p in (stack.mlps[1].w_down, stack.mlps[0].w_gate):  # torch's optimisers write in place
        with torch.no_grad():
            p.add_(1.0)
        stale()
        stale(copy.deepcopy(stack)), stale(pickle.loads(pickle.dumps(stack)))
        serve(copy.deepcopy(stack.quantize())), serve(pickle.loads(pickle.dumps(stack))), serve()
    other = copy.deepcopy(stack)
    serve(other)
    with torch.no_grad():
        other.mlps[0].w_up.zero_()
    stale(other), serve()
    stack.load_state_dict(other.state_dict())
    stale()
    stack.quantize().load_state_dict(other.state_dict(), assign=True)
    stale()
    with torch.no_grad():
        stack.quantize().norms[0].weight.add_(1.0)  # read as it is
    serve()
    flat = FlatParameters(stack.parameters())  # (moves them)
    stale()
    serve(stack.quantize())
    flat.writes[0] += 1  # what FusedAdam.step does
    stale()
    stack.dequantize()
    monkeypatch.setattr(mlp.GatedMLP, "forward", lambda self, x: x)
    serve()


class IdentityBlock:
    def __init__(self, m):
        pass

    def __call__(self, q, scales, t):
        return q


def product_of(rows, n, k, projections):
    import ctypes

    splits = ctypes.c_int32(-1)
    return _nn.load().sdfnn_int8_product(rows, n, k, projections, ctypes.byref(splits)), splits.value


def test_the_large_tiles_are_tested():
    """The shapes of test_gpu_nn_tiles.py reach the 256 x 256 tiles of every product of the gated block, whole along k and split."""
    from test_gpu_nn_tiles import TILES_16, TILES_F32, TILES_INT8, chosen

    def reached(dtype, shapes):
        return {(i, split) for s in shapes for i, (tile, split) in enumerate(chosen(dtype, s)) if tile == 256}

    assert reached(0, TILES_F32) == {(i, split) for i in range(6) for split in (False, True)}
    for dtype in (1, 2):
        got = reached(dtype, TILES_16)
        assert {i for i, _ in got} == set(range(6)) and {i for i, split in got if split} >= {1, 3, 4, 5}
    assert {(s[3], product_of(*s)[1] > 1) for s in TILES_INT8 if product_of(*s)[0] == 256} == {(p, split) for p in (1, 2) for split in (False, True)}


def test_the_kernel_is_chosen_by_rows_and_size():
    """Few rows stream the weights: up to 32 (fp32: 64, both passes); beyond, tiles, also for the backward pass of few 16-bit rows.  Long products take
    large tiles, narrow ones small tiles, and k is split where tiles are few."""
    from test_gpu_nn_tiles import chosen

    for rows, few in ((1, True), (32, True), (33, False)):
        assert (product_of(rows, 4096, 4096, 2)[0] == 0) == few
        for dtype in (1, 2):
            assert [t == 0 for t, _ in chosen(dtype, (rows, 512, 1024, 512))] == [few, few, False, False, False, False]
    for rows, few in ((1, True), (64, True), (65, False)):
        assert [t == 0 for t, _ in chosen(0, (rows, 512, 1024, 512))] == [few] * 6
    assert product_of(16384, 8192, 4096, 1) == (256, 1) and product_of(524288, 512, 256, 2) == (128, 1)
    assert product_of(200, 64, 131072, 1)[1] > 1
    lib = _nn.load()
    assert lib.sdfnn_int8_product(1, 1, 0, 1, None) == -1 and lib.sdfnn_gated_product(1, 1, 64, 64, 64, 0, 2, None) == -1
    assert lib.sdfnn_gated_product(0, 100, 64, 64, 64, 1, 3, None) in (128, 256) and lib.sdfnn_gated_product(5, 1, 64, 64, 64, 0, 0, None) == -1


@pytest.mark.parametrize("background", ["grid", "none"])
def test_blocks_of_a_background_without_them_are_refused(background):
    """background_feature_blocks belongs to the "mlp" background; another one would train without the blocks it was asked for."""
    from types import SimpleNamespace

    from sdfstudio_amd.models.background import build_background

    with pytest.raises(ValueError, match="background_feature_blocks"):
        build_background(SimpleNamespace(), SimpleNamespace(background_model=background, background_feature_blocks=2))
