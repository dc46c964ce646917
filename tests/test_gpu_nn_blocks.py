"""The gated block's operators together, as the framework uses them: the residual stack and the background field that carries it, training and 8-bit
serving, and what a user's program does around the calls - captured graphs, other streams, strides, empty batches, tensors beyond 2^32 bytes.

Tolerances: see test_gpu_nn_operators.py.  A stack of B blocks passes every value through B sums of products and norms of relative error below
2^-19 each, on magnitudes up to ~8 times the result's (residual additions, gates): 2^-19 * 8 * (2 B + 1) of the tensor's largest value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rms(h, w, eps=1e-6):
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w


def act(name, z):
    return z * torch.sigmoid(z) if name == "silu" else z * 0.5 * torch.erfc(-z / 2 ** 0.5)


def stack_ref(p, x, blocks, name):
    """GatedStack in fp64 from its named parameters."""
    h = x
    for b in range(blocks):
        n = rms(h, p[f"norms.{b}.weight"])
        h = h + (act(name, n @ p[f"mlps.{b}.w_gate"].t()) * (n @ p[f"mlps.{b}.w_up"].t())) @ p[f"mlps.{b}.w_down"].t()
    return rms(h, p[f"norms.{blocks}.weight"])


def make_stack(dim, hidden, blocks, name="silu", dtype=F32):
    from sdfstudio_amd.field_components.mlp import GatedStack

    stack = GatedStack(dim, hidden, blocks, activation=name)
    with torch.no_grad():
        for n in stack.norms:
            n.weight.add_(0.2 * torch.randn(dim))
    return stack.to("cuda", dtype)


def near(name, got, want, rel):
    err = (got.detach().double() - want.detach()).abs().max()
    top = want.detach().abs().max()
    assert float(err) <= rel * float(top), f"{name}: {float(err):.3e} of {float(top):.3e}"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,hidden,blocks,name", [((70,), 48, 1, "gelu"), ((3, 50), 130, 3, "silu"), ((1,), 64, 2, "silu"), ((33, 1, 2), 96, 2, "gelu")])
def test_stack_trains(device, dtype, shape, hidden, blocks, name):
    dim = 72
    stack = make_stack(dim, hidden, blocks, name, dtype)
    x = torch.randn(*shape, dim, device="cuda").to(dtype).requires_grad_(True)
    dy = torch.randn(*shape, dim, device="cuda").to(dtype)
    params = dict(stack.named_parameters())
    y = stack(x)
    grads = torch.autograd.grad(y, [x, *params.values()], dy)
    p = {k: v.detach().double().requires_grad_(True) for k, v in params.items()}
    xd = x.detach().double().requires_grad_(True)
    yd = stack_ref(p, xd, blocks, name)
    want = torch.autograd.grad(yd, [xd, *p.values()], dy.double())
    # 16-bit: y, delta, hidden and residual are rounded in every block (half a step each, up to ~4 times the result's size), and once more on the way back
    rel = {F32: 2.0 ** -19, BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype] * 8 * (2 * blocks + 1)
    near("y", y, yd, rel)
    for k, g, w in zip(["x", *params], grads, want):
        assert g.dtype == dtype
        near(k, g, w, rel)


def test_gradients_against_differences(device):
    stack = make_stack(40, 64, 2)
    x = torch.randn(50, 40, device="cuda", requires_grad=True)
    c = torch.randn(50, 40, device="cuda", dtype=torch.float64)

    def loss():
        return (stack(x).double() * c).sum()

    leaves = [x, *stack.parameters()]
    grads = torch.autograd.grad(loss(), leaves)
    for leaf, g in zip(leaves, grads):
        v = torch.randn_like(leaf)
        v = v / v.norm() * leaf.detach().norm().clamp_min(1.0)
        e = 2.0 ** -9
        with torch.no_grad():
            old = leaf.detach().clone()
            leaf.copy_(old + e * v)
            up = loss()
            leaf.copy_(old - e * v)
            down = loss()
            leaf.copy_(old)
        diff = float((up - down) / (2 * e))
        want = float((g.double() * v.double()).sum())
        # fp32 values: 2^-19 |f| / e; third order: e^2 times the gradient's scale
        assert abs(diff - want) <= 2e-3 * float(g.double().norm() * v.double().norm()) + 0.05, (tuple(leaf.shape), diff, want)


def test_second_derivatives_are_refused(device):
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm

    x, w = torch.randn(40, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(rms_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiat"):
        g.sum().backward()
    ws = [torch.randn(32, 64, device="cuda", requires_grad=True), torch.randn(32, 64, device="cuda"), torch.randn(64, 32, device="cuda")]
    (g,) = torch.autograd.grad(gated_mlp(x, *ws).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiat"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_stack_serves_in_8_bits(device, dtype, rows):
    """8-bit codes of a normal row of 128 are off by 0.7 % (half a step of max / 127 = 3.2 sigma / 127), three products in a row; 5 % of the
    output's norm leaves room for their growth through two blocks."""
    stack = make_stack(128, 256, 2, dtype=dtype)
    x = torch.randn(rows, 128, device="cuda").to(dtype)
    with torch.no_grad():
        plain = stack(x)
    served = stack.quantize()
    with torch.no_grad():
        y = served(x)
    assert y.dtype == dtype and not torch.equal(y, plain)
    want = stack_ref({k: v.detach().double() for k, v in stack.named_parameters()}, x.double(), 2, "silu")
    assert float((y.double() - want).norm() / want.norm()) < 0.05
    assert float((plain.double() - want).norm() / want.norm()) < (1e-5 if dtype == F32 else 0.02)
    xg = x.clone().requires_grad_(True)
    assert torch.equal(stack(xg), plain)  # training calls are unaffected
    keys = set(stack.state_dict())
    assert all(k.split(".")[0] in ("norms", "mlps") and "_q" not in k for k in keys)
    with torch.no_grad():
        assert torch.equal(stack.dequantize()(x), plain)
    stack.quantize().to(F16)
    with torch.no_grad():
        assert stack(x.to(F16)).dtype == F16


def test_background_field_with_feature_blocks(device):
    """NeRFField(feature_blocks): the blocks' share of the field - rgb and every gradient of theirs - against the fp64 stack between the same
    two kernels; density is theirs alone; the field trains and serves."""
    from sdfstudio_amd.cameras.rays import RayBundle
    from sdfstudio_amd.fields.field_heads import FieldHeadNames
    from sdfstudio_amd.fields.vanilla_nerf_field import NeRFEncoding, NeRFField

    n, s = 23, 7
    o = torch.randn(n, 3, device="cuda") * 0.3
    d = torch.nn.functional.normalize(torch.randn(n, 3, device="cuda"), dim=-1)
    starts = torch.sort(torch.rand(n, s, device="cuda") * 2.0, dim=-1)[0]
    rs = RayBundle(origins=o, directions=d, camera_indices=torch.zeros(n, 1, dtype=torch.long, device="cuda"), nears=torch.zeros(n, 1, device="cuda"),
                   fars=torch.full((n, 1), 4.0, device="cuda")).get_ray_samples(starts, starts + 0.2)
    torch.manual_seed(5)
    fld = NeRFField(position_encoding=NeRFEncoding(3, 10, 0.0, 9.0, include_input=True), direction_encoding=NeRFEncoding(3, 4, 0.0, 3.0, include_input=True),
                    feature_blocks=2).to(device)
    out = fld(rs)
    assert out[FieldHeadNames.RGB].shape == (n, s, 3) and out[FieldHeadNames.DENSITY].shape == (n, s, 1)
    cot = torch.randn(n, s, 3, device="cuda")
    names = [k for k, _ in fld.feature_blocks.named_parameters()]
    (out[FieldHeadNames.RGB] * cot).sum().backward()
    got = {k: v.grad.clone() for k, v in fld.feature_blocks.named_parameters()}
    base_grad = fld.mlp_base.layers[0].weight.grad.clone()
    assert all(v.grad is not None for v in fld.mlp_head.parameters())

    stack, fld.feature_blocks = fld.feature_blocks, None
    density, (part, theta, x) = fld.get_density(rs)
    assert torch.equal(density, out[FieldHeadNames.DENSITY])
    p = {k: v.detach().double().requires_grad_(True) for k, v in stack.named_parameters()}
    fld.zero_grad()
    rgb = fld.get_outputs(rs, (stack_ref(p, part.double(), 2, "silu").float(), theta, x))[FieldHeadNames.RGB]
    (rgb * cot).sum().backward()
    assert float((out[FieldHeadNames.RGB] - rgb).detach().abs().max()) < 1e-4  # the colour kernel's own bar
    for k in names:
        near(k, got[k], p[k].grad, 1e-3)
    near("base", base_grad, fld.mlp_base.layers[0].weight.grad.double(), 1e-3)
    fld.feature_blocks = stack
    with torch.no_grad():
        plain = fld(rs)[FieldHeadNames.RGB]
        stack.quantize()
        served = fld(rs)[FieldHeadNames.RGB]
    assert float((plain - rgb.detach()).abs().max()) < 1e-4 and 0 < float((served - plain).abs().max()) < 0.1


# ------------------------------------------------------------------------------------------------ around the calls
def test_empty_batches(device):
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm, rms_norm_quantized
    from sdfstudio_amd.field_components.quantization import int8_gated_linear, int8_linear, quantize_rows

    x, w = torch.zeros(0, 5, 24, device="cuda", requires_grad=True), torch.ones(24, device="cuda", requires_grad=True)
    y, h = rms_norm(x, w, residual=x)
    gx, gw = torch.autograd.grad(y.sum() + h.sum(), (x, w))
    assert y.shape == x.shape and gx.shape == x.shape and gw.shape == (24,) and not gw.any()
    q, s, h = rms_norm_quantized(x.detach(), w.detach(), residual=x.detach())
    assert q.shape == x.shape and s.shape == (0, 5)
    q, s = quantize_rows(x.detach())
    wq, ws = quantize_rows(torch.randn(7, 24, device="cuda"))
    assert int8_linear(q, s, wq, ws).shape == (0, 5, 7) and int8_gated_linear(q, s, wq, ws, wq, ws).shape == (0, 5, 7)
    ws = [torch.randn(16, 24, device="cuda", requires_grad=True), torch.randn(16, 24, device="cuda", requires_grad=True),
          torch.randn(9, 16, device="cuda", requires_grad=True)]
    y = gated_mlp(x, *ws)
    assert y.shape == (0, 5, 9)
    for g, v in zip(torch.autograd.grad(y.sum(), (x, *ws)), (x, *ws)):
        assert g.shape == v.shape and not g.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_offsets_and_partial_gradients(device, dtype):
    """Views give what copies give, bit for bit: rows of a wider tensor, rows that start off a 16-byte boundary, transposed and broadcast
    tensors; and each gradient alone equals its share of all of them."""
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.quantization import int8_linear, quantize_rows

    flat = torch.randn(3 * 48 * 64 + 1, device="cuda").to(dtype)
    ws = [flat[1:1 + 48 * 64].view(48, 64), flat[1 + 48 * 64:1 + 2 * 48 * 64].view(48, 64), flat[1 + 2 * 48 * 64:].view(64, 48)]  # slices of one buffer
    copies = [w.clone() for w in ws]
    wide = torch.randn(90, 200, device="cuda").to(dtype)
    for x in (wide[:, :64], wide[:, 8:72], wide[:, 3:67], wide[::2, :64], wide.t()[:64].t(), wide[:1, :64].expand(90, 64), wide[:20, 5:69]):
        c = x.contiguous()
        assert torch.equal(gated_mlp(x, *ws), gated_mlp(c, *copies))
        dy = torch.randn(2, x.shape[0], 64, device="cuda").to(dtype)[1]
        xs, cs = x.detach().requires_grad_(True), c.detach().clone().requires_grad_(True)
        lw = [w.detach().requires_grad_(True) for w in ws]
        lc = [w.detach().clone().requires_grad_(True) for w in copies]
        for a, b in zip(torch.autograd.grad(gated_mlp(xs, *lw), (xs, *lw), dy), torch.autograd.grad(gated_mlp(cs, *lc), (cs, *lc), dy.clone())):
            assert torch.equal(a, b)
        qa, qb = quantize_rows(x), quantize_rows(c)
        assert torch.equal(qa[0], qb[0]) and torch.equal(qa[1], qb[1])
    x = torch.randn(70, 64, device="cuda").to(dtype)
    dy = torch.randn(70, 64, device="cuda").to(dtype)
    leaves = [v.detach().clone().requires_grad_(True) for v in (x, *copies)]
    every = torch.autograd.grad(gated_mlp(*leaves), leaves, dy)
    for i in range(4):
        one = [v.detach().clone().requires_grad_(i == j) for j, v in enumerate(leaves)]
        (g,) = torch.autograd.grad(gated_mlp(*one), one[i], dy)
        assert torch.equal(g, every[i])
    q = torch.randint(-127, 128, (300, 81), device="cuda", dtype=torch.int8)
    s, sw = torch.rand(300, device="cuda"), torch.rand(40, device="cuda")
    w8 = torch.randint(-127, 128, (40, 100), device="cuda", dtype=torch.int8)
    for k in (64, 63):
        for rows in (300, 9):
            assert torch.equal(int8_linear(q[:rows, 1:1 + k], s[:rows], w8[:, 2:2 + k], sw),
                               int8_linear(q[:rows, 1:1 + k].contiguous(), s[:rows], w8[:, 2:2 + k].contiguous(), sw))


def test_masked_values_stay_in_their_rows(device):
    """An infinity or a NaN in one row reaches that row's outputs and the weights' gradients, no other row."""
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm

    for dtype in (F32, BF16, F16):
        for rows in (20, 150):
            x = torch.randn(rows, 64, device="cuda").to(dtype)
            ws = [torch.randn(*sh, device="cuda").to(dtype) for sh in ((96, 64), (96, 64), (64, 96))]
            w = torch.ones(64, device="cuda").to(dtype)
            want, want_n = gated_mlp(x, *ws), rms_norm(x, w)
            bad = x.clone()
            bad[3, 5], bad[7, 0], bad[9] = float("nan"), float("inf"), torch.finfo(dtype).min
            y, yn = gated_mlp(bad, *ws), rms_norm(bad, w)
            keep = torch.ones(rows, dtype=torch.bool, device="cuda")
            keep[[3, 7, 9]] = False
            assert torch.equal(y[keep], want[keep]) and torch.equal(yn[keep], want_n[keep])
            assert not torch.isfinite(y[3]).any() and not torch.isfinite(y[7]).all() and torch.isnan(yn[3]).all()
            leaf = bad.clone().requires_grad_(True)
            (g,) = torch.autograd.grad(gated_mlp(leaf, *ws), leaf, torch.ones_like(want))
            clean = x.clone().requires_grad_(True)
            (gc,) = torch.autograd.grad(gated_mlp(clean, *ws), clean, torch.ones_like(want))
            assert torch.equal(g[keep], gc[keep])


def test_results_do_not_change_from_run_to_run(device):
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm

    leaves = [torch.randn(*sh, device="cuda").requires_grad_(True) for sh in ((5000, 96), (160, 96), (160, 96), (96, 160))]
    dy, w = torch.randn(5000, 96, device="cuda"), torch.ones(96, device="cuda", requires_grad=True)
    runs = []
    for _ in range(3):
        y = gated_mlp(*leaves)
        n = rms_norm(leaves[0], w)
        runs.append([y, *torch.autograd.grad(y, leaves, dy), n, *torch.autograd.grad(n, (leaves[0], w), dy)])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_captured_and_replayed(device):
    """A training step and a serving step in one graph each, replayed in turn with eager work and new inputs between: every replay equals the
    eager result."""
    stack = make_stack(64, 96, 2)
    params = list(stack.parameters())
    served = make_stack(64, 96, 2).quantize()
    x = torch.randn(200, 64, device="cuda", requires_grad=True)
    x2 = torch.randn(24, 64, device="cuda")
    dy = torch.randn(200, 64, device="cuda")

    def train():
        y = stack(x)
        return [y.detach(), *torch.autograd.grad(y, [x, *params], dy)]

    def serve():
        with torch.no_grad():
            return [served(x2)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train(), serve()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (train, serve):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for r in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(200, 64, device="cuda"))
            x2.copy_(torch.randn(24, 64, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        want = [train(), serve()]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b)), r


def test_two_streams_at_once(device):
    stack = make_stack(128, 256, 2, dtype=BF16)
    xs = [torch.randn(3000, 128, device="cuda").to(BF16) for _ in range(2)]
    with torch.no_grad():
        want = [stack(x) for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(3):
            got = [[], []]
            for s in streams:
                s.wait_stream(torch.cuda.current_stream())
            for _ in range(4):
                for i, s in enumerate(streams):
                    with torch.cuda.stream(s):
                        got[i].append(stack(xs[i]))
            torch.cuda.synchronize()
            for i in range(2):
                assert all(torch.equal(g, want[i]) for g in got[i])


def test_beyond_32_bit_offsets(device):
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows are right, and sums over all rows count every one."""
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm
    from sdfstudio_amd.field_components.quantization import int8_linear, quantize_rows

    rows = (1 << 20) + 7
    x = torch.randn(rows, 2056, device="cuda", dtype=BF16)  # 2.2e9 elements
    w = torch.ones(2056, device="cuda", dtype=BF16, requires_grad=True)
    pick = torch.tensor([0, 5, rows // 2, rows - 2, rows - 1], device="cuda")
    with torch.no_grad():
        y = rms_norm(x, w)
    h = x[pick].double()
    want = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    assert float((y[pick].double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
    del y
    q, s = quantize_rows(x)
    assert float((q[pick].double() * s[pick].double()[:, None] - h).abs().max()) <= 0.51 * float(s[pick].max())
    wq, sw = quantize_rows(torch.randn(2100, 2056, device="cuda"))
    y = int8_linear(q, s, wq, sw, out_dtype=BF16)  # 2.2e9 results
    want = (q[pick].double() @ wq.double().t()) * s[pick].double()[:, None] * sw.double()
    assert float((y[pick].double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
    del y, q, s, x
    x = torch.randn(rows, 64, device="cuda", dtype=BF16, requires_grad=True)
    ws = [torch.randn(2048, 64, device="cuda").div_(8).to(BF16).requires_grad_(True) for _ in range(2)]  # intermediates of 2.1e9 elements
    wd = torch.randn(64, 2048, device="cuda").div_(45).to(BF16).requires_grad_(True)
    y = gated_mlp(x, *ws, wd)
    dy = torch.zeros(rows, 64, device="cuda", dtype=BF16)
    dy[pick] = torch.randn(5, 64, device="cuda").to(BF16)  # the gradients come from the picked rows alone
    grads = torch.autograd.grad(y, (x, *ws, wd), dy)
    small = [v.detach().double().requires_grad_(True) for v in (x.detach()[pick], *ws, wd)]
    yd = (act("silu", small[0] @ small[1].t()) * (small[0] @ small[2].t())) @ small[3].t()
    want = torch.autograd.grad(yd, small, dy[pick].double())
    near("y", y[pick], yd, 2.0 ** -7)
    near("dx", grads[0][pick], want[0], 2.0 ** -6)
    assert int((grads[0].abs().sum(-1) > 0).sum()) == 5
    for g, v in zip(grads[1:], want[1:]):
        near("dw", g, v, 2.0 ** -6)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,dim", [(70001, 24), (33333, 200), (20001, 333), (3001, 1500)])
def test_norm_of_many_rows_with_a_frozen_weight(device, dtype, rows, dim):
    """More rows than one turn of the chip and an odd number of them; the weight has no gradient; rows that start off every boundary."""
    from sdfstudio_amd.field_components.normalization import rms_norm, rms_norm_quantized

    wide = torch.randn(rows, dim + 3, device="cuda").to(dtype)
    x, r = wide[:, 1:1 + dim], torch.randn(rows, dim, device="cuda").to(dtype)
    w = (1 + 0.2 * torch.randn(dim, device="cuda")).to(dtype)
    dy, dh = torch.randn(rows, dim, device="cuda").to(dtype), torch.randn(rows, dim, device="cuda").to(dtype)
    xl, wl = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
    (frozen,) = torch.autograd.grad(rms_norm(xl, w, residual=r), xl, (dy, dh))
    both = torch.autograd.grad(rms_norm(xl, wl, residual=r), (xl, wl), (dy, dh))
    assert torch.equal(frozen, both[0])
    hd = x.double() + r.double()
    inv = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    u, n = dy.double() * w.double(), hd * inv
    want = inv * (u - n * (u * n).mean(-1, keepdim=True)) + dh.double()
    # dx: half a step of the type, and eight of fp32 (inv, n, u, the mean, products and sums) on terms of up to twice the result
    near("dx", frozen, want, torch.finfo(dtype).eps / 2 + 2.0 ** -20)
    # dw: a sum of `rows` fp32 products in chains of at most 100 (a workgroup's turns, its rows, 32 + 32 of the parts): 100 half steps of 2^-24 on the
    # sum of the magnitudes at the worst, a third of that (2^-19) with room for rounding either way
    terms = dy.double() * n
    assert ((both[1].double() - terms.sum(0)).abs() <= 2.0 ** -19 * terms.abs().sum(0) + torch.finfo(dtype).eps / 2 * terms.sum(0).abs()).all()
    q, s, h = rms_norm_quantized(x, w, residual=r)
    v = hd * w.double()
    top = v.abs().amax(-1, keepdim=True)
    assert torch.equal(q.double(), torch.round(127 * v / top))
    near("scales", s, (top * inv / 127).squeeze(-1), 2.0 ** -21)
    near("h", h, hd, torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_codes_of_the_smallest_rows(device, dtype):
    """Rows whose largest value lies among the smallest numbers of the type, where 127 over it exceeds every number: the codes are exact still."""
    from sdfstudio_amd.field_components.quantization import quantize_rows

    x = torch.randn(40, 300, device="cuda", dtype=torch.float64) * torch.logspace(-44, -34, 40, device="cuda", dtype=torch.float64)[:, None]
    x = (x * (1e30 if dtype == F16 else 1.0)).to(dtype)
    q, s = quantize_rows(x)
    v = x.double()
    top = v.abs().amax(-1, keepdim=True)
    assert torch.equal(q.double(), torch.where(top > 0, torch.round(127 * v / torch.where(top > 0, top, 1.0)), 0.0))
    # half a step of fp32, whose smallest is 2^-149
    assert ((s.double() - top[:, 0] / 127).abs() <= 2.0 ** -24 * top[:, 0] / 127 + 2.0 ** -150).all()


def test_model_with_a_background_of_blocks_trains_and_serves(device):
    """background_feature_blocks of a surface model: one optimiser step of the method's own optimisers on flat parameters moves the blocks, and the
    rendered image of the served form stays near the trained one (5 % as in test_stack_serves_in_8_bits; the background is a part of it)."""
    import copy

    import bench as B
    from sdfstudio_amd.cameras.rays import RayBundle
    from sdfstudio_amd.configs.method_configs import method_configs
    from sdfstudio_amd.engine.optimizers import Optimizers
    from sdfstudio_amd.models.neus_facto import SceneBox

    m = method_configs["neus-facto"]
    cfg = copy.deepcopy(m.model)
    cfg.background_model, cfg.background_feature_blocks = "mlp", 2
    torch.manual_seed(0)
    model = cfg.setup(scene_box=SceneBox(aabb=torch.tensor([[-1.0, -1, -1], [1, 1, 1]]), near=0.5, far=4.5), num_train_data=49).to(device).train()
    groups = {k: v for k, v in model.get_param_groups().items() if v}
    opts = Optimizers({k: m.optimizers[k] for k in groups}, groups)
    blocks = model.field_background.feature_blocks
    before = {k: v.detach().clone() for k, v in blocks.named_parameters()}
    gen = torch.Generator(device=device)
    gen.manual_seed(1)
    centers, rot = B.synthetic_cameras(device)
    for step in range(2):
        o, d, norm, cam = B.draw_rays(centers, rot, 256, gen)
        bundle = RayBundle(origins=o, directions=d, directions_norm=norm, camera_indices=cam[:, None])
        loss = model.get_loss_dict(model(bundle), {"image": torch.rand(256, 3, device=device, generator=gen)})
        opts.zero_grad_all()
        sum(loss.values()).backward()
        for k, v in blocks.named_parameters():
            assert torch.isfinite(v.grad).all() and v.grad.any(), k
        opts.optimizer_scaler_step_all(torch.amp.GradScaler("cuda", enabled=False))
        opts.scheduler_step_all(step)  # (the warm-up starts at a rate of zero)
    for k, v in blocks.named_parameters():
        assert torch.isfinite(v).all() and not torch.equal(v, before[k]), k
    model.eval()
    with torch.no_grad():
        plain = model(bundle)["rgb"]
        blocks.quantize()
        served = model(bundle)["rgb"]
    assert torch.isfinite(served).all() and float((served - plain).norm() / plain.norm()) < 0.05


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_grad_keeps_nothing(device, dtype):
    """Under torch.no_grad() a module, whose parameters require gradients, neither writes nor holds what a backward pass would read, and gives the same
    values."""
    from sdfstudio_amd.field_components.mlp import GatedMLP, GatedStack

    mlp = GatedMLP(64, 512).to("cuda", dtype)
    x = torch.randn(40000, 64, device="cuda").to(dtype)
    want = mlp(x)
    assert want.requires_grad
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        y = mlp(x)
    # the hidden rows in the type (fp32: three parts) and x's and the weights' parts; act(g) and u act'(g) would be 40000 x 512 x 8 bytes more
    assert torch.cuda.max_memory_allocated() - before < 40000 * 512 * (6 if dtype == F32 else 2) + 40000 * 64 * 16 + (4 << 20)
    assert torch.equal(y, want) and not y.requires_grad
    stack = GatedStack(64, 128, 2).to("cuda", dtype)
    want = stack(x)
    with torch.inference_mode():
        assert torch.equal(stack(x), want)
    for p in stack.parameters():
        p.requires_grad_(False)
    assert torch.equal(stack(x), want) and not stack(x).requires_grad


def test_more_rows_than_one_launch_has_threads(device):
    """A launch has less than 2^32 threads: norms of narrow rows beyond 2^29 and of wide ones beyond 2^21, operand copies of more than 2^35 elements
    and products of 2^31 - 1 rows come in pieces; rows at every border are right."""
    from sdfstudio_amd.field_components.normalization import rms_norm
    from sdfstudio_amd.field_components.quantization import int8_linear, quantize_rows

    def rows_at(*borders):
        return torch.tensor([b + i for b in borders for i in range(-3, 3)], device="cuda")

    rows = (1 << 29) + 70
    pick = rows_at(3, 1 << 28, 1 << 29, rows - 3)
    x = torch.zeros(rows, 2, device="cuda", dtype=BF16)
    x[pick] = torch.randn(len(pick), 2, device="cuda").to(BF16)
    w = torch.tensor([1.0, 2.0], device="cuda", dtype=BF16)
    h = x[pick].double().requires_grad_(True)
    want = rms(h, w.double())
    leaf = x.requires_grad_(True)
    y = rms_norm(leaf, w)
    near("y", y[pick], want, 2.0 ** -8)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    (dh,) = torch.autograd.grad(want, h, torch.ones_like(want))
    # dx is a difference of terms: half a step of bf16, and 2^-20 of inv times the largest weight, each
    inv = 1.0 / torch.sqrt(h.detach().square().mean(-1, keepdim=True) + 1e-6)
    assert ((dx[pick].double() - dh).abs() <= 2.0 ** -8 * dh.abs() + 2.0 ** -19 * 2.0 * inv).all()
    del y, dx
    q, s = quantize_rows(leaf)
    top = h.detach().abs().amax(-1, keepdim=True)
    assert torch.equal(q[pick].double(), torch.round(127 * h.detach() / top)) and not q[10:1000].any() and not s[10:1000].any()
    del q, s, x, leaf
    rows = (1 << 28) + 100
    q = torch.randint(-127, 128, (rows, 1), device="cuda", dtype=torch.int8)
    s, wq, sw = torch.rand(rows, device="cuda"), torch.tensor([[5], [-7]], device="cuda", dtype=torch.int8), torch.tensor([0.5, 0.25], device="cuda")
    y = int8_linear(q, s, wq, sw)
    for i in range(2):
        assert torch.equal(y[:, i], q[:, 0] * wq[i].float() * s * sw[i])
    del q, s, y
    torch.cuda.empty_cache()
    rows = (1 << 31) - 1
    pick = rows_at(3, 1 << 30, rows - 3)
    q = torch.zeros(rows, 16, device="cuda", dtype=torch.int8)
    q[pick] = torch.randint(-127, 128, (len(pick), 16), device="cuda", dtype=torch.int8)
    wq = torch.randint(-127, 128, (1, 16), device="cuda", dtype=torch.int8)
    y = int8_linear(q, torch.ones(rows, device="cuda"), wq, torch.ones(1, device="cuda"))
    assert torch.equal(y[pick].double(), q[pick].double() @ wq.double().t()) and not y[10:1000].any()
    del q, y
    torch.cuda.empty_cache()
    rows = (1 << 21) + 5
    pick = rows_at(3, 1 << 20, 1 << 21, rows - 3)
    x = torch.zeros(rows, 8200, device="cuda", dtype=F16)
    x[pick] = torch.randn(len(pick), 8200, device="cuda").to(F16)
    q, s = quantize_rows(x)
    v = x[pick].double()
    assert torch.equal(q[pick].double(), torch.round(127 * v / v.abs().amax(-1, keepdim=True))) and not s[10:1000].any()
    del x, q, s
    torch.cuda.empty_cache()
