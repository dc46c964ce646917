"""The gated block's operators (libsdfnn.so) inside what a user's program does around them: traces, modes, optimisers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_traces_replay_on_other_values(device):
    from sdfstudio_amd.field_components.mlp import gated_mlp
    from sdfstudio_amd.field_components.normalization import rms_norm

    def draw():
        return [torch.randn(*s, device="cuda") for s in ((40, 64), (64,), (48, 64), (48, 64), (64, 48))]

    def block(x, w, wg, wu, wd):
        return x + gated_mlp(rms_norm(x, w), wg, wu, wd)

    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            args = [t.requires_grad_(grad) for t in draw()]
            graph = torch.jit.trace(block, args, check_trace=False)
            for _ in range(2):
                other = draw()
                assert torch.equal(graph(*other), block(*other))


def test_a_served_stack_follows_its_weights(device):
    """quantize(), then a step of the fused optimiser or load_state_dict: the next served call raises, and after another quantize() equals that of a
    stack that has held these weights from the start."""
    import copy

    from sdfstudio_amd._nn import SdfNnError
    from sdfstudio_amd.engine.optimizers import Optimizers
    from sdfstudio_amd.field_components.mlp import GatedStack

    stack, x = GatedStack(64, 96, 2).to(device), torch.randn(50, 64, device=device)
    opts = Optimizers({"blocks": {"lr": 0.1}}, {"blocks": list(stack.parameters())})

    def check():
        with torch.no_grad():
            with pytest.raises(SdfNnError, match="since quantize"):
                stack(x)
            y = stack.quantize()(x)
            fresh = GatedStack(64, 96, 2).to(device)
            fresh.load_state_dict(stack.state_dict())
            assert torch.equal(y, fresh.quantize()(x)) and torch.equal(y, copy.deepcopy(stack)(x)) and torch.equal(y, stack(x))

    before = copy.deepcopy(stack.state_dict())
    stack.quantize()
    for _ in range(2):
        opts.zero_grad_all()
        stack(x).square().sum().backward()
        opts.optimizer_step_all()
        check()
    assert not torch.equal(before["mlps.0.w_up"], stack.mlps[0].w_up)
    stack.load_state_dict(before)
    check()
    stack.to(torch.bfloat16)  # makes the form anew
    with torch.no_grad():
        assert stack(x.bfloat16()).dtype == torch.bfloat16
