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
