"""What a saved-tensor hook hands back in place of V-trace's kept values is checked before the backward kernel reads it."""
import pytest
import torch

from torchrl_amd.objectives.value import functional as F


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_vtrace(device):
    g = torch.Generator().manual_seed(0)
    lp, lm, v, nv, r = (torch.randn(4, 9, 1, generator=g).to(device) for _ in range(5))
    done = (torch.rand(4, 9, 1, generator=g) < 0.2).to(device)

    def gradients(change):
        leaves = [x.clone().requires_grad_() for x in (lp, v, r)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            adv, _ = F.vtrace_advantage_estimate(0.9, leaves[0], lm, leaves[1], nv, leaves[2], done)
        return torch.autograd.grad(adv.sum(), leaves)

    want = gradients(lambda t: t)
    for a, b in zip(gradients(lambda t: t.double()), want):
        assert torch.equal(a, b)
    for a, b in zip(gradients(lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)), want):
        assert torch.equal(a, b)
    for change in [lambda t: t[:-1], lambda t: t[:, :3]] + ([lambda t: t.cpu()] if device == "cuda" else []):
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            gradients(change)
