"""A loss that is trained beside an output (functional.with_loss), on the CPU: what callers may do with the output, and its scale."""
import pytest
import torch

from piper_amd import functional as F_


def leaf():
    return torch.tensor([2.0, 3.0], requires_grad=True)


def test_the_output_may_be_changed_in_place():
    x = leaf()
    out = F_.with_loss(x * 5, (x * x).sum())
    out.reshape(1, 2).add_(x)
    assert torch.equal(out, 6 * x)
    out.mul_(2)
    out.sum().backward()
    assert torch.equal(x.grad, 12 + 2 * x.detach())


def test_a_change_in_place_that_the_backward_needs_is_refused():
    x = leaf()
    h = torch.exp(x)      # keeps its result
    out = F_.with_loss(h, (x * x).sum())
    out.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("scale", [3, 0.5, torch.tensor(4.0), torch.tensor([4.0])])
def test_scale(scale):
    x = leaf()
    out = F_.with_loss(x * 5, (x * x).sum(), scale)
    if isinstance(scale, torch.Tensor):
        scale.fill_(7)                     # between the forward and the backward
    (1024 * out).sum().backward()
    assert torch.equal(x.grad, 1024 * 5 + 2 * float(scale) * x.detach())


def test_compiled():
    @torch.compile(fullgraph=True, backend="eager")
    def step(x):
        return F_.with_loss(x * 5, (x * x).sum(), 2.0).add_(1)
    x = leaf()
    step(x).sum().backward()
    assert torch.equal(x.grad, 5 + 4 * x.detach())
