"""Which of its ways a module with a balance loss takes, on the CPU."""
import torch
from torch import nn

from piper_amd.moe import AnnotatedMoE, MoEArgs, MoEFeedForwardBlock


class Doubling(nn.Module):
    """Somebody else's experts, which know nothing of a balance loss."""

    fused = True

    def forward(self, x, residual):
        return residual + 2 * x


def test_a_block_with_somebody_elses_experts():
    block = MoEFeedForwardBlock(MoEArgs(), 8, 8)
    block.ffn_norm, block.moe = nn.Identity(), Doubling()
    x = torch.randn(1, 3, 8)
    assert torch.equal(block(x), 3 * x)
    del Doubling.fused
    assert torch.equal(block(x), 3 * x)


def test_without_gradients_a_block_is_the_one_without_a_loss():
    plain, with_it = (MoEFeedForwardBlock(MoEArgs(num_experts=4, top_k=2, **more), 16, 8) for more in ({}, dict(balance_loss_coeff=0.1)))
    assert plain._one_node() and not with_it._one_node()
    with torch.no_grad():
        assert plain._one_node() and with_it._one_node()
        with_it.moe.balance_loss_without_grad = True
        assert not with_it._one_node()
    assert isinstance(with_it.moe, AnnotatedMoE) and not AnnotatedMoE.balance_loss_without_grad
