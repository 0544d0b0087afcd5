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
