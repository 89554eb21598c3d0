"""The step's attention inputs on the CPU (no GPU call: the projections here are torch's)."""

import pytest
import torch

from mlx_tree_spec_amd import AttentionInputs, attention_inputs


class Projection(torch.nn.Module):
    def __init__(self, n):
        super().__init__()
        self.n = n

    def forward(self, x):
        return x[..., :1].expand(*x.shape[:-1], self.n).contiguous()


def layer(q, gated):
    norm = torch.nn.RMSNorm(64, eps=1e-6, dtype=torch.bfloat16)
    return AttentionInputs(Projection(q), Projection(2 * 64), Projection(2 * 64), norm, norm, 4, 2, 64, torch.ones(16), gated)


@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 2), (1,)])
@pytest.mark.parametrize("gated", [False, True])
def test_any_number_of_rows(lead, gated):
    """A step of no rows comes as far as one with rows does on the CPU: to the head norms."""
    x = torch.zeros(*lead, 8, dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
        attention_inputs(x, layer(4 * 64 * (1 + gated), gated), torch.zeros(lead, dtype=torch.int32))


@pytest.mark.parametrize("lead", [(0,), (2,)])
@pytest.mark.parametrize("q,gated", [(4 * 64, True), (8 * 64, False), (4 * 64 + 8, False), (4 * 65, False)])
def test_widths_that_do_not_match_are_refused(lead, q, gated):
    x = torch.zeros(*lead, 8, dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(ValueError, match="q_proj"):
        attention_inputs(x, layer(q, gated), torch.zeros(lead, dtype=torch.int32))
