"""Sampling of rows in several batches (needs an MI355X): the lists' bound ends a batch before its number of rows does.
Counts are whole numbers, so a row's result does not hang on the batch it is in."""

import pytest
import torch

from mlx_tree_spec_amd import sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("m,v", [(18, 1 << 24), (300, 1000003)])
def test_each_row_as_alone(m, v):
    g = torch.Generator(device=DEV).manual_seed(m)
    logits = torch.empty(m, v, dtype=torch.bfloat16, device=DEV)
    for i in range(m):
        logits[i] = torch.randn(v, generator=g, device=DEV) * 2
    u = torch.rand(m, generator=g, device=DEV)
    settings = dict(temperature=0.5 + torch.rand(m, generator=g, device=DEV), top_p=0.9)
    tokens, logprobs = sample(logits, u, **settings)
    for i in sorted({0, 1, m // 2, m - 3, m - 2, m - 1} | set(range(0, m, 7))):
        one, p = sample(logits[i], u[i], temperature=settings["temperature"][i], top_p=0.9)
        assert one.item() == tokens[i].item() and p.item() == logprobs[i].item()
