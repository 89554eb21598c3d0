"""Attention over cached values near the ends of what bf16 holds (needs an MI355X): a mean of finite values is finite, however many
they are and in whatever order the logits rise, and small values keep their bits. Against 64 bits, with the bound of cache_refs."""

import pytest
import torch

from test_gpu_paged import Case

pytestmark = pytest.mark.gpu
CONTEXTS = [0, 40, 300, 5030]


def sized(size, rows, group, dim, bits, positive):
    """Requests whose values are between size / 2 and size, of both signs or of one."""
    case = Case(CONTEXTS, [rows] * 4, 2 * group, 2, dim, bits=bits, tree=rows > 1, gated=rows == 1, seed=dim + rows, max_rows=rows)
    g = torch.Generator().manual_seed(rows)
    if bits == 8:
        case.cache.value_scales.mul_(size / 127 / 0.02)  # (they were 0.01 to 0.02)
        if positive:
            case.cache.values.copy_(torch.randint(64, 128, case.cache.values.shape, generator=g, dtype=torch.int8))
    else:
        x = size * (0.5 + 0.5 * torch.rand(case.cache.values.shape, generator=g))
        if not positive:
            x = torch.where(torch.rand(x.shape, generator=g) < 0.5, x, -x)
        case.cache.values.copy_(torch.where(case.cache.values.isnan().cpu(), float("nan"), x))
    return case


@pytest.mark.parametrize("positive", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,group", [(1, 3), (20, 3), (40, 3)])
def test_largest_values(rows, group, dim, bits, positive):
    case = sized(3e38, rows, group, dim, bits, positive)
    out = case.run()
    assert torch.isfinite(out.float()).all()
    case.check(out)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("rows,group", [(1, 3), (20, 3), (40, 3)])
def test_small_values(rows, group, bits):
    """(1e-28: beside it the bound's 1e-37 for numbers below the smallest does not count.)"""
    case = sized(1e-28, rows, group, 128, bits, False)
    case.check(case.run())
