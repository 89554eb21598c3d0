"""Adapters in every form of the GEMM (needs an MI355X): tiles of one adapter and of many, odd and even numbers of the
adapters' own K steps, ranks up to the largest (test_adapter_routes.py checks each shape's form)."""

import pytest
import torch

from adapter_cases import GEMM
from adapter_checks import DEV, check, inputs
from mlx_tree_spec_amd import quantized_matmul, quantized_matmul_lora

pytestmark = pytest.mark.gpu


def adapters(m, count, kind):
    if kind == "one":
        return torch.full((m,), count - 1)
    if kind == "runs":  # a few runs, their ends inside tiles, one of them without an adapter
        return torch.tensor([0, -1, 2, 1])[torch.arange(m) * 4 // m]
    return torch.randint(-1, count, (m,), generator=torch.Generator().manual_seed(m))


@pytest.mark.parametrize("rank,count,kind", [(8, 3, "runs"), (24, 40, "mixed"), (64, 5, "one"), (256, 3, "runs")])
@pytest.mark.parametrize("m,k,n", [case[:3] for case in GEMM])
def test_gemm_forms(m, k, n, rank, count, kind):
    args = inputs(m, k, n, rank, count, m + k + n + rank, adapters(m, count, kind))
    y = quantized_matmul_lora(*args)
    check(args, y)
    bare = args[7] < 0
    assert torch.equal(y[bare], quantized_matmul(*args[:4])[bare])


def test_scales_of_unaligned_rows():
    """Scales on a 4-byte boundary: the whole tiles without split roles at a K that otherwise has them."""
    args = inputs(2304, 512, 4096, 24, 5, 1)
    want = quantized_matmul_lora(*args)
    check(args, want)
    for i in (2, 3):
        off = torch.empty(args[i].numel() + 2, dtype=torch.bfloat16, device=DEV)[2:].reshape(args[i].shape)
        args[i] = off.copy_(args[i])
    check(args, quantized_matmul_lora(*args))
