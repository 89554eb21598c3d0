"""Adapters in every form of the row-split kernel (needs an MI355X), every column: ranges whose threads take several
items and whose last range is cut short among them (test_adapter_routes.py checks each shape's form)."""

import pytest
import torch

from adapter_cases import ROWSPLIT
from adapter_checks import check, inputs
from mlx_tree_spec_amd import quantized_matmul, quantized_matmul_lora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [8, 24])
@pytest.mark.parametrize("m,k,n", [case[:3] for case in ROWSPLIT])
def test_rowsplit_forms(m, k, n, rank):
    ids = [i % 5 - 1 for i in range(m - 1)] + [3]  # the last row, alone in its lane group at 9 and 13, has one
    args = inputs(m, k, n, rank, 4, m + k + n + rank, ids)
    y = quantized_matmul_lora(*args)
    check(args, y)
    bare = args[7] < 0
    assert torch.equal(y[bare], quantized_matmul(*args[:4])[bare])
    assert torch.equal(quantized_matmul_lora(*args), y)
