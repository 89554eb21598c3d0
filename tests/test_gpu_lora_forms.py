"""Adapters in every variant of the row-phase kernel, in the verify and skinny kernels and in the general kernel's
tiles (needs an MI355X): rows of one, two and many adapters to a tile of 16 (test_adapter_routes.py checks the routes)."""

import pytest
import torch

import test_gpu_lora
from adapter_cases import ROWPHASE, SKINNY, VERIFY
from adapter_checks import DEV, check, inputs
from mlx_tree_spec_amd import quantized_matmul, quantized_matmul_lora

pytestmark = pytest.mark.gpu


def adapters(m):
    """The first 16 rows of one adapter, the next of two, the rest mixed with rows without one."""
    return [3] * min(m, 16) + [1 + i % 2 for i in range(max(0, min(m - 16, 16)))] + [i % 5 - 1 for i in range(max(0, m - 32))]


@pytest.mark.parametrize("m,k,n", [case[:3] for case in ROWPHASE] + VERIFY + SKINNY)
def test_forms(m, k, n):
    for ids in (adapters(m), [i % 5 - 1 for i in range(m - 1)] + [2]):
        args = inputs(m, k, n, 24, 4, m + k + n, ids)
        y = quantized_matmul_lora(*args)
        check(args, y)
        bare = args[7] < 0
        assert torch.equal(y[bare], quantized_matmul(*args[:4])[bare])


@pytest.mark.parametrize("bits,group", [(2, 32), (4, 128), (8, 64)])
@pytest.mark.parametrize("m,k,n", [(3, 512, 77), (16, 512, 8197), (32, 256, 99), (20, 512, 4099), (64, 512, 200), (50, 512, 4101)])
def test_general_tiles(m, k, n, bits, group):
    args = test_gpu_lora.inputs(m, k, n, 16, 4, m + n, bits, group, [i % 5 - 1 for i in range(m)])
    test_gpu_lora.check(args, quantized_matmul_lora(*args, group_size=group, bits=bits), group, bits)


def test_skinny_kernel_past_4_rows():
    """Weights past the 2 GiB that the verify kernel's offsets reach."""
    k, n = 16512, 262144
    for m in (6, 12, 20, 33):
        if m == 6:
            args = inputs(33, k, n, 8, 3, 1)
        part = [args[0][:m], *args[1:7], args[7][:m]]
        check(part, quantized_matmul_lora(*part))


def test_indices_past_32_bits():
    """64-bit indices that are those of an adapter in their lower half only name none."""
    args = inputs(16, 512, 272, 8, 3, 5, [1] * 16)
    far = torch.tensor([2**32, 2**32 + 1, -2**32, 2**40 + 2, 2**63 - 1, -2**63] + [2] * 10, device=DEV)
    for m in (4, 7, 16):
        y = quantized_matmul_lora(*[args[0][:m], *args[1:7], far[:m]])
        near = torch.where(far[:m] == 2, 2, -1).to(torch.int32)
        assert torch.equal(y, quantized_matmul_lora(*[args[0][:m], *args[1:7], near]))
        assert torch.equal(y[:4], quantized_matmul(args[0][:m], *args[1:4])[:4])
