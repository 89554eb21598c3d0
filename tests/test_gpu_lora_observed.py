"""Adapters under autocast, on every form of the projection (needs an MI355X): the result is bf16 with the bits of the
plain call."""

import pytest
import torch

from mlx_tree_spec_amd import quantized_matmul_lora
from test_gpu_lora import check, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# (m, k, n, bits, group, whether a library product computes the projection)
FORMS = [(7, 256, 96, 4, 64, False), (9, 512, 96, 8, 32, False), (7, 96, 40, 4, 32, True), (300, 128, 77, 8, 64, False)]


def call(form):
    m, k, n, bits, group, _ = form
    args = inputs(m, k, n, 16, 3, m + n, bits, group)
    return args, lambda x=args[0]: quantized_matmul_lora(x, *args[1:], group_size=group, bits=bits)


@pytest.mark.parametrize("context", [lambda: torch.autocast("cuda", dtype=torch.float16), lambda: torch.autocast("cuda"),
                                     lambda: torch.autocast("cuda", dtype=torch.bfloat16), lambda: torch.device(DEV)],
                         ids=["float16", "default", "bfloat16", "device"])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_autocast_and_default_device(form, context):
    args, f = call(form)
    want = f()
    check(args, want, form[4], form[3], twice=form[5])
    with context():
        got = f()
    assert got.dtype == torch.bfloat16 and torch.equal(got, want)
