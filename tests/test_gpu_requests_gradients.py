"""Inputs of the per-request operators that ask for a gradient, on the GPU, where the native calls come first (needs an
MI355X)."""

import pytest
import torch

from test_requests_gradients import CASES, IDS

pytestmark = pytest.mark.gpu


def on_gpu(args):
    return {k: v.to("cuda:0") if isinstance(v, torch.Tensor) else v for k, v in args.items()}


@pytest.mark.parametrize("op,args,name", CASES, ids=IDS)
def test_inputs_that_require_a_gradient(op, args, name):
    a = on_gpu(args())
    want = op(**a)
    a[name].requires_grad_(True)
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        op(**a)
    with torch.no_grad():
        got = op(**a)
    for x, y in zip(*(t if isinstance(t, tuple) else (t,) for t in (got, want))):
        assert torch.equal(x, y)
