"""Inputs of the per-request operators that ask for a gradient, on the GPU, where the native calls come first (needs an
MI355X)."""

import pytest
import torch
from torch.autograd import forward_ad

from test_requests_gradients import CASES, IDS, TANGENT_IDS, TANGENTS

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


@pytest.mark.parametrize("op,args,name", TANGENTS, ids=TANGENT_IDS)
def test_inputs_with_a_tangent(op, args, name):
    a = on_gpu(args())
    with forward_ad.dual_level():
        op(**a)
        dual = {**a, name: forward_ad.make_dual(a[name], torch.ones_like(a[name]))}
        with torch.no_grad(), pytest.raises(ValueError, match=f"{name} carries a tangent"):
            op(**dual)
