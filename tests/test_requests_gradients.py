"""The per-request operators have no gradient: every floating-point input that asks for one is refused, but for the head
norms' weights (CPU only: each call ends before any GPU work)."""

import pytest
import torch
from torch.autograd import forward_ad

from mlx_tree_spec_amd import qk_norm_rope, quantized_matmul_lora, sample
from test_requests_host import lora_args, rope_args, z


def sample_args(m=4, v=100):
    full = lambda x: torch.full((m,), x)  # noqa: E731
    return dict(logits=z(m, v), uniform=full(0.5), temperature=full(1.0), top_p=full(0.9), min_p=full(0.1))


CASES = ([(quantized_matmul_lora, lora_args, n) for n in ("x", "scales", "biases", "lora_a", "lora_b", "lora_scale")]
         + [(qk_norm_rope, rope_args, n) for n in ("q", "k", "inv_freq")]
         + [(sample, sample_args, n) for n in ("logits", "uniform", "temperature", "top_p", "min_p")])
IDS = [f"{f.__name__}-{n}" for f, _, n in CASES]


@pytest.mark.parametrize("op,args,name", CASES, ids=IDS)
def test_inputs_that_require_a_gradient(op, args, name):
    a = args()
    a[name].requires_grad_(True)
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        op(**a)
    with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
        op(**a)
    a[name] = a[name] * 2  # not a leaf
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        op(**a)


TANGENTS = CASES + [(qk_norm_rope, rope_args, n) for n in ("q_weight", "k_weight")]
TANGENT_IDS = [f"{f.__name__}-{n}" for f, _, n in TANGENTS]


@pytest.mark.parametrize("op,args,name", TANGENTS, ids=TANGENT_IDS)
def test_inputs_with_a_tangent(op, args, name):
    a = args()
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="no CPU path"):
            op(**a)
        dual = {**a, name: forward_ad.make_dual(a[name], torch.ones_like(a[name]))}
        with torch.no_grad(), pytest.raises(ValueError, match=f"{name} carries a tangent"):
            op(**dual)
    with pytest.raises(ValueError, match="carries a tangent"):
        torch.func.jvp(lambda t: op(**{**a, name: t}), (a[name],), (torch.ones_like(a[name]),))
