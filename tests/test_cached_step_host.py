"""What cached_attention refuses before anything is computed or stored (CPU only: its layer here has no projections)."""

import types

import pytest
import torch

from mlx_tree_spec_amd import CacheStep, KVCache, cached_attention

BF, I32 = torch.bfloat16, torch.int32


def cache(pages=4, page=16, heads=2, dim=64):
    return KVCache.empty(pages, page, heads, dim, 16, "cpu")


def step(page=16, capacity=4):
    i = torch.zeros(5, dtype=I32)
    return CacheStep(i, i, i, torch.zeros(40, dtype=I32), torch.zeros(3, capacity, dtype=I32), page, 8, 2, 64, 5)


@pytest.mark.parametrize("change,msg", [
    (dict(step=step(page=32)), "the step was made for"),
    (dict(cache=cache(heads=4)), "the step was made for"),
    (dict(cache=cache(pages=0)), "without pages"),
    (dict(step=step(capacity=0)), "without pages"),
    (dict(step=step()._replace(plan=None)), "no plan"),
    (dict(step=step()._replace(plan=torch.zeros(40))), "plan must be"),
    (dict(step=step()._replace(request=torch.zeros(10, dtype=I32)[::2])), "request must be contiguous"),
    (dict(scale=float("inf")), "must be finite"),
    (dict(scale=float("nan")), "must be finite"),
    (dict(scale=1e300), "must be finite"),
    (dict(ancestors=torch.zeros(5, dtype=I32)), "ancestors must be"),
    (dict(ancestors=torch.zeros(4, dtype=torch.int64)), "ancestors must be"),
    (dict(), "HIP device"),
])
def test_refused_before_the_projections(change, msg):
    layer = types.SimpleNamespace(heads=8, kv_heads=2, head_dim=64)
    args = {**dict(cache=cache(), step=step()), **change}
    with pytest.raises(ValueError, match=msg):
        cached_attention(torch.zeros(5, 32, dtype=BF), layer, **args)
