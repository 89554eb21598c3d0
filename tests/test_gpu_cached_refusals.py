"""Calls of cached_attention that are refused leave the cache as it was (needs an MI355X)."""

import pytest
import torch

from cache_refs import i32
from mlx_tree_spec_amd import KVCache, _lib, cached_attention
from test_gpu_cached_step import D, DEV, DIM, KV, Server

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
def test_refused_calls_store_nothing(bits, native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    server = Server(2, bits)
    step, cache = server.tables.step(i32([3, 2]), 5), server.caches[0]
    x = torch.randn(5, DIM, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    wide = KVCache.empty(12, 32, KV, D, bits, DEV)
    for c in (cache, wide):
        for t in c:
            if t is not None:
                t.fill_(7)
    masks = torch.tensor([1, 3, 5, 1, 3], dtype=torch.int64, device=DEV)
    for change, msg in ((dict(cache=wide), "the step was made for"), (dict(scale=float("inf")), "must be finite"),
                        (dict(scale=1e300), "must be finite"), (dict(ancestors=masks.to(torch.int32)), "ancestors must be"),
                        (dict(ancestors=masks[:4]), "ancestors must be"), (dict(ancestors=masks.cpu()), "all tensors must be on"),
                        (dict(step=step._replace(plan=step.plan[:-8])), "the step's plan must be"),
                        (dict(step=step._replace(block_table=step.block_table[:1])), "the step's plan must be")):
        with pytest.raises(ValueError, match=msg):
            cached_attention(x, server.layers[0], **{**dict(cache=cache, step=step), **change})
    for c in (cache, wide):
        assert all((t == 7).all() for t in c if t is not None)
    a, _, _ = cached_attention(x, server.layers[0], cache, step, ancestors=masks, scale=0.2)
    assert torch.isfinite(a.float()).all() and not (cache.keys == 7).all()
