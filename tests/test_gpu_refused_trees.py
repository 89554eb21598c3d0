"""A tree verify that refuses a request for want of pages (needs an MI355X): with keep & (request >= 0) none of its nodes enters
the cache in the step that keeps the accepted ones, though they would fit there."""

import numpy as np
import pytest
import torch

import cache_refs as R
from cache_refs import i32
from mlx_tree_spec_amd import cached_attention, store_kv_
from request_refs import f64
from test_gpu_cached_step import DEV, DIM, PAGE, Server

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
def test_nodes_of_a_refused_request_are_not_kept(captured):
    server = Server(3, 16)
    cache, layer = server.caches[0], server.layers[0]
    x = torch.randn(30, DIM, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    first = server.tables.step(i32([5, PAGE, 9]), 30)
    cached_attention(x, layer, cache, first)
    server.tables.free_count.fill_(1)  # (a page is left: the second request's tree needs two, so neither it nor the third, which needs one, gets any)
    nodes, before = i32([4, PAGE + 1, 8]), server.tables.lengths.clone()
    masks = torch.tensor([1, 3, 5, 11, *(1 << i for i in range(PAGE + 1)), *(1 << i for i in range(8))], dtype=torch.int64, device=DEV)
    kept = torch.zeros(29, dtype=torch.bool, device=DEV)
    kept[[0, 1, 4, 21, 22]] = True
    held = f64(cache.keys).copy()

    def verify():
        step = server.tables.step(nodes, 29, base=before)
        a, k, v = cached_attention(x[:29], layer, cache, step, ancestors=masks)
        accepted = server.tables.step(nodes, 29, base=before, keep=kept & (step.request >= 0))
        store_kv_(k, v, cache, accepted.slots)
        return step, a, k, accepted

    if captured:
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            verify()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step, a, k, accepted = verify()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
    else:
        step, a, k, accepted = verify()
    assert step.request.tolist() == [0] * 4 + [-1] * (PAGE + 1 + 8)
    assert not a[4:].any() and a[:4].any()
    assert server.tables.lengths.tolist() == [7, PAGE, 9]
    assert accepted.request.tolist() == [0, 0, *[-1] * 27] and accepted.positions.tolist()[:2] == [5, 6]
    keys, _ = R.token_rows(cache)
    slots = accepted.slots.tolist()
    assert (keys[slots[:2]] == f64(k[:2])).all()
    table = server.tables.block_table.cpu().numpy()
    old = held.transpose(0, 3, 1, 2, 4).reshape(keys.shape)
    for r, n in ((1, PAGE), (2, 9)):  # the refused requests' tokens are as they were
        at = table[r, 0] * PAGE + np.arange(n)
        assert (keys[at] == old[at]).all()
    server.tables.step(nodes, 29, base=before, keep=kept)
    assert server.tables.lengths.tolist() == [7, PAGE + 1, 11]
