"""Stores into the paged cache on the GPU (needs an MI355X). bf16 is stored as it is; of 8 bits the scale is fp32's value of
max|x| / 127, and a code off from x / scale by half, and by 127 half steps of fp32 (the quotient's own rounding)."""

import random

import numpy as np
import pytest
import torch

import cache_refs as R
from cache_refs import i32
from mlx_tree_spec_amd import KVCache, store_kv_
from request_refs import HALF_STEP_F32, f64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def filled(pages, page, heads, dim, bits):
    """A cache whose every byte is known."""
    cache = KVCache.empty(pages, page, heads, dim, bits, DEV)
    for t in cache:
        if t is not None:
            t.fill_(7)
    return cache


def rows(m, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(m, heads, dim, generator=g) * 2).to(torch.bfloat16).to(DEV) for _ in range(2)]


def some_slots(m, pages, page, seed, dropped=0.1):
    """Runs of neighbouring slots that begin anywhere, and rows without one."""
    rng = random.Random(seed)
    pages_left, out = list(range(pages)), []
    rng.shuffle(pages_left)
    while len(out) < m:
        if not pages_left:
            out.append(-1)
            continue
        p, at = pages_left.pop(), rng.choice([0, 0, 1, 7, 8, 15, page - 1])
        out += [p * page + i for i in range(at, at + rng.randint(1, page - at))]
    return [-1 if rng.random() < dropped else s for s in out[:m]]


def check(cache, before, k, v, slots):
    at = [i for i, s in enumerate(slots) if 0 <= s < cache.keys.shape[0] * cache.keys.shape[3]]
    where = np.array([slots[i] for i in at], np.int64)
    rest = np.setdiff1d(np.arange(cache.keys.shape[0] * cache.keys.shape[3]), where)
    bare, old = cache._replace(key_scales=None, value_scales=None), before._replace(key_scales=None, value_scales=None)
    for name, got, was, x, scales, was_scales in zip(("keys", "values"), R.token_rows(bare), R.token_rows(old), (k, v),
                                                     cache[2:], before[2:]):
        assert (got[rest] == was[rest]).all(), f"{name}: another token changed"
        x = f64(x)[at]
        if scales is None:
            assert (got[where] == x).all(), name
            continue
        per_token = lambda t: f64(t).transpose(0, 2, 1).reshape(-1, t.shape[1])  # noqa: E731
        assert (per_token(scales)[rest] == per_token(was_scales)[rest]).all()
        scale, exact = R.codes(x)
        s = per_token(scales)[where]
        assert (np.abs(s - scale) <= 2 * HALF_STEP_F32 * scale).all()
        exact = x / np.where(s > 0, s, 1)[..., None]
        assert (np.abs(got[where] - exact) <= 0.5 + 127 * HALF_STEP_F32).all() and (np.abs(got[where]) <= 127).all()


def run(m, heads, dim, page, bits, seed, pages=None):
    pages = pages or m // page * 3 + 6
    cache = filled(pages, page, heads, dim, bits)
    before = KVCache(*(t if t is None else t.clone() for t in cache))
    k, v = rows(m, heads, dim, seed)
    slots = some_slots(m, pages, page, seed)
    assert store_kv_(k, v, cache, i32(slots)) is None
    check(cache, before, k, v, slots)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("m,heads,dim,page", [(1, 1, 64, 16), (1, 4, 256, 64), (16, 4, 256, 64), (37, 8, 128, 32), (200, 3, 192, 16),
                                              (5, 17, 64, 128), (300, 2, 256, 1024), (1000, 8, 128, 64), (33, 40, 128, 16)])
def test_matches_the_rows(m, heads, dim, page, bits):
    run(m, heads, dim, page, bits, m + dim)


@pytest.mark.parametrize("m", [1, 50])
def test_heads_of_96(m):
    run(m, 5, 96, 32, 16, m)


def test_slots_out_of_range_are_skipped():
    cache = filled(3, 16, 2, 64, 16)
    before = KVCache(*(t if t is None else t.clone() for t in cache))
    k, v = rows(8, 2, 64, 1)
    slots = [47, 48, -1, 0, 2**31 - 1, -2**31, 1, 2]
    store_kv_(k, v, cache, i32(slots))
    check(cache, before, k, v, slots)


@pytest.mark.parametrize("bits", [16, 8])
def test_views_of_projections(bits):
    """Rows and heads read in place from a fused projection, and layouts that are copied."""
    k, v = rows(20, 4, 128, 3)
    slots = i32(list(range(5, 25)))
    want = filled(4, 16, 4, 128, bits)
    store_kv_(k, v, want, slots)
    fused = torch.full((20, 16, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    fused[:, 8:12], fused[:, 12:] = k, v
    odd = torch.empty(20 * 4 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].reshape(20, 4, 128)
    odd.copy_(k)
    turned = v.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for a, b in ((fused[:, 8:12], fused[:, 12:]), (odd, turned)):
        cache = filled(4, 16, 4, 128, bits)
        store_kv_(a, b, cache, slots)
        assert all(torch.equal(x, y) for x, y in zip(cache, want) if x is not None)


def test_codes_of_zeros_and_of_what_is_not_finite():
    k, v = rows(4, 2, 64, 5)
    k[0, 0], v[1, 1] = 0, 0
    k[2, 1, 63], v[3, 0, 5] = float("inf"), float("nan")
    k[1, 0, 7], v[0, 0, 9] = 3e38, 1e-40
    cache = filled(2, 16, 2, 64, 8)
    store_kv_(k, v, cache, i32([0, 1, 2, 3]))
    ks, vs = cache.key_scales[0, :, :4].T, cache.value_scales[0, :, :4].T
    assert ks[0, 0] == 0 and vs[1, 1] == 0 and ks[2, 1].isnan() and vs[3, 0].isnan()
    assert ks.isnan().sum() == 1 and vs.isnan().sum() == 1
    keys, values = R.token_rows(cache)
    assert not keys[0, 0].any() and not values[1, 1].any() and np.isnan(keys[2, 1]).all() and np.isnan(values[3, 0]).all()
    assert abs(keys[1, 0, 7] / 3e38 - 1) < 0.01


def test_no_rows_and_captured():
    cache = filled(4, 16, 4, 128, 8)
    k, v = rows(0, 4, 128, 1)
    store_kv_(k, v, cache, i32([]))
    assert all((t == 7).all() for t in cache)
    k, v = rows(6, 4, 128, 2)
    slots = i32([3, 4, 5, 20, 21, -1])
    store_kv_(k, v, cache, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        store_kv_(k, v, cache, slots)
    for i in range(3):
        for t, x in zip((k, v), rows(6, 4, 128, 10 + i)):
            t.copy_(x)
        slots.copy_(slots.roll(1))
        want = KVCache(*(t.clone() for t in cache))
        store_kv_(k, v, want, slots)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cache, want))
