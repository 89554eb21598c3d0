"""Caches past 4 GiB (needs an MI355X): what lies in far pages is stored and read as it is in near ones, and long requests' numbers
past 2^16 tokens. Every result is compared bit by bit with the one of a cache that holds the same in other pages."""

import pytest
import torch

from cache_refs import i32
from mlx_tree_spec_amd import KVCache, paged_attention, step_tables_, store_kv_

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS, D, PAGE = 4, 256, 64


def run(pages, order, bits, rows, tokens=1000):
    """A request of `tokens` cached tokens in pages of `order`, stored and attended to by `rows` rows."""
    g = torch.Generator().manual_seed(rows)
    cache = KVCache.empty(pages, PAGE, HEADS, D, bits, DEV)
    held = -(-tokens // PAGE)
    free = torch.zeros(pages, dtype=torch.int32, device=DEV)
    free[:held] = i32(order[:held][::-1])
    tables = [i32([0]), torch.full((1, held), -1, dtype=torch.int32, device=DEV), free, i32([held])]
    out = None
    for n in (tokens - rows, rows):
        step = step_tables_(*tables, i32([n]), n, PAGE, 24, HEADS, D)
        k, v, q = (torch.randn(n, h, D, generator=g).to(torch.bfloat16).to(DEV) for h in (HEADS, HEADS, 24))
        store_kv_(k, v, cache, step.slots)
        out = paged_attention(q, cache, step)
    return out


@pytest.mark.parametrize("bits,pages", [(16, 70000), (8, 140000)])
@pytest.mark.parametrize("rows", [1, 12])
def test_far_pages(bits, pages, rows):
    size = PAGE * HEADS * D * bits // 8
    assert pages * size > 2 * 2**32
    far = [pages - 1 - 3 * i for i in range(8)] + [2**32 // size - 4 + i for i in range(8)]
    assert torch.equal(run(pages, far, bits, rows), run(16, list(range(16)), bits, rows))


def test_many_tokens():
    """A request of 600000 tokens whose last page alone is not zero: its few rows there see the mean over all tokens."""
    tokens, pages = 600000, 600000 // 64 + 1
    cache = KVCache(torch.zeros(pages, 1, 8, 64, 8, dtype=torch.bfloat16, device=DEV),
                    torch.zeros(pages, 1, 8, 64, 8, dtype=torch.bfloat16, device=DEV))
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None].contiguous()
    tables = [i32([tokens]), table, torch.zeros(pages, dtype=torch.int32, device=DEV), i32([0])]
    cache.values[(tokens - 1) // 64, 0, (tokens - 1) % 64 // 8, :, (tokens - 1) % 8] = 4096.0
    for heads in (1, 20):
        step = step_tables_(*tables, i32([1]), 1, 64, heads, 1, 64, base=i32([tokens - 1]))
        assert step.positions.item() == tokens - 1
        q = torch.randn(1, heads, 64, device=DEV).to(torch.bfloat16)
        out = paged_attention(q, cache, step).double()
        want = 4096.0 / tokens  # (equal logits: every probability 1 / tokens; one rounding of it, the sum of 600000 ones, one of the result)
        assert ((out - want).abs() <= want * (2 * 2.0**-8 + tokens * 2.0**-24)).all()
