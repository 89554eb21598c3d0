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


@pytest.mark.parametrize("bits", [16, 8])
def test_far_pages_of_narrow_heads(bits):
    """One row over heads of 128 in pages around 4 and 8 GiB."""
    heads, dim, q_heads, tokens = 8, 128, 32, 500
    size, held = PAGE * heads * dim * bits // 8, 8
    pages = 2**33 // size + 4
    outs = []
    for count, order in ((pages, [pages - 1, pages - 3, pages // 2, pages // 2 - 1, pages // 2 + 1, pages - 4, 0, pages - 2]),
                         (held, list(range(held)))):
        g = torch.Generator().manual_seed(3)
        cache = KVCache.empty(count, PAGE, heads, dim, bits, DEV)
        free = torch.zeros(count, dtype=torch.int32, device=DEV)
        free[:held] = i32(order[::-1])
        tables = [i32([0]), torch.full((1, held), -1, dtype=torch.int32, device=DEV), free, i32([held])]
        for n in (tokens - 1, 1):
            step = step_tables_(*tables, i32([n]), n, PAGE, q_heads, heads, dim)
            k, v, q = (torch.randn(n, h, dim, generator=g).to(torch.bfloat16).to(DEV) for h in (heads, heads, q_heads))
            store_kv_(k, v, cache, step.slots)
        outs.append(paged_attention(q, cache, step))
        del cache
    assert torch.equal(*outs) and outs[0].isfinite().all()


def test_many_rows():
    """A prompt of 70000 rows: the first ones, those around 2^16 and the last against 64 bits, the row of another request too."""
    n, dim, heads, page = 70000, 64, 2, 128
    g = torch.Generator(device=DEV).manual_seed(5)
    pages = -(-n // page) + 1
    tables = [i32([0, 0]), torch.full((2, pages), -1, dtype=torch.int32, device=DEV),
              torch.arange(pages, dtype=torch.int32, device=DEV), i32([pages])]
    step = step_tables_(*tables, i32([n, 1]), n + 3, page, heads, 1, dim)
    cache = KVCache.empty(pages, page, 1, dim, 16, DEV)
    k, v, q = (torch.randn(n + 3, h, dim, generator=g, device=DEV).to(torch.bfloat16) for h in (1, 1, heads))
    store_kv_(k, v, cache, step.slots)
    out = paged_attention(q, cache, step)
    assert torch.equal(out[n], v[n].expand(heads, dim)) and not out[n + 1:].any()
    k64, v64, scale = k[:n, 0].double(), v[:n, 0].double(), dim ** -0.5
    for i in (0, 1, 127, 128, 65534, 65535, 65536, 65537, n - 1):
        s = scale * (q[i].double() @ k64[:i + 1].T)
        p = torch.softmax(s, -1)
        want, mag = p @ v64[:i + 1], p @ v64[:i + 1].abs()
        # (Two roundings to bf16, of each probability and of the result; in fp32 the sums over the tokens, and a logit's error: dim + 4
        # half steps of its terms' magnitudes.)
        terms = scale * (q[i].double().abs() @ k64[:i + 1].abs().T).max()
        bound = want.abs() * 2.0**-8 * 1.01 + mag * (2.0**-8 * 1.01 + 2.1 * (dim + 36) * 2.0**-24 * terms + (2 * i + 18) * 2.0**-24)
        assert ((out[i].double() - want).abs() <= bound).all(), i
