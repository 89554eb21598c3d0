"""Attention over the paged cache on the GPU (needs an MI355X), against 64 bits. The bound is derived in cache_refs."""

import random

import numpy as np
import pytest
import torch

import cache_refs as R
from cache_refs import i32
from mlx_tree_spec_amd import KVCache, _lib, paged_attention, step_tables_
from request_refs import f64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Case:
    """Requests of `cached` tokens with `rows` new ones each over a cache that holds NaN wherever no token lies."""

    def __init__(self, cached, rows, hq, hk, dim, page=64, bits=16, tree=False, gated=False, pad=0, seed=0, max_rows=None, size=1.0):
        g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.cached, self.rows = list(cached), list(rows)
        lengths = [c + n for c, n in zip(cached, rows)]
        held = [R.ceil(n, page) for n in lengths]
        pages, capacity = sum(held) + 3, max(held) + 1
        order = list(range(pages))
        rng.shuffle(order)
        table, at = np.full((len(cached), capacity), -1, np.int32), 0
        for r, n in enumerate(held):
            table[r, :n] = order[at:at + n]
            at += n
        e = 8 if bits == 16 else 16
        empty = np.ones(pages * page, bool)
        for r, n in enumerate(lengths):
            for t in range(n):
                empty[table[r, t // page] * page + t % page] = False
        empty = torch.from_numpy(empty).reshape(pages, page)
        if bits == 16:
            keys = (randn(pages, hk, dim // 8, page, 8) * size).to(torch.bfloat16)
            values = randn(pages, hk, page // 8, dim, 8).to(torch.bfloat16)
            keys.masked_fill_(empty[:, None, None, :, None], float("nan"))
            values.masked_fill_(empty.reshape(pages, 1, page // 8, 1, 8), float("nan"))
            self.cache = KVCache(keys.to(DEV), values.to(DEV))
        else:
            codes = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int8).to(DEV)  # noqa: E731
            scales = [((1 + torch.rand(pages, hk, page, generator=g)) / 100).masked_fill(empty[:, None], float("nan")).to(DEV)
                      for _ in range(2)]
            self.cache = KVCache(codes(pages, hk, dim // e, page, e), codes(pages, hk, page // e, dim, e), *scales)
        self.m = sum(rows) + pad
        self.q = randn(self.m, hq, dim).to(torch.bfloat16).to(DEV)
        self.gate = (2 * randn(self.m, hq, dim)).to(torch.bfloat16).to(DEV) if gated else None
        masks = [m for n in rows for m in R.tree_masks(rng, n)] + [0] * pad
        self.ancestors = torch.tensor(masks, dtype=torch.int64, device=DEV) if tree else None
        self.scale, self.table = dim ** -0.5, table
        self.tables = [i32(lengths), torch.from_numpy(table).to(DEV), i32(order[at:] + [-1] * at), i32([pages - at])]
        self.make_step(hq, hk, dim, page, max_rows)

    def make_step(self, hq, hk, dim, page, max_rows):
        self.step = step_tables_(*self.tables, i32(self.rows), self.m, page, hq, hk, dim, base=i32(self.cached),
                                 max_rows=max_rows)

    def run(self, **changes):
        args = {"q": self.q, "cache": self.cache, "step": self.step, "scale": self.scale, "ancestors": self.ancestors,
                "gate": self.gate, **changes}
        return paged_attention(**args)

    def check(self, out, finite=True):
        assert out.shape == self.q.shape and out.dtype == torch.bfloat16 and out.is_contiguous()
        k, v = R.token_rows(self.cache)
        q, got, page = f64(self.q), f64(out), self.step.page_size
        row = 0
        for r, (c, n) in enumerate(zip(self.cached, self.rows)):
            if n == 0:
                continue
            t = np.arange(c + n)
            at = self.table[r, t // page].astype(np.int64) * page + t % page
            masks = None if self.ancestors is None else self.ancestors[row:row + n].tolist()
            want, mag, delta = R.attention(q[row:row + n], k[at], v[at], self.scale, R.visible(c, n, masks))
            if self.gate is not None:
                s = 1 / (1 + np.exp(-f64(self.gate[row:row + n])))
                want, mag = want * s, mag * s
            bound = R.attention_bound(want, mag, delta, c + n)
            err = np.abs(got[row:row + n] - want)
            assert (err <= bound).all(), (r, c, n, float(np.nanmax(err - bound)), float(np.nanmax(err)))
            row += n
        assert not got[row:].any()


HEADS = [(1, 1, 64), (6, 1, 256), (24, 4, 256), (8, 2, 128), (7, 7, 96), (10, 2, 192), (16, 1, 128), (17, 1, 64), (40, 2, 64)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hq,hk,dim", HEADS)
def test_decode_of_ragged_requests(hq, hk, dim, bits):
    if bits == 8 and dim == 96:
        pytest.skip("heads of 96 are not held in 8 bits")
    case = Case([0, 1, 15, 31, 32, 63, 64, 65, 300, 1000], [1] * 10, hq, hk, dim, bits=bits, pad=2, seed=dim + hq, max_rows=1)
    case.check(case.run())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("tree,gated", [(False, False), (True, True)])
@pytest.mark.parametrize("hq,hk,dim", HEADS)
def test_several_rows(hq, hk, dim, tree, gated, bits):
    """Trees and runs of rows, requests without a context or without rows, padding."""
    if bits == 8 and dim == 96:
        pytest.skip("heads of 96 are not held in 8 bits")
    case = Case([0, 40, 7, 500, 130, 64], [5, 0, 1, 17, 33, 64], hq, hk, dim, page=32, bits=bits, tree=tree, gated=gated, pad=3,
                seed=dim + hq)
    case.check(case.run())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("bits", [16, 8])
def test_pages(page, bits):
    case = Case([1, 17, 200, 900], [3, 1, 2, 1], 12, 2, 128, page=page, bits=bits, seed=page)
    case.check(case.run())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("rows", [1, 20])
def test_one_long_request(rows, dim, bits):
    """Many splits of one request, joined."""
    case = Case([20011], [rows], 6, 1, dim, bits=bits, tree=rows > 1, gated=True, seed=rows, max_rows=rows)
    case.check(case.run())


def test_rows_of_a_prompt():
    """More rows than a tree may have, past a context, some hundred of them."""
    case = Case([0, 100], [300, 150], 4, 2, 64, seed=1)
    case.check(case.run())


@pytest.mark.parametrize("hq,hk,dim,bits", [(4, 1, 64, 16), (4, 2, 128, 16), (12, 4, 256, 16), (9, 3, 64, 8), (5, 5, 96, 16),
                                            (4, 1, 256, 8)])
@pytest.mark.parametrize("cached,rows", [([0], [230]), ([70, 5, 0], [100, 1, 150])])
def test_row_blocks_of_few_heads(cached, rows, hq, hk, dim, bits):
    """Several row blocks of so few requests and heads that each is shared out."""
    case = Case(cached, rows, hq, hk, dim, bits=bits, gated=True, pad=1, seed=hk)
    case.check(case.run())


@pytest.mark.parametrize("hq,hk,dim,bits", [(8, 2, 64, 16), (4, 2, 256, 16), (8, 2, 128, 8)])
def test_most_requests(hq, hk, dim, bits):
    """As many requests as a step takes, of a few tokens each."""
    rng = random.Random(7)
    case = Case([rng.randrange(0, 4) for _ in range(2048)], [rng.choice([0, 1, 1]) for _ in range(2048)], hq, hk, dim, page=16,
                bits=bits, max_rows=1, seed=11)
    case.check(case.run())


@pytest.mark.parametrize("hq,hk,dim", [(6, 1, 256), (24, 4, 256), (32, 8, 128), (16, 16, 64), (40, 2, 64), (129, 1, 64)])
def test_partial_results_fit_the_workspace(hq, hk, dim):
    """Plans of all kinds of batches: the partial rows and items that a plan names fit what is set aside for them."""
    lib, rng, page = _lib.load(), random.Random(hq), 64
    for _ in range(40):
        n = rng.choice([1, 2, 3, 17, 300])
        most = rng.choice([1, 2, 5, 22, 64, 200])
        rows = [rng.choice([0, 1, most, rng.randrange(most + 1)]) for _ in range(n)]
        longest = rng.choice([70, 1000, 30000, 1 << 19])
        cached = [min(longest, (1 << 24) // n) if rng.random() < 0.3 else rng.randrange(longest // 8 + 1) for _ in range(n)]
        held = [R.ceil(c + k, page) for c, k in zip(cached, rows)]
        lengths, table = i32([c + k for c, k in zip(cached, rows)]), torch.zeros(n, max(held) + 1, dtype=torch.int32, device=DEV)
        step = step_tables_(lengths, table, torch.zeros(sum(held) + 1, dtype=torch.int32, device=DEV), i32([0]), i32(rows), sum(rows), page,
                            hq, hk, dim, base=i32(cached), max_rows=most)
        words = step.plan.tolist()
        size = lib.qmm4_paged_workspace(sum(rows), n, hq, hk, dim, step.max_rows)
        room = size // (4 * (dim + 2) * hq)  # rows of the step, each with all its heads
        items = 0
        for r, (c, k) in enumerate(zip(cached, rows)):
            first, count, length, per, splits, part = words[8 + 8 * r:14 + 8 * r]
            assert count == k and (k == 0 or (first, length) == (sum(rows[:r]), c + k))
            items += splits
            if splits > 1:
                assert per * (splits - 1) < length <= per * splits and 0 <= part and part + splits * k <= room
        assert words[0] == items and 8 * (1 + n + items) <= len(words)


def test_rows_that_see_nothing():
    """Masks of zero without a context give zeros, with one the context; bits of rows that are not there see nothing."""
    case = Case([0, 9, 0], [4, 3, 2], 6, 2, 64, tree=True, gated=True, seed=2)
    case.ancestors[:] = torch.tensor([0, 1, 0, -16, 0, 2, -1, 1 << 40, 3], dtype=torch.int64, device=DEV)
    out = case.run()
    case.check(out)
    assert not out[0].any() and not out[2].any() and not out[3].any() and out[1].any() and out[4].any() and not out[7].any()


def test_refused_requests_give_zeros():
    case = Case([10, 20, 30], [2, 3, 1], 4, 2, 64, page=16, seed=3)
    case.tables[3].fill_(0)
    step = step_tables_(*case.tables, i32([2, 30, 1]), 33, 16, 4, 2, 64, base=i32(case.cached))
    q = torch.randn(33, 4, 64, device=DEV).to(torch.bfloat16)
    out = case.run(q=q, step=step)
    assert step.request[2:32].eq(-1).all() and not out[2:32].any() and out[:2].any() and out[32].any()


@pytest.mark.parametrize("tree", [False, True])
def test_what_is_not_finite_reaches_who_sees_it(tree):
    """Infinities and NaN in a token's key or value, in front of the rows and among them."""
    case = Case([40], [20], 6, 2, 128, tree=tree, seed=4)
    page = case.step.page_size
    def token(t):
        return int(case.table[0, t // page]), t % page
    clean = case.run()
    for t, value in ((45, float("nan")), (50, float("inf")), (59, -float("inf"))):
        for which in ("keys", "values"):
            p, o = token(t)
            keys, values = case.cache.keys.clone(), case.cache.values.clone()
            if which == "keys":
                keys[p, 1, 3, o, 2] = value
            else:
                values[p, 1, o // 8, 77, o % 8] = value
            out = case.run(cache=KVCache(keys, values))
            sees = R.visible(40, 20, None if case.ancestors is None else case.ancestors.tolist())[:, t]
            assert torch.equal(out[:, :3], clean[:, :3])                      # the other key head's rows
            unseen = torch.from_numpy(~sees).to(DEV)
            assert torch.equal(out[unseen], clean[unseen])
            seen = out[torch.from_numpy(sees).to(DEV)][:, 3:]
            if which == "values":
                assert not torch.isfinite(seen[..., 77].float()).any()
                rest = clean[torch.from_numpy(sees).to(DEV)][:, 3:].clone()
                rest[..., 77] = seen[..., 77]
                assert torch.equal(torch.nan_to_num(rest.float()), torch.nan_to_num(seen.float()))
            elif value != value:
                assert torch.isnan(seen.float()).all()


def test_far_logits():
    """Logits hundreds apart, so that the running maximum moves often and far."""
    case = Case([3000, 50], [1, 4], 6, 1, 128, seed=6, size=25.0)
    case.check(case.run())


def test_views_scale_and_default_scale():
    case = Case([100, 3], [2, 5], 6, 2, 128, gated=True, seed=7)
    want = case.run()
    fused = torch.full((7, 6, 256), float("nan"), dtype=torch.bfloat16, device=DEV)
    fused[..., :128], fused[..., 128:] = case.q, case.gate
    assert torch.equal(case.run(q=fused[..., :128], gate=fused[..., 128:], scale=None), want)
    odd = torch.empty(7 * 6 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].reshape(7, 6, 128)
    odd.copy_(case.q)
    turned = case.gate.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    assert torch.equal(case.run(q=odd, gate=turned), want)
    case.scale = -0.3
    case.check(case.run())
    case.scale = 0.0
    case.check(case.run())


def test_repeatable_and_on_streams():
    """Two calls at once on streams of their own give the bits of one alone."""
    cases = [Case([5000, 70], [1, 1], 24, 4, 256, gated=True, seed=8, max_rows=1), Case([900], [30], 8, 2, 128, tree=True, seed=9)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append([c.run() for _ in range(4)])
        torch.cuda.synchronize()
        for outs, w in zip(got, want):
            assert all(torch.equal(o, w) for o in outs)


def test_captured_with_its_tables():
    """A step captured once, tables and attention, replayed as the requests grow."""
    case = Case([100, 30, 0], [1, 1, 1], 6, 2, 128, page=16, pad=1, seed=10, max_rows=1)
    keys, values = (torch.randn(t.shape, device=DEV).to(torch.bfloat16) for t in case.cache[:2])
    case.cache = KVCache(keys, values)
    rows = i32([1, 1, 1])
    def step():
        s = step_tables_(*case.tables, rows, 4, 16, 6, 2, 128, max_rows=1)
        return case.run(step=s)
    kept = [t.clone() for t in case.tables]
    step()
    for t, k in zip(case.tables, kept):
        t.copy_(k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        rows.copy_(i32([[1, 1, 0], [0, 1, 1], [1, 0, 1], [1, 1, 1]][i]))
        before = [t.clone() for t in case.tables]
        want = step()
        for t, k in zip(case.tables, before):
            t.copy_(k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_plain_and_native_calls_agree(monkeypatch):
    from mlx_tree_spec_amd import _lib
    cases = [Case([500, 3], [1, 2], 24, 4, 256, gated=True, seed=11), Case([70], [9], 8, 2, 128, bits=8, tree=True, seed=12)]
    want = [c.run() for c in cases]
    monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    for c, w in zip(cases, want):
        assert torch.equal(c.run(), w)


def test_no_rows_and_no_requests():
    case = Case([5, 9], [0, 0], 6, 2, 64, pad=3, seed=13)
    case.check(case.run())
    case = Case([5, 9], [2, 1], 6, 2, 64, seed=14, max_rows=0)
    assert case.step.request.tolist() == [-1] * 3 and not case.run().any()
    case = Case([5], [0], 6, 2, 64, seed=15)
    assert case.run().shape == (0, 6, 64)
    step = step_tables_(i32([]), torch.empty((0, 2), dtype=torch.int32, device=DEV), i32([0]), i32([1]), i32([]), 2, 64, 6, 2, 64)
    q = torch.randn(2, 6, 64, device=DEV).to(torch.bfloat16)
    assert not case.run(q=q, step=step).any()


def test_plans_of_other_steps_are_refused():
    """A plan whose size is not that of the step's requests and heads is refused before anything is launched."""
    c = Case([100, 40], [1, 1], 8, 2, 64)
    for change in (dict(plan=c.step.plan[:-8]), dict(plan=torch.cat((c.step.plan, c.step.plan[:8]))),
                   dict(block_table=c.step.block_table[:1])):
        with pytest.raises(ValueError, match="the step's plan must be"):
            paged_attention(c.q, c.cache, c.step._replace(**change))


def test_nan_queries_stay_in_their_rows():
    for rows, max_rows in ((1, 1), (9, None)):
        case = Case([200, 50, 70], [rows] * 3, 6, 2, 128, seed=16, max_rows=max_rows)
        want = case.run()
        case.q[rows, 4, 7] = float("nan")
        case.q[2 * rows, 1, 3] = float("inf")
        out = case.run()
        assert torch.isnan(out[rows, 4].float()).all() and not torch.isfinite(out[2 * rows, 1].float()).all()
        out[rows, 4], out[2 * rows, 1] = want[rows, 4], want[2 * rows, 1]
        assert torch.equal(out, want)
