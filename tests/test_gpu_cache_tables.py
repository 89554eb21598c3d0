"""The paged cache's tables on the GPU (needs an MI355X), against a plain loop over requests: everything equal."""

import random

import numpy as np
import pytest
import torch

import cache_refs as R
from cache_refs import i32
from mlx_tree_spec_amd import CacheTables, _lib, step_tables_

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Both:
    """The tables on the GPU and as the plain loop has them."""

    def __init__(self, requests, capacity, pages, page, seed=0):
        self.page, self.rng = page, random.Random(seed)
        order = list(range(pages))
        self.rng.shuffle(order)
        self.lengths, self.free, self.count = [0] * requests, order, pages
        self.table = np.full((requests, capacity), -1, np.int32)
        self.t = [i32(self.lengths), torch.from_numpy(self.table.copy()).to(DEV), i32(order), i32([pages])]

    def step(self, rows, total, base=None, keep=None, max_rows=None):
        want = R.tables(self.lengths, self.table, self.free, self.count, rows, total, self.page, base, keep, max_rows)
        self.count = want[3]
        step = step_tables_(*self.t, i32(rows), total, self.page, 24, 4, 256, base=None if base is None else i32(base),
                            keep=None if keep is None else torch.tensor(keep, dtype=torch.bool, device=DEV), max_rows=max_rows)
        for got, w in zip((step.slots, step.positions, step.request), want):
            assert got.dtype == torch.int32 and got.tolist() == w
        assert self.t[0].tolist() == self.lengths and self.t[3].item() == self.count
        assert (self.t[1].cpu().numpy() == self.table).all()
        assert self.t[2].tolist()[:self.count] == self.free[:self.count]
        held = [p for row, n in zip(self.table, self.lengths) for p in row[:R.ceil(n, self.page)]]
        assert len(set(held)) == len(held) and not set(held) & set(self.free[:self.count])
        return step


@pytest.mark.parametrize("requests,page", [(1, 16), (3, 64), (16, 32), (64, 16), (65, 128), (1025, 16), (2048, 32)])
def test_steps_of_a_server(requests, page):
    """Prompts, decode steps, trees kept in part, releases, with idle requests and padding."""
    rng = random.Random(requests)
    b = Both(requests, 12, requests * 6 + 3, page, requests)
    b.step([rng.randrange(0, 3 * page) for _ in range(requests)], 3 * page * requests)
    for _ in range(3):
        rows = [rng.choice([0, 1, 1]) for _ in range(requests)]
        b.step(rows, sum(rows) + rng.randrange(4))
        nodes, before = [rng.randrange(1, 9) for _ in range(requests)], list(b.lengths)
        b.step(nodes, sum(nodes) + 2, max_rows=9)
        keep = [rng.random() < 0.4 for _ in range(sum(nodes) + 2)]
        b.step(nodes, sum(nodes) + 2, base=before, keep=keep)
        gone = [0 if rng.random() < 0.3 else n for n in b.lengths]
        b.step([0] * requests, 1, base=gone)


@pytest.mark.parametrize("total", [4096, 4097, 20000])
@pytest.mark.parametrize("keep", [False, True])
def test_many_rows(total, keep):
    """Either side of the rows that one workgroup places."""
    rng = random.Random(total)
    b = Both(7, 700, 4000, 16, 1)
    rows = [total // 10, 0, total // 3, 1, 0, total // 4, 17]
    b.step(rows, total, keep=[rng.random() < 0.6 for _ in range(total)] if keep else None)
    b.step([0] * 7, 3, base=[0] * 7)


@pytest.mark.parametrize("total", [100, 4096, 4097, 20000])
def test_steps_without_a_plan(total):
    """At the C entry a step whose plan nobody needs places its rows like one with a plan."""
    requests, page, capacity, pages = 9, 32, 800, 1500
    lib, rows = _lib.load(), i32([total // 9 - 3] * 8 + [total // 3])
    out = []
    for planned in (True, False):
        tables = [i32([0, 40, 7, 0, 31, 32, 33, 1, 5]), torch.full((requests, capacity), -1, dtype=torch.int32, device=DEV),
                  i32(list(range(pages))), i32([pages - 10])]
        tables[1][:, :2] = torch.arange(pages - 18, pages, dtype=torch.int32, device=DEV).reshape(9, 2)
        places = [torch.full((total,), -7, dtype=torch.int32, device=DEV) for _ in range(3)]
        plan = torch.empty(lib.qmm4_cache_plan_words(requests, 24, 4, 128, total), dtype=torch.int32, device=DEV) if planned else None
        rc = lib.qmm4_cache_step(*(t.data_ptr() for t in tables), rows.data_ptr(), None, None, *(t.data_ptr() for t in places),
                                 plan.data_ptr() if planned else None, requests, capacity, pages, total, total, page, 24, 4, 128,
                                 torch.cuda.current_stream().cuda_stream)
        assert rc == 0, _lib.last_error()
        out.append(places + tables)
    for a, b in zip(*out):
        assert torch.equal(a, b) and a.min() > -7
    assert (out[0][2] >= 0).sum() == min(total, int(rows.sum()))


def test_pages_given_back_are_taken_again():
    b = Both(5, 20, 60, 16, 2)
    b.step([30, 5, 64, 16, 1], 116)
    before, table = list(b.lengths), b.table.copy()
    one = b.step([20] * 5, 100)
    b.step([0] * 5, 1, base=before)
    assert (b.table == table).all()
    two = b.step([20] * 5, 100)
    assert torch.equal(one.slots, two.slots)


def test_too_few_pages_refuse_from_the_first_that_lacks_them():
    b = Both(5, 20, 8, 16, 3)
    step = b.step([30, 100, 1, 0, 5], 136)  # 2 pages, 7 of the 6 left, then every request that needs any
    assert b.lengths == [30, 0, 0, 0, 0] and (step.request[30:] == -1).all()
    b.step([2, 0, 0, 0, 0], 2)              # within its last page
    b.step([0, 1, 1, 0, 1], 3)
    b.step([1, 0, 0, 0, 80], 81, base=[32, 0, 0, 0, 0])  # what comes back may be taken at once
    b.step([0] * 5, 1, base=[0] * 5)
    assert b.count == 8


def test_a_full_table_refuses_its_request_only():
    b = Both(3, 2, 20, 16, 4)
    b.step([33, 32, 1], 66)
    assert b.lengths == [0, 32, 1]
    b.step([32, 1, 5], 38)
    assert b.lengths == [32, 32, 6]


def test_odd_arguments():
    """Rows below zero and past max_rows or total, bases out of range."""
    b = Both(4, 10, 40, 16, 5)
    b.step([-3, 9, 4, 2], 12, max_rows=5)
    b.step([1, 1, 1, 1], 2)
    b.step([1, 1, 1, 1], 9, base=[-5, 2, 100, 0])
    b.step([5, 5, 5, 5], 0)
    b.step([5, 5, 5, 5], 20, max_rows=0)


def test_no_requests_and_no_pages():
    t = [i32([]), torch.empty((0, 4), dtype=torch.int32, device=DEV), i32([3, 1]), i32([2])]
    step = step_tables_(*t, i32([]), 3, 16, 8, 2, 64)
    assert step.slots.tolist() == step.positions.tolist() == step.request.tolist() == [-1] * 3 and t[3].item() == 2
    b = Both(2, 3, 0, 16)
    b.step([1, 0], 2)


def test_broken_numbers_stay_in_bounds():
    """Lengths and counts that cannot be are taken as the nearest that can."""
    t = [i32([-5, 10**9, 20]), torch.full((3, 4), -1, dtype=torch.int32, device=DEV), i32([0, 1, 2, 3]), i32([9])]
    step = step_tables_(*t, i32([1, 1, 1]), 3, 16, 8, 2, 64, base=i32([0, 40, -1]))
    assert t[0].tolist()[0] == 1 and t[3].item() <= 4 and step.request.shape == (3,)


def test_captured():
    """A captured step is replayed with other rows between the program's own work."""
    tables, mirror = CacheTables(6, 40, 200, 16, 24, 4, 256, DEV), CacheTables(6, 40, 200, 16, 24, 4, 256, DEV)
    rows, keep = i32([0] * 6), torch.zeros(12, dtype=torch.bool, device=DEV)
    tables.step(rows, 12), mirror.step(rows, 12)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    base = i32([0] * 6)
    with torch.cuda.graph(graph):
        base.copy_(tables.lengths)
        one = tables.step(rows, 12)
        two = tables.step(rows, 12, base=base, keep=keep)
    rng = random.Random(8)
    for _ in range(5):
        rows.copy_(i32([rng.randrange(4) for _ in range(6)]))
        keep.copy_(torch.tensor([rng.random() < 0.5 for _ in range(12)], device=DEV))
        before = mirror.lengths.clone()
        want = mirror.step(rows, 12), mirror.step(rows, 12, base=before, keep=keep)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip((one, two), want):
            assert all(torch.equal(a, b) for a, b in zip(g[:3], w[:3]))
        for name in ("lengths", "block_table", "free_count"):
            assert torch.equal(getattr(tables, name), getattr(mirror, name))


def test_plain_and_native_calls_agree(monkeypatch):
    from mlx_tree_spec_amd import _lib
    rows = i32([3, 0, 40, 7])
    out = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_native", _lib._NoNative)
        tables = CacheTables(4, 40, 60, 16, 24, 4, 256, DEV)
        out.append([*tables.step(rows, 51)[:4], tables.lengths, tables.block_table])
    words = int(out[0][3][0])
    assert words == int(out[1][3][0])
    for i in (0, 1, 2, 4, 5):
        assert torch.equal(out[0][i], out[1][i])
