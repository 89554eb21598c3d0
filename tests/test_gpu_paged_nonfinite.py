"""Infinities and NaN in the paged cache (needs an MI355X): each row has what the formula gives of the tokens that it sees, in 64
bits: NaN and infinities of the same sign where that has them, and finite values within the attention's bound elsewhere."""

import numpy as np
import pytest
import torch

import cache_refs as R
from request_refs import f64
from test_gpu_paged import Case

pytestmark = pytest.mark.gpu
KINDS = (float("nan"), float("inf"), -float("inf"))


def put(case, request, token, which, head, d, x):
    """x as dimension d of a token's key or value."""
    page = case.step.page_size
    p, o = int(case.table[request, token // page]), token % page
    if which == "keys":
        case.cache.keys[p, head, d // 8, o, d % 8] = x
    else:
        case.cache.values[p, head, o // 8, d, o % 8] = x


def poison_values(case, request, tokens):
    """A dimension of its own that is not finite in the value of each of the tokens, in the last key head."""
    head, dim = case.cache.keys.shape[1] - 1, case.q.shape[2]
    assert len(set(tokens)) == len(tokens) < dim
    for i, t in enumerate(tokens):
        put(case, request, t, "values", head, i * 5 % dim, KINDS[i % 3])


def check(case, out):
    k, v = R.token_rows(case.cache)
    q, got, page, row = f64(case.q), f64(out), case.step.page_size, 0
    for r, (c, n) in enumerate(zip(case.cached, case.rows)):
        if n == 0:
            continue
        t = np.arange(c + n)
        at = case.table[r, t // page].astype(np.int64) * page + t % page
        masks = None if case.ancestors is None else case.ancestors[row:row + n].tolist()
        with np.errstate(all="ignore"):
            want, mag, delta = R.attention(q[row:row + n], k[at], v[at], case.scale, R.visible(c, n, masks))
            if case.gate is not None:
                s = 1 / (1 + np.exp(-f64(case.gate[row:row + n])))
                want, mag = want * s, mag * s
            bound = R.attention_bound(want, mag, delta, c + n)
            here = got[row:row + n]
            assert np.array_equal(np.isnan(here), np.isnan(want)), (r, c, n)
            inf = np.isinf(want)
            assert np.array_equal(np.isinf(here), inf) and (here[inf] == want[inf]).all(), (r, c, n)
            finite = np.isfinite(want)
            assert (np.abs(here - want)[finite] <= bound[finite]).all(), (r, c, n)
        row += n
    assert not got[row:].any()


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("rows", [20, 40])
def test_values_of_the_first_stage(rows, dim, tree):
    """Requests of one stage and no context: what is not finite in it is known from the first barrier on."""
    case = Case([0, 0], [rows, 7], 6, 2, dim, tree=tree, gated=tree, seed=dim + rows)
    poison_values(case, 0, [0, 5, 13, rows - 1])
    poison_values(case, 1, [1, 6])
    check(case, case.run())


CONTEXTS = [40, 10, 31, 100, 63, 64, 700, 5030]
# Query rows of a key head: up to 16 (one wave's), up to 64 and more (trees; 16 and 32 rows to a wave of the narrower heads).
FORMS = [(1, 3), (5, 3), (20, 3), (40, 3), (64, 1)]


def interesting(c, n):
    """Tokens in and in front of the stage that the context ends in, in both of its halves, and among the step's."""
    stage = c // 64 * 64
    return sorted({t for t in (0, 3, stage - 33, stage - 1, stage, stage + 10, stage + 31, stage + 32, c - 1, c, c + 1, c + n // 2,
                               c + n - 1) if 0 <= t < c + n})


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("rows,group", FORMS)
def test_values(rows, group, dim, page, tree):
    """Cached tokens' values and the step's own, in every kernel's form, in requests of one split and of many."""
    case = Case(CONTEXTS, [rows] * len(CONTEXTS), 2 * group, 2, dim, page=page, tree=tree, gated=tree, seed=dim + rows, max_rows=rows)
    for r, c in enumerate(CONTEXTS):
        poison_values(case, r, interesting(c, rows))
    check(case, case.run())


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("rows,group", FORMS)
def test_keys(rows, group, dim):
    """A key that is not finite in each request, at another place."""
    case = Case(CONTEXTS, [rows] * len(CONTEXTS), 2 * group, 2, dim, tree=True, seed=dim + rows, max_rows=rows)
    for r, c in enumerate(CONTEXTS):
        tokens = interesting(c, rows)
        put(case, r, tokens[-1 - r % len(tokens)], "keys", r % 2, r * 7, KINDS[r % 3])
    check(case, case.run())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,group", FORMS)
def test_scales_of_8_bits(rows, group, dim):
    """A token of each request whose scale is NaN, as a head that was not finite is stored: of its keys, or of its values."""
    case = Case(CONTEXTS, [rows] * len(CONTEXTS), 2 * group, 2, dim, bits=8, tree=True, gated=True, seed=dim + rows, max_rows=rows)
    for r, c in enumerate(CONTEXTS):
        tokens = interesting(c, rows)
        for h, (scales, t) in enumerate(((case.cache.key_scales, tokens[-1 - r % len(tokens)]), (case.cache.value_scales, tokens[r % len(tokens)]))):
            scales[int(case.table[r, t // 64]), h, t % 64] = float("nan")
    check(case, case.run())


def test_cut_and_whole_requests_agree_about_every_context():
    """Contexts of all lengths modulo a stage, each with an infinite value in the stage it ends in."""
    cached = list(range(64, 128))
    case = Case(cached, [7] * 64, 6, 2, 64, tree=True, seed=3, max_rows=7)
    for r, c in enumerate(cached):
        poison_values(case, r, [64 + r // 2, 63] if r else [63])
    check(case, case.run())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_prompts(dim):
    """Several row blocks of a request, each of which ends in a stage of its own."""
    case = Case([0, 100, 40], [300, 150, 90], 4, 2, dim, gated=True, seed=dim)
    for r, (c, n) in enumerate(zip(case.cached, case.rows)):
        poison_values(case, r, sorted({*interesting(c, n), *(t for t in (c + 63, c + 70, c + 130, c + 200) if t < c + n)}))
    check(case, case.run())
