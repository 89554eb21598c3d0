"""Attention over small pages past 16384 tokens of one split (needs an MI355X): page numbers come in segments of 1024, and a split
that is not cut goes through several. Rows and heads of one request, enough that its plan has one split; some of them against 64 bits."""

import numpy as np
import pytest

import cache_refs as R
from request_refs import f64
from test_gpu_paged import Case

pytestmark = pytest.mark.gpu
GROUP, ROWS = 256, 66  # (132 blocks of 128 query rows: more than half of what the GPU holds at once)


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dim,page,bits", [(64, 16, 16), (128, 16, 8), (256, 16, 16), (64, 32, 16)])
@pytest.mark.parametrize("cached", [16384 - 66, 16384 - 30, 2 * 16384 + 600])
def test_segments_of_pages(cached, dim, page, bits, odd):
    if odd and bits == 8:
        pytest.skip("codes are finite")
    case = Case([cached], [ROWS], GROUP, 1, dim, page=page, bits=bits, seed=dim + page)
    assert int(case.step.plan[8 + 4]) == 1  # splits
    tokens = [3, 16383, 16384, cached // 64 * 64 + 5, cached // 64 * 64 + 40, cached + 1, cached + ROWS - 1]
    if odd:
        for i, t in enumerate(sorted({t for t in tokens if t < cached + ROWS})):
            case.cache.values[int(case.table[0, t // page]), 0, t % page // 8, 9 * i, t % 8] = (float("nan"), float("inf"), -float("inf"))[i % 3]
    out = f64(case.run())
    k, v = R.token_rows(case.cache)
    t = np.arange(cached + ROWS)
    at = case.table[0, t // page].astype(np.int64) * page + t % page
    rows, heads = [0, 1, 33, ROWS - 2, ROWS - 1], list(range(3, GROUP, 36))
    with np.errstate(all="ignore"):
        want, mag, delta = R.attention(f64(case.q)[rows][:, heads], k[at], v[at], case.scale, R.visible(cached, ROWS)[rows])
        bound = R.attention_bound(want, mag, delta, cached + ROWS)
        got, finite = out[rows][:, heads], np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and (got[np.isinf(want)] == want[np.isinf(want)]).all()
        assert (np.abs(got - want)[finite] <= bound[finite]).all()
    assert odd or finite.all()
    assert np.isfinite(out).all() or odd
