"""The routes of the adapters' GPU tests, from the built planners (CPU only, no GPU call)."""

import adapter_cases as C
from test_plans import dispatch_route, planner_exe, query  # noqa: F401  (a fixture among them)

THREADS = 512  # of a row-split workgroup


def first_items(m, n, p):
    """(items of a range, threads of the last range that write an item other than their own number first): item i of a
    range of R columns is column i % R of lane group i / R, thread t takes t, t + 512, .., and items past the range's
    last column or the last row are none."""
    groups, slices = int(p["MP"]) // 4, int(p["KS"])
    width = (-(-n // max(1, C.CUS // slices)) + 3) // 4 * 4
    ranges = -(-n // width)
    assert ranges * slices == int(p["blocks"])
    last = n - (ranges - 1) * width
    late = 0
    for t in range(THREADS):
        mine = [i for i in range(t, width * groups, THREADS) if i % width < last and 4 * (i // width) < m]
        late += bool(mine) and mine[0] != t
    return width * groups, late


def test_rowsplit_cases_take_their_routes(planner_exe):  # noqa: F811
    shapes = [(m, n, k) for m, k, n, *_ in C.ROWSPLIT]
    assert dispatch_route(planner_exe, shapes) == ["row-split"] * len(shapes)
    plans = query(planner_exe, [f"rowsplit {m} {n} {k} {C.CUS}" for m, n, k in shapes])
    for (m, k, n, slices, steps, form, wrapped), p in zip(C.ROWSPLIT, plans):
        takes = "small" if p["small"] == "1" else "groups" if p["pair"] == "1" else "own" if p["own"] == "1" else "slots"
        assert (int(p["KS"]), int(p["V"]), takes) == (slices, steps, form), (m, k, n, p)
        items, late = first_items(m, n, p)
        assert (late > 0) == wrapped and (items > THREADS or not wrapped), (m, k, n, items, late)


def gemm_form(m, k, n, p):
    plain = k % 512 != 0
    if p["sk"] == "1":
        tile = "256x256" if p["sk256"] == "1" else "128x256" if p["sk_wide"] == "1" else "128x128"
        return f"stream-K {tile}" + ", plain" * plain
    tiles = -(-m // 256) * -(-n // 256)
    tail = tiles % C.CUS
    if tail == 0 or 4 * tail > 2 * C.CUS:
        return "whole" + ", plain" * plain
    cut = "stream-K" if p["tail_sk"] == "1" else "quarters"
    return cut + ", plain" * plain if tail == tiles else "whole" + ", plain" * plain + ", tail in " + cut


def test_gemm_cases_take_their_routes(planner_exe):  # noqa: F811
    shapes = [(m, n, k) for m, k, n, _ in C.GEMM]
    assert dispatch_route(planner_exe, shapes) == ["gemm"] * len(shapes)
    plans = query(planner_exe, [f"gemm {m} {n} {k} {C.CUS}" for m, n, k in shapes])
    for (m, k, n, form), p in zip(C.GEMM, plans):
        assert gemm_form(m, k, n, p) == form, (m, k, n, p)


def test_rowphase_cases_take_their_variants(planner_exe):  # noqa: F811
    shapes = [(m, n, k) for m, k, n, *_ in C.ROWPHASE]
    assert dispatch_route(planner_exe, shapes) == ["row-phase"] * len(shapes)
    plans = query(planner_exe, [f"rowphase {m} {n} {k} {C.CUS}" for m, n, k in shapes])
    for (m, k, n, variant, split), p in zip(C.ROWPHASE, plans):
        assert (int(p["variant"]), int(p["S"]) > 1) == (variant, split), (m, k, n, p)
    assert {case[3] for case in C.ROWPHASE} == set(range(2, 28))


def test_other_cases_take_the_remaining_kernels(planner_exe):  # noqa: F811
    shapes = [(m, n, k) for m, k, n in C.VERIFY + C.SKINNY]
    assert dispatch_route(planner_exe, shapes) == ["other"] * len(shapes)
    assert all(m >= 5 for m, *_ in C.VERIFY) and all(m <= 4 for m, *_ in C.SKINNY)
