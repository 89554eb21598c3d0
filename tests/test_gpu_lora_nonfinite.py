"""Adapters with infinities and NaN (needs an MI355X): each value is what the formula gives, whatever shares its tile.

A value with a finite result keeps the bound of test_gpu_lora.py; one that is infinite or NaN in 64 bits is that
infinity or NaN. An infinity's sign is that of its product's other factor, and those lie far from zero here."""

import numpy as np
import pytest
import torch

import request_refs as R
from adapter_cases import GEMM
from mlx_tree_spec_amd import quantized_matmul_lora
from test_gpu_lora import inputs

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def spoil(args):
    """Adapters 1 and 2 with values that are not finite: columns of B, one row of A; x of adapter 3's first row."""
    x, w, s, b, la, lb, scale, ids = args
    n, rank = lb.shape[1:]
    lb[1, 3, 0] = INF                       # alone in its column
    lb[1, 5, 1], lb[1, 5, 2] = INF, -INF    # two, of one sign or of both by t
    lb[1, n - 1, rank - 1] = NAN
    lb[1, n // 2, rank // 2] = -INF
    la[2, 1, 7], lb[2, 11, 1] = INF, 0.0    # t infinite: beside a zero NaN
    lb[2, 12, 1], lb[2, 13, 0] = INF, INF   # .. beside infinities
    rows = (ids == 3).nonzero()
    if len(rows):
        x[rows[0, 0], 0] = INF              # y is infinite or NaN with its projection
        lb[3, 6, 0] = -INF


def check(args, y, group=64, bits=4, twice=False):
    x, w, s, b, la, lb, scale, ids = args
    with np.errstate(invalid="ignore", over="ignore"):
        ref, base, mag = R.lora(x, R.dequantize(w, s, b, group, bits), la, lb, scale, ids)
        rounded = np.abs(ref) + (np.abs(base) if twice else 0)
        bound = R.HALF_STEP_BF16 * rounded * 1.01 + ((x.shape[1] + la.shape[1] + 4) * R.HALF_STEP_F32 + 2.0 ** -18) * mag
        got = R.f64(y)
        fine = np.isfinite(ref)
        assert np.isfinite(got[fine]).all()
        assert (np.abs(got - ref)[fine] <= bound[fine]).all()
    assert np.array_equal(got[~fine], ref[~fine], equal_nan=True), np.argwhere((~fine) & ~((got == ref) | (np.isnan(got) & np.isnan(ref))))[:5]
    assert np.isinf(ref).any() and np.isnan(ref).any()


def mixed(m, kind):
    if kind == "one":
        return [1] * m
    if kind == "runs":
        return [(0, 1, -1, 2, 3, 1)[i * 6 // m] for i in range(m)]
    return [(i * 7 + i // 5) % 5 - 1 for i in range(m)]


# Single rows (row-split, its forms of 5-16 rows), row-phase whole and split, verify, skinny.
@pytest.mark.parametrize("kind", ["one", "mixed"])
@pytest.mark.parametrize("m,k,n", [(4, 1024, 2048), (7, 1024, 10240), (13, 2048, 1024), (16, 5120, 640), (24, 1152, 144),
                                   (40, 640, 512), (64, 4096, 1024), (64, 512, 16384), (90, 384, 1040)])
def test_few_rows(m, k, n, kind):
    args = inputs(m, k, n, 24, 4, m + k, ids=mixed(m, kind))
    spoil(args)
    check(args, quantized_matmul_lora(*args))


@pytest.mark.parametrize("kind,rank", [("one", 24), ("runs", 40), ("mixed", 8)])
@pytest.mark.parametrize("m,k,n", [case[:3] for case in GEMM])
def test_gemm_forms(m, k, n, kind, rank):
    args = inputs(m, k, n, rank, 4, m + k, ids=mixed(m, kind))
    spoil(args)
    check(args, quantized_matmul_lora(*args))


@pytest.mark.parametrize("m,k,n,bits,group", [(5, 192, 33, 4, 64), (24, 512, 515, 8, 32), (70, 160, 300, 4, 32)])
def test_other_formats(m, k, n, bits, group):
    args = inputs(m, k, n, 24, 4, m + n, bits, group, ids=mixed(m, "mixed"))
    spoil(args)
    check(args, quantized_matmul_lora(*args, group_size=group, bits=bits), group, bits, twice=k % 64 != 0)
