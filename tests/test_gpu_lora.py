"""Low-rank adapters beside a quantized projection, on the GPU (needs an MI355X), against 64 bits.

Bound per value: the result rounded to bf16 (half a step; the projection's own rounding as well where a library product
computes it), x A^T kept to 2^-18 of its value, and fp32 sums of n terms, whose error is at most n half steps of fp32
of the sum of the terms' magnitudes, whatever their order (n = K + R + 4 covers the K products, the R products of the
second factor and the scale).
"""

import numpy as np
import pytest
import torch

import request_refs as R
from mlx_tree_spec_amd import LoRALinear, QuantizedLinear, quantized_matmul, quantized_matmul_lora, stack_adapters

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inputs(m, k, n, rank, count, seed, bits=4, group=64, ids=None):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = randn(m, k).to(torch.bfloat16)
    w = torch.randint(-2**31, 2**31, (n, k * bits // 32), generator=g, dtype=torch.int64).to(torch.int32)
    s = ((randn(n, k // group).abs() * 0.004 + 1e-4) * 2.0 ** (4 - bits)).to(torch.bfloat16)
    b = (-(2.0 ** (bits - 1)) * s.float() + randn(n, k // group) * 1e-3).to(torch.bfloat16)
    la = (randn(count, rank, k) / k ** 0.5).to(torch.bfloat16)
    lb = (randn(count, n, rank) * 0.3).to(torch.bfloat16)
    scale = torch.rand(count, generator=g) * 3 - 1.5
    if ids is None:
        ids = torch.randint(-1, count, (m,), generator=g)
    return [t.to(DEV) for t in (x, w, s, b, la, lb, scale, torch.as_tensor(ids, dtype=torch.int32))]


def check(args, y, group=64, bits=4, twice=False):
    x, w, s, b, la, lb, scale, ids = args
    m = x.reshape(-1, x.shape[-1]).shape[0]
    ref, base, mag = R.lora(x.reshape(m, -1), R.dequantize(w, s, b, group, bits), la, lb, scale, ids.reshape(-1))
    k, rank = x.shape[-1], la.shape[1]
    rounded = np.abs(ref) + (np.abs(base) if twice else 0)
    bound = R.HALF_STEP_BF16 * rounded * 1.01 + ((k + rank + 4) * R.HALF_STEP_F32 + 2.0 ** -18) * mag
    err = np.abs(R.f64(y).reshape(m, -1) - ref)
    assert (err <= bound).all(), (float((err - bound).max()), np.unravel_index((err - bound).argmax(), err.shape))


# Every route of the projection (row-split whole K and K slices, 9-16 rows over a small problem, row-phase wide and
# K split, verify, skinny, the GEMM's tiles and stream-K), one row to many, every adapter mixed row by row.
@pytest.mark.parametrize("m,k,n", [(1, 128, 16), (1, 5120, 512), (3, 1024, 2048), (4, 2560, 8192), (7, 1024, 10240),
                                   (8, 4096, 4096), (13, 2048, 1024), (16, 5120, 640), (17, 512, 528), (24, 1152, 144),
                                   (40, 640, 512), (64, 4096, 1024), (64, 512, 16384), (65, 2048, 2048), (90, 384, 1040),
                                   (113, 1024, 256), (130, 512, 2080), (257, 256, 512), (515, 1024, 768)])
@pytest.mark.parametrize("rank", [8, 24])
def test_matches_64_bits(m, k, n, rank):
    args = inputs(m, k, n, rank, 5, m * 31 + k + n + rank)
    check(args, quantized_matmul_lora(*args))


@pytest.mark.parametrize("rank", [8, 16, 32, 64, 72, 128, 256])
@pytest.mark.parametrize("m", [1, 5, 33, 200])
def test_ranks(m, rank):
    args = inputs(m, 512, 272, rank, 3, m + rank)
    check(args, quantized_matmul_lora(*args))


# Formats and shapes of the general path: odd columns, 2- and 8-bit codes, K that is not a multiple of 128.
@pytest.mark.parametrize("m,k,n,bits,group", [(1, 64, 1, 4, 64), (5, 192, 33, 4, 64), (20, 512, 515, 8, 32),
                                              (64, 256, 127, 2, 64), (9, 384, 96, 4, 128), (300, 128, 77, 8, 64)])
def test_general_formats(m, k, n, bits, group):
    args = inputs(m, k, n, 16, 4, m + n, bits, group)
    check(args, quantized_matmul_lora(*args, group_size=group, bits=bits), group, bits)


# K that the general kernel does not take: the projection by dequantization and a library product.
@pytest.mark.parametrize("m,k,n", [(1, 96, 5), (7, 96, 40), (70, 160, 300)])
def test_added_to_a_library_product(m, k, n):
    args = inputs(m, k, n, 24, 4, m + n, 4, 32)
    check(args, quantized_matmul_lora(*args, group_size=32), 32, 4, twice=True)


# Many rows of one adapter next to others (a prompt's tiles), long K in slices, and adapters far apart in the tables.
@pytest.mark.parametrize("m,k,n,rank", [(300, 2048, 1040, 32), (64, 17408, 512, 32), (1030, 512, 2064, 64), (30, 8192, 4096, 8)])
def test_runs_of_requests(m, k, n, rank):
    ids = torch.tensor([2] * (m // 2) + [-1] * (m // 8) + [0] * (m // 4 + 1) + [1] * m)[:m]
    args = inputs(m, k, n, rank, 3, m + k, ids=ids)
    check(args, quantized_matmul_lora(*args))


@pytest.mark.parametrize("m,k,n,bits,group", [(6, 512, 272, 4, 64), (70, 512, 512, 4, 64), (6, 192, 35, 4, 64)])
def test_rows_without_an_adapter_are_the_projection(m, k, n, bits, group):
    ids = torch.tensor([-1, 4, 0, 2**31 - 1, -2**31, 3] + [5] * (m - 6))  # 4 adapters: only 0 and 3 exist
    args = inputs(m, k, n, 8, 4, 3, bits, group, ids)
    y = quantized_matmul_lora(*args)
    base = quantized_matmul(*args[:4])
    bare = torch.tensor([i not in (2, 5) for i in range(m)])
    assert torch.equal(y[bare], base[bare])
    check(args, y)
    none = quantized_matmul_lora(*args[:7], torch.full((m,), -1, dtype=torch.int32, device=DEV))
    assert torch.equal(none, base)


def test_no_adapters_and_no_rows():
    args = inputs(4, 256, 64, 8, 2, 1)
    x, w, s, b, la, lb, scale, ids = args
    y = quantized_matmul_lora(x, w, s, b, la[:0], lb[:0], scale[:0], ids)
    assert torch.equal(y, quantized_matmul(x, w, s, b))
    assert quantized_matmul_lora(x[:0], w, s, b, la, lb, scale, ids[:0]).shape == (0, 64)


def test_nonfinite_adapters_stay_with_their_rows():
    """An adapter of infinities and NaN that no row uses, or that one row uses, touches no other row."""
    args = inputs(20, 512, 256, 8, 3, 11, ids=[0, 2] * 10)
    args[4][1], args[5][1] = float("nan"), float("inf")
    clean = quantized_matmul_lora(*args)
    check([a if i not in (4, 5) else a[[0, 0, 2]] for i, a in enumerate(args)], clean)
    args[7][4] = 1
    y = quantized_matmul_lora(*args)
    keep = torch.arange(20) != 4
    assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[4].float()).any()


def test_shapes_strides_and_index_types():
    args = inputs(12, 512, 272, 16, 3, 8)
    x, w, s, b, la, lb, scale, ids = args
    y = quantized_matmul_lora(*args)
    y3 = quantized_matmul_lora(x.reshape(3, 4, 512), w, s, b, la, lb, scale, ids.reshape(3, 4).long())
    assert y3.shape == (3, 4, 272) and torch.equal(y3.reshape(12, 272), y)
    xs = torch.empty(12, 1024 + 8, dtype=torch.bfloat16, device=DEV)[:, 4:516]
    xs.copy_(x)
    off = torch.empty(la.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].reshape(la.shape)  # 2-byte offset
    off.copy_(la)
    lbt = lb.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.empty(24, dtype=torch.int32, device=DEV)[::2]
    wide.copy_(ids)
    assert torch.equal(quantized_matmul_lora(xs, w, s, b, off, lbt, scale, wide), y)


def test_deterministic_and_on_a_stream():
    args = inputs(64, 2048, 1024, 32, 4, 9)
    y = quantized_matmul_lora(*args)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y2 = quantized_matmul_lora(*args)
    stream.synchronize()
    assert torch.equal(y, y2)


@pytest.mark.parametrize("m,n,bits,group", [(3, 512, 4, 64), (64, 512, 4, 64), (200, 512, 4, 64), (9, 515, 8, 32)])
def test_captured(m, n, bits, group):
    """Two graphs on one stream, each with a workspace of its own, replayed with new inputs between eager work."""
    kw = dict(bits=bits, group_size=group)
    args = inputs(m, 1024, n, 16, 3, m, bits, group)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        quantized_matmul_lora(*args, **kw)
    stream.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(quantized_matmul_lora(*args, **kw))
        graphs.append(g)
    for i in range(4):
        fresh = inputs(m, 1024, n, 16, 3, m + 100 + i, bits, group)
        args[0].copy_(fresh[0])
        args[7].copy_(fresh[7])
        want = quantized_matmul_lora(*args, **kw)
        torch.cuda.synchronize()
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_module_and_stacked_ranks():
    g = torch.Generator().manual_seed(5)
    x, w, s, b, *_ = inputs(10, 512, 256, 8, 1, 2)
    adapters = [(torch.randn(r, 512, generator=g) / 20, torch.randn(256, r, generator=g) / 5, 0.5 + r) for r in (4, 1, 11)]
    la, lb, scale = stack_adapters(adapters, device=DEV)
    assert la.shape == (3, 16, 512) and lb.shape == (3, 256, 16) and not la[1, 1:].any() and not lb[0, :, 4:].any()
    layer = LoRALinear(QuantizedLinear.from_quantized(w, s, b), la, lb, scale)
    ids = torch.tensor([0, 1, 2, -1, 2, 2, 0, 1, -1, 0], dtype=torch.int32, device=DEV)
    check([x, w, s, b, la, lb, scale, ids], layer(x, ids))
    assert torch.equal(layer(x), quantized_matmul(x, w, s, b))
