"""The per-request operators past 4 GiB of an input and past a grid's rows (needs an MI355X).

What lies past 32 bits of offset is compared with 64 bits, by the bounds of the operators' own tests, or with the same
call on a copy of the last rows (each row is computed by itself, so its bits may not change)."""

import numpy as np
import pytest
import torch

import request_refs as R
from mlx_tree_spec_amd import qk_norm_rope, quantized_matmul_lora, sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("m", [4, 13, 40, 300])
@pytest.mark.parametrize("k,n,count", [(512, 8192, 1050), (8192, 512, 1050)])
def test_adapter_tables_past_4_gib(m, k, n, count):
    rank = 256
    g = torch.Generator().manual_seed(m + k)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    used = torch.tensor([0, count // 2, count - 1])
    la = torch.zeros(count, rank, k, dtype=torch.bfloat16, device=DEV)
    lb = torch.zeros(count, n, rank, dtype=torch.bfloat16, device=DEV)
    assert max(la.numel(), lb.numel()) * 2 > 1 << 32
    scale = torch.rand(count, generator=g).to(DEV)
    for a in used.tolist():
        la[a] = (randn(rank, k) / k ** 0.5).to(torch.bfloat16).to(DEV)
        lb[a] = (randn(n, rank) * 0.3).to(torch.bfloat16).to(DEV)
    x = randn(m, k).to(torch.bfloat16).to(DEV)
    w = torch.randint(-2**31, 2**31, (n, k // 8), generator=g, dtype=torch.int64).to(torch.int32).to(DEV)
    s = (randn(n, k // 64).abs() * 0.004 + 1e-4).to(torch.bfloat16).to(DEV)
    b = (-8 * s.float()).to(torch.bfloat16)
    pick = torch.randint(0, 3, (m,), generator=g)
    y = quantized_matmul_lora(x, w, s, b, la, lb, scale, used[pick].to(torch.int32).to(DEV))
    ref, _, mag = R.lora(x, R.dequantize(w, s, b, 64, 4), la[used.to(DEV)], lb[used.to(DEV)], scale[used.to(DEV)], pick)
    bound = R.HALF_STEP_BF16 * np.abs(ref) * 1.01 + ((k + rank + 4) * R.HALF_STEP_F32 + 2.0 ** -18) * mag
    assert (np.abs(R.f64(y) - ref) <= bound).all()


@pytest.mark.parametrize("m,v", [(70000, 32001), (16000, 151936)])
def test_logits_past_4_gib(m, v):
    logits = torch.empty(m, v, dtype=torch.bfloat16, device=DEV)
    assert logits.numel() * 2 > 1 << 32
    g = torch.Generator(device=DEV).manual_seed(v)
    logits.fill_(-1.0)
    logits[-4:] = (torch.randn(4, v, generator=g, device=DEV) * 2).to(torch.bfloat16)
    logits[:3] = (torch.randn(3, v, generator=g, device=DEV) * 2).to(torch.bfloat16)
    uniform = torch.rand(m, generator=g, device=DEV)
    tokens, logprobs = sample(logits, uniform, top_p=0.9)
    for rows in (slice(0, 3), slice(m - 4, m)):
        want, want_p = R.sample(logits[rows], uniform[rows], top_p=0.9)
        assert np.array_equal(tokens[rows].cpu().numpy(), want)
        assert (np.abs(R.f64(logprobs[rows]) - want_p) <= R.HALF_STEP_F32 * np.abs(want_p) * 1.01 + 2.0 ** -40).all()
    assert int(tokens.min()) >= 0 and int(tokens.max()) < v


@pytest.mark.parametrize("m,hq,hk,d", [(600000, 32, 1, 128), ((1 << 24) + 5, 1, 1, 8)])
def test_heads_past_4_gib_and_past_a_grid(m, hq, hk, d):
    g = torch.Generator(device=DEV).manual_seed(d)
    q = torch.randn(m, hq, d, generator=g, device=DEV, dtype=torch.bfloat16)
    k = torch.randn(m, hk, d, generator=g, device=DEV, dtype=torch.bfloat16)
    wq, wk = (torch.rand(d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    positions = torch.randint(0, 1 << 17, (m,), generator=g, device=DEV)
    inv = 1e4 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) / (d // 2))
    out = qk_norm_rope(q, k, wq, wk, 1e-6, positions, inv)
    for at in (0, (1 << 23) - 3 if m > 1 << 23 else 524285, m - 7):
        part = slice(at, at + 7)
        same = qk_norm_rope(q[part].clone(), k[part].clone(), wq, wk, 1e-6, positions[part].clone(), inv)
        for a, b, x, w in ((out[0], same[0], q, wq), (out[1], same[1], k, wk)):
            assert torch.equal(a[part], b)
            ref, mag = R.rope(x[part], w, 1e-6, positions[part], inv, False)
            bound = R.HALF_STEP_BF16 * np.abs(ref) * 1.001 + (d / 2 + 16) * R.HALF_STEP_F32 * mag
            assert (np.abs(R.f64(a[part]) - ref) <= bound).all()


def test_adapter_rows_past_a_grid():
    """More than 2^22 rows: several launches of the shrink; a library product's result with the adapters added."""
    m, k, n = (1 << 22) + 37, 32, 8
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(m, k, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randint(-2**31, 2**31 - 1, (n, k // 8), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    s = torch.full((n, 1), 2.0 ** -6, dtype=torch.bfloat16, device=DEV)
    b = torch.full((n, 1), -0.125, dtype=torch.bfloat16, device=DEV)
    la, lb = (torch.randn(3, *shape, generator=g, device=DEV).to(torch.bfloat16) for shape in ((8, k), (n, 8)))
    scale = torch.tensor([0.5, 1.0, -0.25], device=DEV)
    ids = torch.randint(-1, 3, (m,), generator=g, device=DEV)
    y = quantized_matmul_lora(x, w, s, b, la, lb, scale, ids, group_size=32)
    wd = R.dequantize(w, s, b, 32, 4)
    for at in (0, (1 << 22) - 20, m - 30):
        part = slice(at, at + 30)
        ref, base, mag = R.lora(x[part], wd, la, lb, scale, ids[part])
        bound = R.HALF_STEP_BF16 * (np.abs(ref) + np.abs(base)) * 1.01 + ((k + 12) * R.HALF_STEP_F32 + 2.0 ** -18) * mag
        assert (np.abs(R.f64(y[part]) - ref) <= bound).all()


def sampled(logits, uniform, **settings):
    tokens, logprobs = sample(logits, uniform, **settings)
    want, want_p = R.sample(logits, uniform, **settings)
    assert np.array_equal(tokens.cpu().numpy(), want)
    assert (np.abs(R.f64(logprobs) - want_p) <= R.HALF_STEP_F32 * np.abs(want_p) * 1.01 + 2.0 ** -40).all()


@pytest.mark.parametrize("settings", [dict(), dict(top_k=100000, top_p=0.8, min_p=1e-5)], ids=str)
def test_largest_vocabulary(settings):
    g = torch.Generator().manual_seed(24)
    logits = (torch.randn(2, 1 << 24, generator=g) * 2).to(torch.bfloat16).to(DEV)
    sampled(logits, torch.tensor([0.25, 0.875], device=DEV), **settings)


@pytest.mark.parametrize("v", [65535, 65536, 1 << 20])
def test_equal_logits_fill_the_counts(v):
    """Every logit the same (16-bit counts at their most), but one above and one below in other slices."""
    logits = torch.full((4, v), -3.0, dtype=torch.bfloat16, device=DEV)
    logits[1, v - 1], logits[2, 0] = -2.984375, -3.015625
    logits[3, v // 2] = -2.984375
    sampled(logits, torch.tensor([0.5, 0.25, 0.75, 0.125], device=DEV), top_p=0.75)


def test_calls_on_two_streams_at_once():
    """Each call has a workspace of its own (the adapters' also their stream's): the results are those of one stream."""
    g = torch.Generator(device=DEV).manual_seed(5)
    logits = (torch.randn(2, 3, 151936, generator=g, device=DEV) * 2).to(torch.bfloat16)
    uniform = torch.rand(2, 3, generator=g, device=DEV)
    x = torch.randn(2, 7, 1024, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randint(-2**31, 2**31 - 1, (512, 128), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    s = torch.full((512, 16), 2.0 ** -6, dtype=torch.bfloat16, device=DEV)
    b = torch.full((512, 16), -0.125, dtype=torch.bfloat16, device=DEV)
    la, lb = (torch.randn(3, *shape, generator=g, device=DEV).to(torch.bfloat16) for shape in ((16, 1024), (512, 16)))
    scale = torch.tensor([0.5, 1.0, -0.25], device=DEV)
    ids = torch.randint(-1, 3, (2, 7), generator=g, device=DEV)
    both = lambda i: (*sample(logits[i], uniform[i], top_p=0.9),  # noqa: E731
                      quantized_matmul_lora(x[i], w, s, b, la, lb, scale, ids[i]))
    want = [both(0), both(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(both(i))
    torch.cuda.synchronize()
    for i in range(2):
        for result in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(result, want[i]))
