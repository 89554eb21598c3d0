"""Head norms with rotation on the GPU (needs an MI355X), against 64 bits.

Bound per value: one rounding to bf16 (half a step of the value), and of the magnitude of its terms (both values of
its pair) fp32 errors: a sum of D squares is off by at most D half steps, its inverse root by half as many, and 16
more cover the division, root, products, sum, sine and cosine (a few half steps each) and the angle (rounded to
fp32 as at most half a turn: pi half steps).
"""

import numpy as np
import pytest
import torch

import request_refs as R
from mlx_tree_spec_amd import qk_norm_rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


def inputs(m, hq, hk, d, p, seed, far=5000, freq=torch.float64):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = (randn(m, hq, d) * 2).to(torch.bfloat16), randn(m, hk, d).to(torch.bfloat16)
    wq, wk = ((1 + 0.3 * randn(d)).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, far + 1, (m,), generator=g, dtype=torch.int32)
    inv = (1e6 ** (-torch.arange(p, dtype=torch.float64) / max(p, 1))).to(freq)
    return [t.to(DEV) for t in (q, k, wq, wk, pos, inv)]


def check(args, out, interleaved=False, eps=EPS):
    q, k, wq, wk, pos, inv = args
    for x, w, y in ((q, wq, out[0]), (k, wk, out[1])):
        assert y.shape == x.shape and y.dtype == torch.bfloat16 and y.is_contiguous()
        m = pos.numel()
        x3 = x.reshape(m, *x.shape[-2:])
        if x3.numel() == 0:
            continue
        ref, mag = R.rope(x3, w, eps, pos.reshape(-1), inv, interleaved)
        bound = R.HALF_STEP_BF16 * np.abs(ref) * 1.001 + (x.shape[-1] / 2 + 16) * R.HALF_STEP_F32 * mag
        err = np.abs(R.f64(y).reshape(ref.shape) - ref)
        assert (err <= bound).all(), float((err - bound).max())


def run(args, interleaved=False, eps=EPS):
    q, k, wq, wk, pos, inv = args
    return qk_norm_rope(q, k, wq, wk, eps, pos, inv, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("m,hq,hk,d,p", [
    (1, 1, 1, 8, 4), (3, 24, 4, 256, 32), (5, 7, 3, 80, 40), (5, 8, 2, 80, 10), (2, 3, 1, 96, 48), (4, 5, 2, 128, 64),
    (7, 16, 16, 64, 32), (2, 64, 8, 192, 96), (3, 2, 2, 512, 256), (2, 3, 3, 40, 1), (3, 4, 2, 24, 0), (130, 33, 5, 72, 20),
    (1000, 9, 2, 128, 32), (2, 200, 50, 16, 8), (3, 10, 2, 504, 252)])
def test_matches_64_bits(m, hq, hk, d, p, interleaved):
    args = inputs(m, hq, hk, d, p, m + hq + d + p)
    check(args, run(args, interleaved), interleaved)


@pytest.mark.parametrize("far,freq", [(0, torch.float64), (1 << 20, torch.float64), (1 << 20, torch.float32),
                                      (2**31 - 1, torch.float64)])
def test_far_positions(far, freq):
    """Angles of up to 2^31 radians still turn by what inv_freq says: in fp32 they would be off by whole turns."""
    args = inputs(40, 3, 2, 64, 32, 4, far, freq)
    if far == 2**31 - 1:  # fp64 products of 2^31: 2^-22 radians off, about as much again as the rounded angle
        args[4][:4] = torch.tensor([far, -far, far - 1, -1], dtype=torch.int32, device=DEV)
    check(args, run(args))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("m,hq,hk,d,p", [(6, 5, 2, 128, 32), (6, 4, 2, 72, 18)])
def test_views_of_projections(m, hq, hk, d, p, interleaved):
    """Rows and heads read in place from a fused projection, heads followed by gates, and layouts that are copied."""
    args = inputs(m, hq, hk, d, p, 7)
    q, k = args[:2]
    want = run(args, interleaved)
    fused = torch.full((m, hq + 2 * hk, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    fused[:, :hq], fused[:, hq:hq + hk] = q, k
    gated = torch.full((m, hq, 2, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    gated[:, :, 0] = q
    odd = torch.empty(m * hq * d + 1, dtype=torch.bfloat16, device=DEV)[1:].reshape(m, hq, d)
    odd.copy_(q)
    turned = q.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    for view in (fused[:, :hq], gated[:, :, 0], odd, turned, heads_first):
        got = run([view, fused[:, hq:hq + hk], *args[2:]], interleaved)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    shared = q[:1].expand(m, hq, d)
    check([shared, *args[1:]], run([shared, *args[1:]], interleaved), interleaved)


def test_leading_shapes_and_index_types():
    q, k, wq, wk, pos, inv = args = inputs(12, 4, 2, 64, 32, 1)
    want = run(args)
    got = run([q.reshape(3, 4, 4, 64), k.reshape(3, 4, 2, 64), wq, wk, pos.reshape(3, 4).long(), inv])
    assert got[0].shape == (3, 4, 4, 64) and torch.equal(got[0].reshape(12, 4, 64), want[0])
    assert torch.equal(got[1].reshape(12, 2, 64), want[1])
    one = run([q[0], k[0], wq, wk, pos[0], inv])
    assert torch.equal(one[0], want[0][0]) and torch.equal(one[1], want[1][0])
    check([q[:0], k[:0], wq, wk, pos[:0], inv], run([q[:0], k[:0], wq, wk, pos[:0], inv]))
    no_k = run([q, k[:, :0], wq, wk, pos, inv])
    assert torch.equal(no_k[0], want[0]) and no_k[1].shape == (12, 0, 64)


def test_zero_and_nonfinite_heads():
    """A head of zeros stays zero; one with an infinity or NaN touches no other head or row."""
    args = inputs(5, 4, 2, 128, 64, 3)
    want = run(args)
    args[0][2, 1] = 0
    args[0][3, 3, 5] = float("inf")
    args[1][1, 0, 127] = float("nan")
    q, k = run(args)
    assert not q[2, 1].any() and not torch.isfinite(q[3, 3].float()).all() and not torch.isfinite(k[1, 0].float()).any()
    q[2, 1], q[3, 3], k[1, 0] = want[0][2, 1], want[0][3, 3], want[1][1, 0]
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_largest_batch_of_rows_on_a_stream():
    args = inputs(70000, 1, 1, 8, 4, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = run(args)
    stream.synchronize()
    check(args, out)


def test_captured():
    args = inputs(9, 6, 2, 256, 32, 5)
    run(args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(args)
    for i in range(4):
        for t, fresh in zip(args[:5], inputs(9, 6, 2, 256, 32, 50 + i)):
            t.copy_(fresh)
        want = run(args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
