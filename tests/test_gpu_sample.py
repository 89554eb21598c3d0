"""Sampling on the GPU (needs an MI355X), against 64 bits: tokens equal, log probabilities as fp32.

Tokens are whole numbers and have to be equal: both sides hold masses in 64 bits, so that they could differ only
where a random number lies within about V * 2^-53 of a border, which no seed here does. A log probability is one
rounding to fp32 (half a step), and 2^-40 for masses that differ by V * 2^-53 (V = 8192 covers the bound at 2^-40;
larger rows sum fewer than that many distinct values).
"""

import numpy as np
import pytest
import torch

import request_refs as R
from mlx_tree_spec_amd import sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def logits_of(m, v, seed, spread=2.0, boosted=0):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(m, v, generator=g) * spread
    if boosted:
        l.scatter_(1, torch.randint(0, v, (m, boosted), generator=g), 8 + 3 * torch.randn(m, boosted, generator=g))
    return l.to(torch.bfloat16).to(DEV), torch.rand(m, generator=g).to(DEV)


def check(logits, uniform, **settings):
    tokens, logprobs = sample(logits, uniform, **settings)
    want, want_p = R.sample(logits, uniform, **settings)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    got = tokens.cpu().numpy()
    assert np.array_equal(got, want), (got, want)
    p = R.f64(logprobs)
    same = p == want_p  # (infinities)
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(p - want_p) <= R.HALF_STEP_F32 * np.abs(want_p) * 1.01 + 2.0 ** -40)).all(), (p, want_p)
    return tokens, logprobs


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=1e-6), dict(min_p=0.05),
            dict(temperature=1.7, top_k=300, top_p=0.95, min_p=0.001), dict(temperature=0.0), dict(min_p=1.0),
            dict(temperature=30.0, top_k=10**6, top_p=0.5)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("m,v", [(1, 1), (3, 2), (5, 63), (4, 1000), (2, 4097), (3, 65537), (1, 151936)])
def test_matches_64_bits(m, v, settings):
    logits, u = logits_of(m, v, m + v, boosted=min(v, 5) if v > 1000 else 0)
    check(logits, u, **settings)


@pytest.mark.parametrize("m,v", [(64, 2000), (7, 40001), (33, 248320), (300, 513)])
def test_settings_of_each_row(m, v):
    logits, u = logits_of(m, v, v, boosted=20)
    g = torch.Generator().manual_seed(m)
    rand = lambda: torch.rand(m, generator=g)  # noqa: E731
    off = lambda t, p: torch.where(rand() < 0.3, p, t)  # noqa: E731
    settings = dict(temperature=off(rand() * 2, 0.0), top_k=off(rand() * 2000, -3.0).int(), top_p=off(rand(), 1.0),
                    min_p=off(rand() * 0.2, 0.0))
    check(logits, u, **{k: t.to(DEV) for k, t in settings.items()})


@pytest.mark.parametrize("settings", [dict(), dict(temperature=3e4), dict(temperature=1e5, top_p=0.99, min_p=1e-9),
                                      dict(temperature=1e38, top_k=9000), dict(temperature=1e38, top_p=0.7)], ids=str)
@pytest.mark.parametrize("v", [30000, 65535, 65536, 100003])
def test_more_values_than_a_page(v, settings):
    """Logits spread over many octaves: more than 4096 different values, over more than one histogram."""
    g = torch.Generator().manual_seed(v)
    l = torch.randn(6, v, generator=g) * 2.0 ** torch.randint(-60, 60, (6, v), generator=g)
    l[3:] = torch.randn(3, v, generator=g) * 2.0 ** torch.randint(-12, 9, (3, v), generator=g)  # one histogram
    logits = l.to(torch.bfloat16).to(DEV)
    logits[1, ::3] = torch.finfo(torch.bfloat16).min
    logits[4, 5::7] = -float("inf")
    check(logits, torch.tensor([0.0, 0.99, 0.5, 0.3, 0.7, 0.9], device=DEV), **settings)


def test_more_rows_than_a_batch():
    logits, u = logits_of(300, 65601, 8, boosted=9)
    g = torch.Generator().manual_seed(1)
    check(logits, u, temperature=(torch.rand(300, generator=g) * 1.5).to(DEV), top_p=0.97)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=7), dict(top_p=0.4), dict(top_k=5000, top_p=0.77, min_p=0.5)], ids=str)
def test_every_border_of_a_small_vocabulary(settings):
    """512 random numbers walk through the whole order: falling logits, equal ones by index, -0 with +0."""
    values = torch.tensor([0.0, 1.0, -0.0, 2.0, 1.0, -1.0, 0.0, 2.0, 1.5, -float("inf"), -0.0, 3e-39, 1.0])
    m = 512
    logits = values.to(torch.bfloat16).expand(m, -1).contiguous().to(DEV)
    u = ((torch.arange(m) + 0.37) / m).to(DEV)
    tokens, _ = check(logits, u, **settings)
    if not settings:
        first = {0: 0.0, 3: 2.0, 7: 2.0}
        assert tokens[0].item() == 3 and set(tokens.tolist()) >= set(first)


@pytest.mark.parametrize("v", [10, 70001])
def test_equal_logits_go_by_index(v):
    logits = torch.full((8, v), 1.25, dtype=torch.bfloat16, device=DEV)
    u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.75, 0.9, 0.999, 1 - 2.0**-24], device=DEV)
    want = torch.tensor([int(float(x) * v) for x in u.cpu().double()], device=DEV)
    assert torch.equal(sample(logits, u)[0], want)
    assert sample(logits, u, top_k=3)[0].max().item() == 2
    assert torch.equal(sample(logits, u, temperature=0.0)[0], torch.zeros(8, dtype=torch.int64, device=DEV))


def test_masks_infinities_and_nan():
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.bfloat16).min
    v = 3000
    logits, u = logits_of(10, v, 5)
    logits[0] = -inf                       # nothing left
    logits[1] = nan
    logits[2, :] = -inf
    logits[2, 2999] = -50.0                # one left
    logits[3, :] = low                     # masked by the lowest value, a few left
    logits[3, 100:105] = 1.0
    logits[4, :] = low                     # all at the lowest value: equal
    logits[5, 7] = nan                     # NaN among others
    logits[6, [5, 2000]] = inf             # two infinities share everything
    logits[7, ::2] = -inf
    logits[8, :] = -inf
    logits[8, [3, 9]] = torch.tensor([low, -low], dtype=torch.bfloat16, device=DEV)
    for settings in (dict(), dict(temperature=0.0), dict(top_k=4, top_p=0.9, min_p=0.1), dict(temperature=1e-30)):
        tokens, logprobs = check(logits, u, **settings)
        assert tokens[:2].tolist() == [-1, -1] and (logprobs[:2] == -inf).all() and tokens[2].item() == 2999


def test_settings_at_and_past_their_ends():
    """Rows' settings are not seen by the host: those out of range mean what the documentation says."""
    inf, nan = float("inf"), float("nan")
    logits, _ = logits_of(1, 500, 2)
    logits = logits.expand(12, -1).contiguous()
    f = lambda *x: torch.tensor(x, dtype=torch.float32, device=DEV)  # noqa: E731
    u = f(0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.0, 1.0, -1.0, nan)
    tokens, _ = sample(logits, u, temperature=f(nan, -1, inf, 1, 1, 1, 1, 1, 1, 1, 1, 1),
                       top_p=f(1, 1, 1, nan, 0, -1, 1, 1, 1, 1, 1, 1), min_p=f(0, 0, 0, 0, 0, 0, nan, 2, 0, 0, 0, 0),
                       top_k=torch.tensor([0, 0, 0, -1, 0, 0, 0, 0, 0, 0, 0, 0], dtype=torch.int32, device=DEV))
    row = R.f64(logits)[0]
    order = np.argsort(-row, kind="stable")
    median = R.sample_row(row, 0.5)[0]
    want = [order[0], order[0], order[250], median, order[0], order[0], median, order[0], order[0], order[-1], order[0], order[0]]
    assert tokens.tolist() == [int(t) for t in want]


def test_views_and_leading_shapes():
    logits, u = logits_of(6, 1001, 4)
    want, want_p = sample(logits, u, top_p=0.9)
    wide = torch.full((6, 1100), 100.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:1004] = logits                       # rows that start at odd places, larger values around them
    every = torch.full((6, 2002), 100.0, dtype=torch.bfloat16, device=DEV)
    every[:, ::2] = logits
    for view in (wide[:, 3:1004], every[:, ::2], logits.t().contiguous().t(), logits.reshape(2, 3, 1001)):
        got, got_p = sample(view, u.reshape(view.shape[:-1]), top_p=torch.full(view.shape[:-1], 0.9, device=DEV))
        assert got.shape == view.shape[:-1] and torch.equal(got.reshape(-1), want) and torch.equal(got_p.reshape(-1), want_p)
    one, one_p = sample(logits[2], u[2], top_p=0.9)
    assert one.shape == () and one.item() == want[2].item() and one_p.item() == want_p[2].item()
    none, none_p = sample(logits[:0], u[:0])
    assert none.shape == (0,) and none_p.shape == (0,)
    same = logits[:1].expand(6, -1)
    check(same, u)


def test_deterministic_on_a_stream_and_captured():
    logits, u = logits_of(20, 50000, 6, boosted=10)
    settings = dict(temperature=0.9, top_k=200, top_p=0.99)
    want = sample(logits, u, **settings)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = sample(logits, u, **settings)
    stream.synchronize()
    assert torch.equal(want[0], other[0]) and torch.equal(want[1], other[1])
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sample(logits, u, **settings))
        graphs.append(g)
    for i in range(4):
        fresh, fresh_u = logits_of(20, 50000, 60 + i, boosted=10)
        logits.copy_(fresh)
        u.copy_(fresh_u)
        want = sample(logits, u, **settings)
        torch.cuda.synchronize()
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("count", [65535, 65536, 70000])
@pytest.mark.parametrize("settings", [dict(), dict(temperature=3e38), dict(temperature=1e38, top_k=30000, top_p=0.9, min_p=0.1)],
                         ids=str)
def test_every_bit_pattern(count, settings):
    """All bf16 words, NaN of either sign among them, in any order; rows with +infinity, without, and of NaN alone."""
    g = torch.Generator().manual_seed(count)
    words = torch.stack([torch.randperm(count, generator=g) % 65536 for _ in range(4)])
    words[1:][words[1:] == 0x7F80] = 0xFF80
    words[3] = torch.where((words[3] & 0x7F80) == 0x7F80, words[3], 0xFFFF)
    words[2, ::2] |= 0x7F80
    words[2][words[2] == 0x7F80] = 0x7FFF
    logits = torch.where(words >= 32768, words - 65536, words).to(torch.int16).view(torch.bfloat16).to(DEV)
    check(logits, torch.tensor([0.25, 0.5, 0.75, 0.125], device=DEV), **settings)
