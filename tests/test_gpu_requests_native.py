"""The native form of the per-request operators' calls against their Python form: the same bits for every form of the
arguments that it takes, and None (the Python form runs, or raises) for every other (needs an MI355X)."""

import pytest
import torch

from mlx_tree_spec_amd import _lib, qk_norm_rope, quantized_matmul_lora, sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Declines:
    def __getattr__(self, name):
        return lambda *args: None


def tensors(out):
    return out if isinstance(out, tuple) else (out,)


def both(monkeypatch, call, native=True):
    """The call's result, the same without native code; `native`: whether native code is expected to take it."""
    taken = []
    real = _lib.native()

    class Watch:
        def __getattr__(self, name):
            def f(*args):
                out = getattr(real, name)(*args)
                taken.append(out is not None)
                return out
            return f

    with monkeypatch.context() as m:
        m.setattr(_lib, "native", lambda: Watch())
        got = tensors(call())
    assert taken[0] == native
    with monkeypatch.context() as m:
        m.setattr(_lib, "native", lambda: _Declines())
        want = tensors(call())
    for a, b in zip(got, want):
        assert a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous() and torch.equal(a, b)


def rand(*shape, seed=1, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def lora_args(lead, k=256, n=96, rank=16, count=3, bits=4, group=64):
    g = torch.Generator().manual_seed(5)
    w = torch.randint(-2**31, 2**31, (n, k * bits // 32), generator=g, dtype=torch.int64).to(torch.int32).to(DEV)
    ids = torch.randint(-1, count, lead, generator=g).to(torch.int32).to(DEV)
    return [rand(*lead, k), w, rand(n, k // group) * 0.01, rand(n, k // group, seed=2) * 0.01, rand(count, rank, k, seed=3),
            rand(count, n, rank, seed=4), rand(count, dtype=torch.float32), ids]


@pytest.mark.parametrize("lead", [(1,), (5,), (2, 3), (70,)])
def test_lora(monkeypatch, lead):
    a = lora_args(lead)
    both(monkeypatch, lambda: quantized_matmul_lora(*a))
    both(monkeypatch, lambda: quantized_matmul_lora(*a[:7], a[7].long()))
    both(monkeypatch, lambda: quantized_matmul_lora(a[0], a[1].view(torch.uint32), *a[2:]))
    general = lora_args(lead, n=33, bits=8, group=32)
    both(monkeypatch, lambda: quantized_matmul_lora(*general, bits=8, group_size=32))
    a[0] = torch.empty(*lead, 512, dtype=torch.bfloat16, device=DEV)[..., ::2].copy_(a[0])  # strided: the Python form
    both(monkeypatch, lambda: quantized_matmul_lora(*a), native=False)


def test_lora_declines_what_is_wrong():
    a = lora_args((4,))
    for i, bad in ((0, a[0].float()), (4, a[4][:, :, :128]), (5, a[5][:2]), (6, a[6][:2]), (7, a[7][:3]), (7, a[7].float()),
                   (2, a[2].float())):
        args = list(a)
        args[i] = bad
        with pytest.raises(ValueError):
            quantized_matmul_lora(*args)
    with pytest.raises(ValueError, match="gradient"):
        quantized_matmul_lora(a[0].clone().requires_grad_(True), *a[1:])


@pytest.mark.parametrize("lead", [(1,), (6,), (2, 3), (1, 1, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(monkeypatch, lead, interleaved):
    fused = rand(*lead, 9, 64)
    q, k, wq, wk = fused[..., :5, :], fused[..., 5:7, :], rand(64), rand(64, seed=2)
    pos = torch.arange(torch.Size(lead).numel(), device=DEV).reshape(lead) * 1000
    inv = 1e4 ** (-torch.arange(16, dtype=torch.float64, device=DEV) / 16)
    call = lambda *a: lambda: qk_norm_rope(*a, interleaved=interleaved)  # noqa: E731
    both(monkeypatch, call(q, k, wq, wk, 1e-6, pos, inv))
    both(monkeypatch, call(q, k, wq, torch.nn.Parameter(wk), 1e-5, pos.int(), inv.float()))
    both(monkeypatch, call(q.contiguous(), k.contiguous(), wq, wk, 0, pos, inv))
    both(monkeypatch, call(q, k, wq, wk, 1e-6, pos, inv[:0]), native=False)      # empty frequencies
    both(monkeypatch, call(fused[..., 4:9, ::2], fused[..., :1, ::2], wq[:32], wk[:32], 1e-6, pos, inv), native=False)
    both(monkeypatch, call(q[..., 4:36], k[..., 4:36], wq[:32], wk[:32], 1e-6, pos, inv), native=False)  # 8 bytes off


def test_rope_declines_what_is_wrong():
    q, k, w = rand(4, 3, 64), rand(4, 2, 64), rand(64)
    pos, inv = torch.arange(4, device=DEV), torch.ones(32, device=DEV)
    for args in ((q.float(), k, w, w, 1e-6, pos, inv), (q, k[:3], w, w, 1e-6, pos, inv), (q, k, w[:32], w, 1e-6, pos, inv),
                 (q, k, w, w, 1e-6, pos[:2], inv), (q, k, w, w, 1e-6, pos.float(), inv), (q, k, w, w, 1e-6, pos, inv.half()),
                 (q, k, w, w, -1.0, pos, inv), (q, k, w, w, float("nan"), pos, inv),
                 (q, k, w, w, 1e-6, pos, torch.ones(33, device=DEV))):
        with pytest.raises(ValueError):
            qk_norm_rope(*args)
    with pytest.raises(ValueError, match="gradient"):
        qk_norm_rope(q.clone().requires_grad_(True), k, w, w, 1e-6, pos, inv)


@pytest.mark.parametrize("v", [777, 70000])
@pytest.mark.parametrize("lead", [(), (1,), (5,), (2, 3)])
def test_sample(monkeypatch, lead, v):
    logits = rand(*lead, v) * 3
    u = torch.rand(lead, generator=torch.Generator().manual_seed(3)).to(DEV)
    full = lambda x, dtype=torch.float32: torch.full(lead, x, dtype=dtype, device=DEV)  # noqa: E731
    both(monkeypatch, lambda: sample(logits, u))
    both(monkeypatch, lambda: sample(logits, u, 0.7, 40, 0.9, 0.01))
    both(monkeypatch, lambda: sample(logits, u, full(0.7), full(40, torch.int32), full(0.9), full(0.01)))
    both(monkeypatch, lambda: sample(logits, u, 1, 0, 1, 0))
    if lead == (5,):
        wide = torch.zeros(5, v + 9, dtype=torch.bfloat16, device=DEV)
        wide[:, 3:v + 3] = logits
        both(monkeypatch, lambda: sample(wide[:, 3:v + 3], u, top_p=0.8))
        both(monkeypatch, lambda: sample(logits.t().contiguous().t(), u), native=False)


def test_sample_declines_what_is_wrong():
    logits, u = rand(4, 100), torch.rand(4, device=DEV)
    for kw in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=0.0), dict(min_p=2.0), dict(temperature=u[:3]),
               dict(top_k=torch.zeros(4, device=DEV)), dict(top_p=u.cpu())):
        with pytest.raises(ValueError):
            sample(logits, u, **kw)
    with pytest.raises(ValueError):
        sample(logits.float(), u)
    with pytest.raises(ValueError, match="gradient"):
        sample(logits.clone().requires_grad_(True), u)
