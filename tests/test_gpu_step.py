"""A batched step over several requests' rows, through the operators that differ per request beside the shared
projections (needs an MI355X): attention inputs with adapters, head norms and rotation, the MLP half, and sampling from
the vocabulary head. Each stage is checked against 64 bits on what it was given, with the bounds of its own tests, and
the whole step captured into a graph against the eager one."""

import numpy as np
import pytest
import torch

import request_refs as R
from mlx_tree_spec_amd import (AttentionInputs, LoRALinear, MLPLayer, QuantizedLinear, QuantizedMLP, add_rms_norm,
                               attention_inputs, install, layer_tail, next_tokens, sample, stack_adapters)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DIM, HEADS, KV, D, VOCAB, MLP = 512, 6, 2, 64, 4112, 1024


def linear(k, n, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-2**31, 2**31, (n, k // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = ((torch.randn(n, k // 64, generator=g).abs() * 0.004 + 1e-4)).to(torch.bfloat16)
    b = (-8 * s.float() + torch.randn(n, k // 64, generator=g) * 1e-3).to(torch.bfloat16)
    return QuantizedLinear.from_quantized(w.to(DEV), s.to(DEV), b.to(DEV))


def adapted(k, n, seed):
    g = torch.Generator().manual_seed(seed + 100)
    tables = stack_adapters([(torch.randn(r, k, generator=g) / k ** 0.5, torch.randn(n, r, generator=g) * 0.2, 1.0 + r / 8)
                             for r in (8, 4, 16)], device=DEV)
    return LoRALinear(linear(k, n, seed), *tables)


def norm(dim, seed):
    m = torch.nn.RMSNorm(dim, eps=1e-6, device=DEV, dtype=torch.bfloat16).requires_grad_(False)
    m.weight.copy_(1 + 0.1 * torch.randn(dim, generator=torch.Generator().manual_seed(seed)))
    return m


class Model:
    def __init__(self):
        inv = 1e4 ** (-torch.arange(16, dtype=torch.float64, device=DEV) / 16)
        self.attn = [AttentionInputs(adapted(DIM, HEADS * 2 * D, 10 * i), adapted(DIM, KV * D, 10 * i + 1),
                                     linear(DIM, KV * D, 10 * i + 2), norm(D, i), norm(D, i + 9), HEADS, KV, D, inv,
                                     gated=True) for i in range(2)]
        self.out = [linear(HEADS * D, DIM, 10 * i + 3) for i in range(2)]
        self.mlp = [MLPLayer(norm(DIM, 20 + i), QuantizedMLP(linear(DIM, MLP, 30 + i), linear(DIM, MLP, 40 + i),
                                                             linear(MLP, DIM, 50 + i))) for i in range(2)]
        self.norms = [norm(DIM, 60), norm(DIM, 61), norm(DIM, 62)]
        self.head = linear(DIM, VOCAB, 70)
        install(torch.nn.ModuleList([*self.out, *self.mlp, self.head]), verbose=False)

    def step(self, h, positions, adapters, uniform, settings, seen=None):
        h, x = add_rms_norm(h, torch.zeros_like(h), self.norms[0])
        for i in range(2):
            q, k, v, gate = attention_inputs(x, self.attn[i], positions, adapters)
            if seen is not None:
                seen.append((x, q, k, v, gate))
            # (attention itself is not this package's: each head here takes its own value head)
            a = (q + k.repeat_interleave(HEADS // KV, 1) + v.repeat_interleave(HEADS // KV, 1)) * torch.sigmoid(gate)
            h, x = layer_tail(h, self.out[i](a.reshape(len(x), -1)), self.mlp[i], self.norms[i + 1])
        return x, *next_tokens(x, self.head, uniform, **settings)


def batch(m, seed):
    g = torch.Generator().manual_seed(seed)
    request = torch.arange(m) * 4 // m  # four requests; the last has no adapter
    rand = lambda lo, hi: lo + (hi - lo) * torch.rand(4, generator=g)[request]  # noqa: E731
    settings = dict(temperature=torch.where(request == 1, torch.zeros(m), rand(0.5, 1.5)), top_k=(rand(1, 200)).int(),
                    top_p=rand(0.5, 1.0), min_p=rand(0.0, 0.05))
    return (torch.randn(m, DIM, generator=g).to(torch.bfloat16).to(DEV),
            (torch.randint(0, 100000, (4,), generator=g)[request] + torch.arange(m)).to(torch.int32).to(DEV),
            torch.where(request == 3, -1, (request + 1) % 3).to(torch.int32).to(DEV), torch.rand(m, generator=g).to(DEV),
            {k: t.to(DEV) for k, t in settings.items()})


@pytest.mark.parametrize("m", [4, 23, 64, 130])
def test_step_stage_by_stage(m):
    model = Model()
    h, positions, adapters, uniform, settings = batch(m, m)
    seen = []
    x, tokens, logprobs = model.step(h, positions, adapters, uniform, settings, seen)
    for (xin, q, k, v, gate), layer in zip(seen, model.attn):
        raw = {}
        for name, proj in (("q", layer.q_proj), ("k", layer.k_proj)):
            base = proj.base
            wd = R.dequantize(base.weight, base.scales, base.biases, 64, 4)
            ref, _, mag = R.lora(xin, wd, proj.lora_a, proj.lora_b, proj.lora_scale, adapters)
            y = proj(xin, adapters)
            bound = R.HALF_STEP_BF16 * np.abs(ref) * 1.01 + ((DIM + 20) * R.HALF_STEP_F32 + 2.0 ** -18) * mag
            assert (np.abs(R.f64(y) - ref) <= bound).all()
            raw[name] = y
        q_raw = raw["q"].reshape(m, HEADS, 2 * D)
        assert torch.equal(gate, q_raw[..., D:]) and torch.equal(v, layer.v_proj(xin).reshape(m, KV, D))
        for y, x_raw, w in ((q, q_raw[..., :D], layer.q_norm.weight), (k, raw["k"].reshape(m, KV, D), layer.k_norm.weight)):
            ref, mag = R.rope(x_raw, w, 1e-6, positions, layer.inv_freq, False)
            bound = R.HALF_STEP_BF16 * np.abs(ref) * 1.001 + (D / 2 + 16) * R.HALF_STEP_F32 * mag
            assert (np.abs(R.f64(y) - ref) <= bound).all()
    logits = model.head(x)
    want, want_p = R.sample(logits, uniform, **settings)
    assert np.array_equal(tokens.cpu().numpy(), want)
    assert (np.abs(R.f64(logprobs) - want_p) <= R.HALF_STEP_F32 * np.abs(want_p) * 1.01 + 2.0 ** -40).all()
    again = sample(logits, uniform, **settings)
    assert torch.equal(again[0], tokens) and torch.equal(again[1], logprobs)


@pytest.mark.parametrize("m", [3, 40, 130])
def test_step_captured(m):
    model = Model()
    h, positions, adapters, uniform, settings = batch(m, 7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        model.step(h, positions, adapters, uniform, settings)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = model.step(h, positions, adapters, uniform, settings)
    for i in range(4):
        fresh = batch(m, 100 + i)
        for t, new in zip((h, positions, adapters, uniform), fresh):
            t.copy_(new)
        for name, t in settings.items():
            t.copy_(fresh[4][name])
        want = model.step(h, positions, adapters, uniform, settings)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_layers_that_do_not_match_are_refused():
    inv = torch.ones(16, device=DEV)
    a, b = norm(D, 1), torch.nn.RMSNorm(D, eps=1e-5, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="eps"):
        AttentionInputs(None, None, None, a, b, 2, 1, D, inv)
