"""The paged cache's operators together, as a server runs them (needs an MI355X): prompts, decode steps and trees of several
requests through two layers' caches, accepted nodes put in a line, requests that leave. Every attention is checked against 64
bits on the keys and values that the layers gave for the tokens its rows see (bf16 caches; with 8 bits, on what the cache
holds for them), with the bound of the attention's own tests."""

import random

import numpy as np
import pytest
import torch

import cache_refs as R
from cache_refs import i32
from mlx_tree_spec_amd import AttentionInputs, CacheTables, QuantizedLinear, attention_inputs, cached_attention, store_kv_
from request_refs import f64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DIM, HEADS, KV, D, PAGE = 256, 6, 2, 64, 16


def linear(k, n, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-2**31, 2**31, (n, k // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = (torch.randn(n, k // 64, generator=g).abs() * 0.02 + 1e-4).to(torch.bfloat16)
    b = (-8 * s.float()).to(torch.bfloat16)
    return QuantizedLinear.from_quantized(w.to(DEV), s.to(DEV), b.to(DEV))


def norm(seed):
    m = torch.nn.RMSNorm(D, eps=1e-6, device=DEV, dtype=torch.bfloat16).requires_grad_(False)
    m.weight.copy_(1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(seed)))
    return m


def make_layer(seed, gated):
    inv = 1e4 ** (-torch.arange(16, dtype=torch.float64, device=DEV) / 16)
    return AttentionInputs(linear(DIM, HEADS * D * (2 if gated else 1), seed), linear(DIM, KV * D, seed + 1), linear(DIM, KV * D, seed + 2),
                           norm(seed), norm(seed + 1), HEADS, KV, D, inv, gated=gated)


class Server:
    def __init__(self, requests, bits):
        self.tables = CacheTables(requests, 12, 12 * requests, PAGE, HEADS, KV, D, DEV)
        self.layers = [make_layer(10 * i, gated=i == 1) for i in range(2)]
        self.caches = [self.tables.cache(bits) for _ in self.layers]
        self.bits = bits
        # The keys and values of each request's tokens, by layer, in 64 bits.
        self.held = [[(np.zeros((0, KV, D)), np.zeros((0, KV, D))) for _ in range(requests)] for _ in self.layers]

    def lengths(self):
        return self.tables.lengths.tolist()

    def stored(self, i, r, length):
        if self.bits == 16:
            k, v = self.held[i][r]
            return k[:length], v[:length]
        k, v = R.token_rows(self.caches[i])
        t = np.arange(length)
        at = self.tables.block_table.cpu().numpy()[r, t // PAGE].astype(np.int64) * PAGE + t % PAGE
        return k[at], v[at]

    def run(self, rows, pad=0, positions=None, ancestors=None):
        """One step of all layers; (step, [(k, v)]) and the checks."""
        before, m = self.lengths(), sum(rows) + pad
        step = self.tables.step(i32(rows), m)
        assert self.lengths() == [b + n for b, n in zip(before, rows)]
        out = []
        for i, (layer, cache) in enumerate(zip(self.layers, self.caches)):
            x = torch.randn(m, DIM, generator=torch.Generator().manual_seed(m + i + sum(before))).to(torch.bfloat16).to(DEV)
            a, k, v = cached_attention(x, layer, cache, step, positions=positions, ancestors=ancestors)
            q, k2, v2, gate = attention_inputs(x, layer, step.positions if positions is None else positions)
            assert torch.equal(k, k2) and torch.equal(v, v2) and a.shape == (m, HEADS * D)
            out.append((k, v))
            row = 0
            for r, n in enumerate(rows):
                if n == 0:
                    continue
                old = self.held[i][r]
                self.held[i][r] = tuple(np.concatenate((o[:before[r]], f64(t[row:row + n]))) for o, t in zip(old, (k, v)))
                keys, values = self.stored(i, r, before[r] + n)
                sees = R.visible(before[r], n, None if ancestors is None else ancestors[row:row + n].tolist())
                want, mag, delta = R.attention(f64(q[row:row + n]), keys, values, D ** -0.5, sees)
                if gate is not None:
                    s = 1 / (1 + np.exp(-f64(gate[row:row + n])))
                    want, mag = want * s, mag * s
                err = np.abs(f64(a[row:row + n]).reshape(want.shape) - want)
                assert (err <= R.attention_bound(want, mag, delta, before[r] + n)).all()
                row += n
            assert not a[row:].any()
        return step, out

    def accept(self, before, rows, kvs, chosen):
        """The chosen nodes of each request's tree put in a line behind `before`."""
        keep = torch.zeros(sum(rows), dtype=torch.bool, device=DEV)
        first = np.cumsum([0, *rows])
        for r, nodes in enumerate(chosen):
            keep[[int(first[r]) + n for n in nodes]] = True
        step = self.tables.step(i32(rows), sum(rows), base=i32(before), keep=keep)
        for i, ((k, v), cache) in enumerate(zip(kvs, self.caches)):
            store_kv_(k, v, cache, step.slots)
            for r, nodes in enumerate(chosen):
                at = [int(first[r]) + n for n in nodes]
                self.held[i][r] = tuple(np.concatenate((o[:before[r]], f64(t)[at])) for o, t in zip(self.held[i][r], (k, v)))
        assert self.lengths() == [b + len(nodes) for b, nodes in zip(before, chosen)]


@pytest.mark.parametrize("bits", [16, 8])
def test_server(bits):
    rng = random.Random(bits)
    server = Server(4, bits)
    server.run([20, 0, 33, 1])                      # prompts
    server.run([1, 5, 1, 1], pad=2)                 # decode beside a prompt, a padded batch
    for _ in range(3):
        before, rows = server.lengths(), [rng.randrange(1, 9) for _ in range(4)]
        depth, masks, parents = [], [], []
        for n in rows:
            tree = []
            for j in range(n):
                tree.append(rng.randrange(j) if j else -1)
            parents.append(tree)
            d, m = [], []
            for j, p in enumerate(tree):
                d.append(d[p] + 1 if j else 0)
                m.append((m[p] if j else 0) | 1 << j)
            depth += d
            masks += m
        at = [b for b, n in zip(before, rows) for _ in range(n)]
        _, kvs = server.run(rows, positions=i32([a + d for a, d in zip(at, depth)]),
                            ancestors=torch.tensor(masks, dtype=torch.int64, device=DEV))
        chosen = []
        for tree in parents:  # a path from the root
            path, node = [], 0
            while node is not None:
                path.append(node)
                below = [j for j, p in enumerate(tree) if p == node]
                node = rng.choice(below) if below and rng.random() < 0.8 else None
            chosen.append(path)
        server.accept(before, rows, kvs, chosen)
        server.run([1, 1, 0, 1])
    lengths = server.lengths()
    lengths[1] = 0
    server.tables.step(i32([0] * 4), 0, base=i32(lengths))  # a request leaves, another takes its place
    for held in server.held:
        held[1] = (np.zeros((0, KV, D)),) * 2
    server.run([1, 40, 1, 0], pad=1)
    server.tables.step(i32([0] * 4), 0, base=i32([0] * 4))
    assert server.tables.free_count.item() == 48 and (server.tables.block_table == -1).all()


def test_refusals():
    server = Server(1, 16)
    step = server.tables.step(i32([2]), 2)
    x = torch.zeros(2, DIM, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="x must be"):
        cached_attention(x[None], server.layers[0], server.caches[0], step)
    with pytest.raises(ValueError, match="the step was made for"):
        cached_attention(x, server.layers[0], server.caches[0], step._replace(heads=4))


def test_captured_server_step():
    """A decode step of tables, layers and attention captured once and replayed while requests grow, against an eager server."""
    servers = [Server(3, 16) for _ in range(2)]
    xs = [torch.zeros(4, DIM, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    rows = i32([0, 0, 0])

    def decode(server):
        step = server.tables.step(rows, 4, max_rows=2)
        return [cached_attention(x, layer, cache, step)[0] for x, layer, cache in zip(xs, server.layers, server.caches)]

    for server in servers:
        for cache in server.caches:
            for t in cache[:2]:
                t.zero_()
        decode(server)
    stream = torch.cuda.Stream()  # (the projections' workspaces are a stream's: their first calls are made on the one captured)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        decode(servers[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = decode(servers[0])
    rng = random.Random(5)
    for i in range(20):
        rows.copy_(i32([rng.randrange(3), rng.randrange(2), 1]))
        for x in xs:
            x.copy_(torch.randn(4, DIM, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        want = decode(servers[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert servers[0].lengths() == servers[1].lengths()
