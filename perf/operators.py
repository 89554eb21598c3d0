"""What the per-request operators of a batched step are timed on, with their plain forms.

A step concatenates several requests' rows and runs each quantized projection once over all of them.
Three operators differ from request to request:

  lora    quantized_matmul_lora: a shared quantized projection with each request's low-rank adapter
          y[m] = W x[m] + scale[a] B[a] (A[a] x[m]), a = adapters[m] (below 0: none), W = bf16(s q + b)
  rope    qk_norm_rope: the norms of the query and key heads and the rotation at each row's position
  sample  sample: the next token of each row, and its log probability, from the vocabulary head's logits and
          a random number, with the request's temperature, top-k, top-p and min-p

Sizes are those of the target model of tests and benchmark (hidden 5120, MLP 17408, fused gate+up 34816,
vocabulary 151936, drafter vocabulary 65984, 24 query heads of 256 that come with their gates beside 4 key
heads) and generic ones, at the rows of decode (1-4), tree verify (5-64), prompt tails and prefill.
"""

import math
import os
import sys

import numpy as np
import torch

own = False
EPS = 1e-6

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _lora(name, m, k, n, rank, requests, loaded, bare=0, bits=4, group=64):
    """`requests` runs of rows, one adapter each out of `loaded` (the last `bare` requests have none)."""
    return {"name": name, "op": "lora", "m": m, "k": k, "n": n, "rank": rank, "requests": requests,
            "loaded": loaded, "bare": bare, "bits": bits, "group": group}


def _rope(name, m, q_heads, k_heads, dim, rotary, layout, requests, far, interleaved=False):
    """layout: "plain" (q and k of their own), "qkv" (views of one fused projection), "gated" (each query
    head followed by its gate); far: the largest position."""
    return {"name": name, "op": "rope", "m": m, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "rotary": rotary, "layout": layout, "requests": requests, "far": far, "interleaved": interleaved}


def _sample(name, m, vocab, params, logits):
    """params: "plain" (temperature alone), "shared" (one setting for all rows), "mixed" (each row its own);
    logits: "peaked" (a model sure of itself), "flat", "masked" (most tokens forbidden)."""
    return {"name": name, "op": "sample", "m": m, "vocab": vocab, "params": params, "logits": logits}


def listed():
    return [
        # Decode, 4 requests with adapters of their own: the fused gate+up projection.
        _lora("lora decode 4x5120-34816 r16", 4, 5120, 34816, 16, 4, 8),
        # One request's tree verify: an attention-sized square projection, where latency counts.
        _lora("lora verify 16x5120-5120 r16", 16, 5120, 5120, 16, 1, 4),
        # Batched tree verify, 4 requests, one of them without an adapter: the down projection.
        _lora("lora verify 64x17408-5120 r32", 64, 17408, 5120, 32, 4, 8, bare=1),
        # Three prompts prefilled together: the up projection with a large rank.
        _lora("lora prompt 2000x5120-17408 r64", 2000, 5120, 17408, 64, 3, 4),
        # A layer that the packed kernels do not take (8-bit codes, ragged columns), many small requests.
        _lora("lora 8-bit 24x2560-4100 r8", 24, 2560, 4100, 8, 20, 32, bare=2, bits=8, group=32),
        # Decode, 3 requests at far positions: the smallest call.
        _rope("rope decode 3x(24+4)x256", 3, 24, 4, 256, 64, "gated", 3, 200000),
        # Batched tree verify: 4 requests of 16 nodes.
        _rope("rope verify 64x(32+8)x128", 64, 32, 8, 128, 128, "qkv", 4, 30000),
        # Chunked prefill.
        _rope("rope prefill 4096x(32+8)x128", 4096, 32, 8, 128, 128, "qkv", 2, 60000),
        # One request, temperature alone.
        _sample("sample 1x151936", 1, 151936, "plain", "peaked"),
        # A verify batch of the vocabulary head, every request with settings of its own.
        _sample("sample 32x151936 mixed", 32, 151936, "mixed", "peaked"),
        # A drafter's vocabulary with a flat distribution and one setting for all.
        _sample("sample 16x65984 flat", 16, 65984, "shared", "flat"),
        # A large batch whose grammar forbids most tokens.
        _sample("sample 200x32001 masked", 200, 32001, "mixed", "masked"),
    ]


LARGEST_MNK = 2000 * 5120 * 17408
LARGEST_ROPE = 4096 * 40 * 128
LARGEST_LOGITS = 200 * 32001


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _draw_lora(rng):
    lo, hi = rng.choice([(1, 4), (5, 16), (17, 64), (65, 2000)])
    m = round(_log_uniform(rng, lo, hi))
    bits, group = (4, 64) if rng.random() < 0.8 else rng.choice([(2, 64), (4, 32), (4, 128), (8, 32), (8, 64)])
    k = 128 * round(_log_uniform(rng, 1024, 17408) / 128)
    if bits == 4 and group == 64:
        n = 32 * round(_log_uniform(rng, 512, 34816) / 32)
    else:
        m, k, n = min(m, 64), min(k, 8192), round(_log_uniform(rng, 512, 8192)) | 1
    m = max(1, min(m, LARGEST_MNK // (n * k)))
    requests = min(m, round(_log_uniform(rng, 1, 16)))
    return _lora("", m, k, n, 8 * round(_log_uniform(rng, 8, 128) / 8), requests, round(_log_uniform(rng, 1, 32)),
                 rng.randint(0, requests) if rng.random() < 0.3 else 0, bits, group)


def _draw_rope(rng):
    q_heads, k_heads = rng.choice([(24, 4), (32, 8), (16, 16), (28, 4), (40, 8), (64, 8), (8, 1), (7, 3)])
    dim = rng.choice([64, 80, 96, 128, 192, 256])
    rotary = rng.choice([dim, dim, dim // 2, dim // 4])
    m = round(_log_uniform(rng, 1, min(8192, LARGEST_ROPE // ((q_heads + k_heads) * dim))))
    return _rope("", m, q_heads, k_heads, dim, rotary, rng.choice(["plain", "qkv", "gated"]), min(m, rng.randint(1, 8)),
                 round(_log_uniform(rng, 100, 1000000)), rng.random() < 0.3)


def _draw_sample(rng):
    vocab = round(_log_uniform(rng, 1000, 151936))
    m = round(_log_uniform(rng, 1, min(200, LARGEST_LOGITS // vocab)))
    return _sample("", m, vocab, rng.choice(["plain", "shared", "mixed"]), rng.choice(["peaked", "flat", "masked"]))


def draw(rng):
    case = rng.choice([_draw_lora, _draw_rope, _draw_sample])(rng)
    del case["name"]
    return case


# Inputs: activations after a norm are about N(0, 1) (0.5 in front of a down projection); codes are uniform, with
# scales and biases as affine quantization of trained weights gives them; adapters like trained ones, whose
# product is about a tenth of the projection. Logits: a model's tail is about normal, a sure one has a few
# tokens far above it; a grammar leaves some hundred tokens.

def _runs(gen, m, requests):
    """The request of each row: `requests` runs of at least one row, ragged."""
    cuts = torch.randperm(m - 1, generator=gen, device="cuda")[:requests - 1] + 1
    start = torch.zeros(m, dtype=torch.int64, device="cuda")
    start[cuts] = 1
    return torch.cumsum(start, 0)


def _lora_inputs(case, gen):
    m, k, n, rank, loaded, bits, group = (case[f] for f in ("m", "k", "n", "rank", "loaded", "bits", "group"))
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    x = (randn(m, k) * (0.5 if k > 6144 else 1.0)).to(torch.bfloat16)
    w = torch.randint(-2**31, 2**31, (n, k * bits // 32), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    s = ((randn(n, k // group).abs() * 0.004 + 1e-4) * 2.0 ** (4 - bits)).to(torch.bfloat16)
    b = (-(2.0 ** (bits - 1)) * s.float() + randn(n, k // group) * 1e-3).to(torch.bfloat16)
    lora_a = (randn(loaded, case["rank"], k) / math.sqrt(k)).to(torch.bfloat16)
    lora_b = (randn(loaded, n, rank) * (0.2 / math.sqrt(rank))).to(torch.bfloat16)
    lora_scale = torch.rand(loaded, generator=gen, device="cuda") * 1.5 + 0.5
    request = _runs(gen, m, case["requests"])
    chosen = torch.randperm(loaded, generator=gen, device="cuda")[request % loaded]
    adapters = torch.where(request < case["requests"] - case["bare"], chosen, -1).to(torch.int32)
    return {"x": x, "w": w, "s": s, "b": b, "lora_a": lora_a, "lora_b": lora_b, "lora_scale": lora_scale,
            "adapters": adapters}


def _rope_inputs(case, gen):
    m, hq, hk, d = case["m"], case["q_heads"], case["k_heads"], case["dim"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    # A projection's heads differ in size.
    if case["layout"] == "qkv":
        qkv = (randn(m, hq + 2 * hk, d) * (0.5 + 2 * torch.rand(hq + 2 * hk, 1, generator=gen, device="cuda"))).to(torch.bfloat16)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    else:
        q = (randn(m, hq, 2 * d if case["layout"] == "gated" else d) * 1.5).to(torch.bfloat16)[..., :d]
        k = (randn(m, hk, d) * 2.0).to(torch.bfloat16)
    wq, wk = ((1.0 + 0.2 * randn(d)).to(torch.bfloat16) for _ in range(2))
    request = _runs(gen, m, case["requests"])
    base = torch.randint(0, case["far"] + 1, (case["requests"],), generator=gen, device="cuda")
    first = torch.searchsorted(request, torch.arange(case["requests"], device="cuda"))
    positions = (base[request] + torch.arange(m, device="cuda") - first[request]).to(torch.int32)
    half = case["rotary"] // 2
    inv_freq = 1.0e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    return {"q": q, "k": k, "wq": wq, "wk": wk, "positions": positions, "inv_freq": inv_freq,
            "interleaved": case["interleaved"]}


def _sample_inputs(case, gen):
    m, vocab = case["m"], case["vocab"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    logits = randn(m, vocab) * (2.0 if case["logits"] != "flat" else 0.5)
    if case["logits"] == "peaked":
        top = torch.randint(0, vocab, (m, 24), generator=gen, device="cuda")
        logits.scatter_(1, top, 8.0 + 3.0 * randn(m, 24))
    if case["logits"] == "masked":
        logits.masked_fill_(rand(m, vocab) > max(0.01, 20.0 / vocab), -math.inf)
    logits = logits.to(torch.bfloat16)
    uniform = rand(m)
    if case["params"] == "plain":
        params = {"temperature": 0.8}
    elif case["params"] == "shared":
        params = {"temperature": 0.7, "top_k": 400, "top_p": 0.95, "min_p": 0.01}
    else:  # a tenth of the requests greedy, each filter off for a part of them
        off = lambda p, t, v: torch.where(rand(m) < p, v, t)  # noqa: E731
        params = {
            "temperature": off(0.1, 0.3 + 1.2 * rand(m), 0.0),
            "top_k": off(0.3, torch.exp(rand(m) * math.log(1000.0)).round(), 0.0).to(torch.int32),
            "top_p": off(0.3, 0.5 + 0.5 * rand(m), 1.0),
            "min_p": off(0.5, 0.1 * rand(m), 0.0),
        }
    return {"logits": logits, "uniform": uniform, "params": params}


_INPUTS = {"lora": _lora_inputs, "rope": _rope_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = _INPUTS[case["op"]](case, gen)
    state["case"] = case
    return state


# The plain forms.

def _plain_dequantize(w, s, b, bits, group):
    shifts = torch.arange(32 // bits, device=w.device, dtype=torch.int32) * bits
    codes = ((w[:, :, None] >> shifts) & (2**bits - 1)).reshape(w.shape[0], -1, group)
    # (s * q is exact in 32 bits; the format's weights are bf16)
    return (s.float()[:, :, None] * codes + b.float()[:, :, None]).to(torch.bfloat16).float().reshape(w.shape[0], -1)


def _plain_lora(st):
    case = st["case"]
    x = st["x"].float()
    y = x @ _plain_dequantize(st["w"], st["s"], st["b"], case["bits"], case["group"]).T
    for a in range(st["lora_a"].shape[0]):
        t = x @ st["lora_a"][a].float().T
        t = torch.where((st["adapters"] == a)[:, None], t * st["lora_scale"][a], 0.0)
        y += t @ st["lora_b"][a].float().T
    return y.to(torch.bfloat16)


def _plain_rope_heads(x, weight, cos, sin, interleaved):
    x = x.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    rot, rest = n[..., :2 * half], n[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    c, s = cos[:, None], sin[:, None]
    ra, rb = a * c - b * s, b * c + a * s
    rot = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((rot, rest), -1).to(torch.bfloat16)


def _plain_rope(st):
    angle = st["positions"].double()[:, None] * st["inv_freq"].double()  # far positions need 64 bits
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    return (_plain_rope_heads(st["q"], st["wq"], cos, sin, st["interleaved"]),
            _plain_rope_heads(st["k"], st["wk"], cos, sin, st["interleaved"]))


def _per_row(value, m, default, dtype=torch.float32):
    if torch.is_tensor(value):
        return value[:, None]
    return torch.full((m, 1), default if value is None else value, dtype=dtype, device="cuda")


def _plain_sample(st):
    logits, p = st["logits"], st["params"]
    m, vocab = logits.shape
    t = _per_row(p.get("temperature"), m, 1.0).double()  # (64 bits: masses next to a border)
    top_k = _per_row(p.get("top_k"), m, 0, torch.int32).long()
    top_p = _per_row(p.get("top_p"), m, 1.0).double()
    min_p = _per_row(p.get("min_p"), m, 0.0).double()
    value = logits.double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    value, order = torch.sort(value, dim=-1, descending=True, stable=True)
    greedy = t <= 0
    w = torch.where(value == value[:, :1], 1.0, torch.exp((value - value[:, :1]) / torch.where(greedy, 1.0, t)))
    rank = torch.arange(vocab, device="cuda")
    w = torch.where((top_k <= 0) | (rank < top_k), w, 0.0)
    cum = torch.cumsum(w, -1)
    keep = (top_p >= 1) | (cum - w < top_p * cum[:, -1:])
    keep &= w >= min_p
    keep[:, 0] = True
    w = torch.where(keep & (~greedy | (rank == 0)), w, 0.0)
    cum = torch.cumsum(w, -1)
    at = (cum <= st["uniform"].double()[:, None] * cum[:, -1:]).sum(-1)
    at = torch.minimum(at, (w > 0).sum(-1) - 1)[:, None]
    empty = value[:, :1] == -math.inf
    token = torch.where(empty, -1, order.gather(1, at))
    logprob = torch.where(empty, -math.inf, torch.log(w.gather(1, at) / cum[:, -1:]))
    return token[:, 0], logprob[:, 0].float()


def run(state):
    op = state["case"]["op"]
    if own:
        path = os.path.join(_ROOT, "mlx-tree-spec_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import mlx_tree_spec_amd as qmm

        if op == "lora":
            case = state["case"]
            return qmm.quantized_matmul_lora(state["x"], state["w"], state["s"], state["b"], state["lora_a"],
                                             state["lora_b"], state["lora_scale"], state["adapters"],
                                             group_size=case["group"], bits=case["bits"])
        if op == "rope":
            return qmm.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"], EPS, state["positions"],
                                    state["inv_freq"], interleaved=state["interleaved"])
        return qmm.sample(state["logits"], state["uniform"], **state["params"])
    return {"lora": _plain_lora, "rope": _plain_rope, "sample": _plain_sample}[op](state)


def work(case):
    m = case["m"]
    if case["op"] == "lora":
        k, n, r = case["k"], case["n"], case["rank"]
        used = min(case["requests"] - case["bare"], case["loaded"])
        weights = n * k * case["bits"] // 8 + 4 * n * (k // case["group"])
        nbytes = weights + 2 * m * (k + n) + used * (2 * r * (k + n) + 4) + 4 * m
        return {"bytes": nbytes, "flops": 2 * m * n * k + 2 * m * r * (k + n)}
    if case["op"] == "rope":
        elements = m * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": 4 * elements + 4 * case["dim"] + 4 * m + 4 * case["rotary"], "flops": 6 * elements}
    per_row = {"plain": 4 + 12, "shared": 4 + 12, "mixed": 4 + 12 + 16}[case["params"]]
    return {"bytes": m * (2 * case["vocab"] + per_row), "flops": m * case["vocab"]}


# The definitions in 64 bits, apart from the plain forms above.

def _exact_lora(st):
    case = st["case"]
    bits, group = case["bits"], case["group"]
    x = st["x"].double()
    n, words = st["w"].shape
    k = words * 32 // bits
    index = torch.arange(k, device="cuda")
    y = torch.empty(x.shape[0], n, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // k)
    for i in range(0, n, step):
        word = st["w"][i:i + step].long() & 0xFFFFFFFF
        q = torch.bitwise_and(word[:, index * bits // 32] >> (index * bits % 32), 2**bits - 1)
        scale, bias = (t[i:i + step].double().repeat_interleave(group, 1) for t in (st["s"], st["b"]))
        w = (scale * q + bias).float().to(torch.bfloat16)  # (exact in 64 bits; 32 bits, then bf16, by the format)
        y[:, i:i + step] = x @ w.double().T
    for row_set in torch.unique(st["adapters"]).tolist():
        if row_set >= 0:
            rows = (st["adapters"] == row_set).nonzero()[:, 0]
            delta = (st["lora_b"][row_set].double() @ (st["lora_a"][row_set].double() @ x[rows].T)).T
            y[rows] += st["lora_scale"][row_set].double() * delta
    return y


def _exact_rope(st):
    def heads(x, weight):
        x = x.double()
        n = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
        half = st["inv_freq"].shape[0]
        first = torch.arange(half, device="cuda") * (2 if st["interleaved"] else 1)
        second = first + (1 if st["interleaved"] else half)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           st["positions"].double()[:, None, None] * st["inv_freq"].double())
        pair = torch.complex(n[..., first], n[..., second]) * turn
        n[..., first], n[..., second] = pair.real, pair.imag
        return n

    return heads(st["q"], st["wq"]), heads(st["k"], st["wk"])


def _exact_sample(st):
    logits = st["logits"].float().cpu().numpy().astype(np.float64)
    uniform = st["uniform"].cpu().numpy().astype(np.float64)
    m = logits.shape[0]

    def rows(name, default):
        v = st["params"].get(name, default)
        return v.cpu().numpy().astype(np.float64) if torch.is_tensor(v) else np.full(m, np.float32(v), np.float64)

    t, top_k, top_p, min_p = (rows(*a) for a in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
    out, logprob = np.empty(m, np.int64), np.zeros(m)
    for i in range(m):
        order = np.argsort(-logits[i], kind="stable")
        if logits[i][order[0]] == -np.inf:
            out[i], logprob[i] = -1, -np.inf
            continue
        if t[i] <= 0:
            out[i] = order[0]
            continue
        p = np.exp((logits[i][order] - logits[i][order[0]]) / t[i])
        if top_k[i] > 0:
            p = p[:int(top_k[i])]
        if top_p[i] < 1:
            before = np.concatenate(([0.0], np.cumsum(p)[:-1]))
            p = p[:max(1, int(np.sum(before < top_p[i] * p.sum())))]
        p = p[:max(1, int(np.sum(p >= min_p[i])))]
        at = min(int(np.sum(np.cumsum(p) <= uniform[i] * p.sum())), int(np.sum(p > 0)) - 1)
        out[i], logprob[i] = order[at], np.log(p[at] / p.sum())
    return torch.from_numpy(out).cuda(), torch.from_numpy(logprob).cuda()


def exact(case, seed):
    state = prepare(case, seed)
    return {"lora": _exact_lora, "rope": _exact_rope, "sample": _exact_sample}[case["op"]](state)
