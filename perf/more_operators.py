"""What the paged key-value cache's operators are timed on, with their plain forms.

A layer of a batched decode or tree-verify step writes its new keys and values into a cache of pages and attends over
it. The pages are handed out on the GPU, once per step for all layers:

  tables  step_tables_: from the requests' lengths and new rows, the pages that they give back and take, and each
          new row's place (slot, position, request)
  store   store_kv_: new keys and values into the cache at their slots, as bf16 or as 8-bit codes with a scale for each
          row and head
  attend  paged_attention: each request's new rows (one, or the nodes of a tree with a mask of ancestors) over its
          cached keys and values, times the sigmoid of a gate where the heads come with one

Heads are those of the target model (24 query heads of 256 with their gates, 4 key heads) and generic ones, at the rows
of decode (1 per request), tree verify (up to 64) and prompts.

The cache's layout: keys [pages, Hk, D / E, page, E], values [pages, Hk, page / E, D, E], where E values are 16 bytes (8 of
bf16, 16 codes); scales fp32 [pages, Hk, page]. Slot s is token s % page of page s // page.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tables(name, kind, requests, rows, longest, page, capacity):
    """kind: "decode" (a row each), "verify" (up to `rows` nodes each, then the accepted ones kept), "admit" (prompts of
    `rows` tokens in all enter, then leave)."""
    return {"name": name, "op": "tables", "kind": kind, "requests": requests, "rows": rows, "longest": longest,
            "page": page, "capacity": capacity}


def _store(name, m, heads, dim, page, requests, bits=16, dropped=0):
    """`requests` runs of consecutive slots; the last `dropped` rows have none."""
    return {"name": name, "op": "store", "m": m, "heads": heads, "dim": dim, "page": page, "requests": requests,
            "bits": bits, "dropped": dropped}


def _attend(name, requests, rows, longest, q_heads, k_heads, dim, page=64, bits=16, tree=False, gated=False, idle=0, pad=0):
    """Requests of longest / 8 to `longest` cached tokens (one alone: `longest`), each with up to `rows` new ones (`idle` of
    them with none), and `pad` rows behind the last."""
    return {"name": name, "op": "attend", "requests": requests, "rows": rows, "longest": longest, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "page": page, "bits": bits, "tree": tree, "gated": gated, "idle": idle,
            "pad": pad}


def listed():
    return [
        # A decode step of a small server: a token each, a page for some.
        _tables("tables decode 16", "decode", 16, 1, 8000, 64, 512),
        # A tree-verify step of a large one: pages for every node, then back to the accepted nodes.
        _tables("tables verify 100x16", "verify", 100, 16, 16000, 64, 512),
        # Long prompts enter and leave.
        _tables("tables admit 50000 rows", "admit", 24, 50000, 20000, 64, 512),
        # Decode: one row of each of 16 requests.
        _store("store decode 16x4x256", 16, 4, 256, 64, 16),
        # A chunk of prompts.
        _store("store prompt 4096x8x128", 4096, 8, 128, 64, 3),
        # The same into a cache of 8 bits, the target model's heads, some rows padding.
        _store("store 8-bit 1500x4x256", 1500, 4, 256, 64, 5, bits=8, dropped=20),
        # One user at a short context, where latency counts.
        _attend("attend decode 1x2000 24/4x256", 1, 1, 2000, 24, 4, 256, gated=True),
        # A server's decode: 64 slots, some idle, ragged contexts.
        _attend("attend decode 64x16000 32/8x128", 64, 1, 16000, 32, 8, 128, idle=3, pad=3),
        # The same out of a cache of 8 bits at longer contexts.
        _attend("attend 8-bit 16x40000 24/4x256", 16, 1, 40000, 24, 4, 256, bits=8, gated=True),
        # Batched tree verify: 4 requests of up to 16 nodes.
        _attend("attend verify 4x16x8000 24/4x256", 4, 16, 8000, 24, 4, 256, tree=True, gated=True),
        # One request's widest tree over a long context.
        _attend("attend verify 1x64x32000 32/8x128", 1, 64, 32000, 32, 8, 128, tree=True),
        # One user at a very long context.
        _attend("attend decode 1x200000 24/4x256", 1, 1, 200000, 24, 4, 256, gated=True),
    ]


LARGEST_TOKENS = 200000 * 4 * 256          # cached tokens x key heads x head width
LARGEST_PRODUCT = 64 * 32000 * 32 * 128    # rows x cached tokens x query heads x head width
LARGEST_STORE = 4096 * 8 * 128
HEADS = [(24, 4), (32, 8), (16, 16), (28, 4), (40, 8), (64, 8), (8, 1), (6, 3)]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _draw_tables(rng):
    kind = rng.choice(["decode", "verify", "admit"])
    requests = round(_log_uniform(rng, 1, 256))
    page = rng.choice([16, 32, 64, 128, 256])
    longest = round(_log_uniform(rng, 50, 30000))
    rows = {"decode": 1, "verify": rng.randint(2, 64), "admit": round(_log_uniform(rng, requests, 50000))}[kind]
    capacity = (max(longest, rows) + 64 + page - 1) // page + rng.randint(0, 20)
    return _tables("", kind, requests, rows, longest, page, capacity)


def _draw_store(rng):
    heads, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 96, 128, 192, 256])
    bits = 8 if dim % 64 == 0 and rng.random() < 0.4 else 16
    m = round(_log_uniform(rng, 1, min(8192, LARGEST_STORE // (heads * dim))))
    dropped = rng.randint(0, m - 1) // 4
    return _store("", m, heads, dim, rng.choice([16, 32, 64, 128]), min(m - dropped, round(_log_uniform(rng, 1, 64))), bits,
                  dropped)


def _draw_attend(rng):
    q_heads, k_heads = rng.choice(HEADS)
    dim = rng.choice([64, 96, 128, 128, 192, 256, 256])
    bits = 8 if dim % 64 == 0 and rng.random() < 0.3 else 16
    requests = round(_log_uniform(rng, 1, 64))
    rows = 1 if rng.random() < 0.5 else rng.randint(2, 64)
    most = min(LARGEST_TOKENS // (k_heads * dim), LARGEST_PRODUCT // (rows * q_heads * dim)) // requests
    longest = round(_log_uniform(rng, 1, max(2, min(200000, most))))
    return _attend("", requests, rows, longest, q_heads, k_heads, dim, rng.choice([16, 32, 64, 64, 128]), bits,
                   rows > 1 and rng.random() < 0.7, rng.random() < 0.4, rng.randint(0, requests - 1) // 4, rng.choice([0, 0, 3]))


def draw(rng):
    case = rng.choice([_draw_tables, _draw_store, _draw_attend, _draw_attend])(rng)
    del case["name"]
    return case


# A case's lengths and rows belong to it; what the seed draws are the values, the pages' order and the trees.

def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """(cached tokens, new rows) of each request."""
    rng, r = _rng(case), case["requests"]
    long = case["longest"]
    cached = [long if r == 1 else rng.randint(long // 8, long) for _ in range(r)]
    if case["op"] == "tables" and case["kind"] == "admit":
        cuts = sorted(rng.sample(range(1, case["rows"]), r - 1)) if r > 1 else []
        rows = [b - a for a, b in zip([0, *cuts], [*cuts, case["rows"]])]
        return [0] * r, rows
    if case["op"] == "tables" and case["kind"] == "decode":
        return cached, [1] * r
    rows = [case["rows"] if r == 1 or case["rows"] == 1 else rng.randint(1, case["rows"]) for _ in range(r)]
    for i in rng.sample(range(r), case.get("idle", 0)):
        rows[i] = 0
    return cached, rows


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages_of(lengths, page, capacity, gen, spare):
    """(block table, free pages, free count): the pages in the order of a server that has run for a while."""
    held = [(n + page - 1) // page for n in lengths]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), capacity), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[:spare] = order[at:]
    return table, free, _int([spare])


def _trees(rows, gen):
    """The mask of each row: itself and its ancestors among its request's rows, a bit each (bit 63 is the sign)."""
    seed = int(torch.randint(0, 2**31, (1,), generator=gen, device="cuda"))
    rng, masks = random.Random(seed), []
    for n in rows:
        first = len(masks)
        for i in range(n):
            up = masks[first + max(rng.randrange(i), rng.randrange(i))] if i else 0
            masks.append(up | 1 << i)
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _tables_inputs(case, gen):
    cached, rows = _lengths(case)
    page, capacity = case["page"], case["capacity"]
    spare = sum((n + page - 1) // page + 1 for n in rows) + 8
    table, free, count = _pages_of(cached, page, capacity, gen, spare)
    keep = None
    if case["kind"] == "verify":  # the accepted path: some of the nodes
        keep = torch.rand(sum(rows), generator=gen, device="cuda") < 0.3
    return {"lengths": _int(cached), "table": table, "free": free, "count": count, "rows": _int(rows),
            "base": _int(cached), "none": _int([0] * len(rows)), "keep": keep, "total": sum(rows)}


def _cache(case, heads, pages, gen):
    """Keys and values of `pages` pages as earlier steps left them, and their scales (None for bf16)."""
    page, d = case["page"], case["dim"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["bits"] == 16:
        keys = randn(pages, heads, d // 8, page, 8).to(torch.bfloat16)
        return keys, randn(pages, heads, page // 8, d, 8).to(torch.bfloat16), None, None
    keys = torch.randint(-127, 128, (pages, heads, d // 16, page, 16), generator=gen, device="cuda", dtype=torch.int8)
    values = torch.randint(-127, 128, (pages, heads, page // 16, d, 16), generator=gen, device="cuda", dtype=torch.int8)
    scales = lambda: (1 + torch.rand(pages, heads, page, generator=gen, device="cuda")) / 127  # noqa: E731
    return keys, values, scales(), scales()


def _store_inputs(case, gen):
    m, heads, d, page, n = case["m"], case["heads"], case["dim"], case["page"], case["m"] - case["dropped"]
    rng = _rng(case)
    cuts = sorted(rng.sample(range(1, n), case["requests"] - 1)) if case["requests"] > 1 else []
    runs = [b - a for a, b in zip([0, *cuts], [*cuts, n])]
    starts = [rng.randrange(4 * page) for _ in runs]  # a request's rows begin anywhere in a page
    held = [(s % page + n + page - 1) // page for s, n in zip(starts, runs)]
    pages = sum(held) + 4
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    slots, at = torch.full((m,), -1, dtype=torch.int32, device="cuda"), 0
    row = 0
    for s, length, h in zip(starts, runs, held):
        token = s % page + torch.arange(length, device="cuda")
        slots[row:row + length] = order[at + token // page] * page + token.to(torch.int32) % page
        row, at = row + length, at + h
    keys, values, k_scales, v_scales = _cache(case, heads, pages, gen)
    size = 0.5 + 2 * torch.rand(heads, 1, generator=gen, device="cuda")
    k = (torch.randn(m, heads, d, generator=gen, device="cuda") * size).to(torch.bfloat16)
    qkv = torch.randn(m, 6 * heads, d, generator=gen, device="cuda").to(torch.bfloat16)
    v = qkv[:, 5 * heads:]  # a part of a fused projection
    return {"k": k, "v": v, "slots": slots, "keys": keys, "values": values, "k_scales": k_scales, "v_scales": v_scales}


def _attend_inputs(case, gen):
    cached, rows = _lengths(case)
    page, d, hq, hk = case["page"], case["dim"], case["q_heads"], case["k_heads"]
    lengths = [c + n for c, n in zip(cached, rows)]
    capacity = max((n + page - 1) // page for n in lengths) + 2
    table, free, count = _pages_of(lengths, page, capacity, gen, 4)
    keys, values, k_scales, v_scales = _cache(case, hk, free.shape[0], gen)
    m = sum(rows) + case["pad"]
    q = (1.5 * torch.randn(m, hq, 2 * d if case["gated"] else d, generator=gen, device="cuda")).to(torch.bfloat16)
    masks = torch.tensor(_trees(rows, gen) + [0] * case["pad"], dtype=torch.int64, device="cuda") if case["tree"] else None
    state = {"q": q[..., :d], "gate": q[..., d:] if case["gated"] else None, "keys": keys, "values": values,
             "k_scales": k_scales, "v_scales": v_scales, "table": table, "ancestors": masks, "scale": d ** -0.5,
             "cached": cached, "rows": rows}
    if own:  # a step's tables, which all its layers share
        state["step"] = _package().step_tables_(_int(lengths), table, free, count, _int(rows), m, page, hq, hk, d,
                                                base=_int(cached), max_rows=case["rows"])
    return state


_INPUTS = {"tables": _tables_inputs, "store": _store_inputs, "attend": _attend_inputs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = _INPUTS[case["op"]](case, gen)
    state["case"] = case
    return state


# The plain forms.

def _plain_step(st, rows, total, page, keep=None):
    lengths, table, free, count = st["lengths"], st["table"], st["free"], st["count"]
    capacity, pages = table.shape[1], free.shape[0]
    base = torch.minimum(st["base"].clamp(min=0), lengths)
    end = torch.cumsum(rows, 0)
    request = torch.searchsorted(end, torch.arange(total, device="cuda"), right=True).clamp(max=rows.shape[0] - 1)
    kept = torch.ones(total, dtype=torch.bool, device="cuda") if keep is None else keep
    new = torch.zeros_like(rows).index_add_(0, request, kept.to(torch.int32))
    had, left = (lengths + page - 1) // page, (base + page - 1) // page
    # What lies past the base goes back, last page lowest.
    column = torch.arange(capacity, device="cuda")
    back = (column >= left[:, None]) & (column < had[:, None])
    rank = torch.cumsum(back.flatten(), 0).reshape(back.shape)
    available = count + rank[-1, -1]
    free_ext = torch.cat((free, free.new_zeros(1)))
    free_ext[torch.where(back, available - rank, pages)] = torch.where(back, table, 0)
    free.copy_(free_ext[:pages])
    table.masked_fill_(back, -1)
    # Then pages are taken in the order of requests.
    want = (base + new + page - 1) // page
    need = torch.where(want > capacity, 0, want - left)
    refused = (want > capacity) | ((need > 0) & (torch.cumsum(need, 0) > available))
    new, want = torch.where(refused, 0, new), torch.where(refused, left, want)
    taken = (column >= left[:, None]) & (column < want[:, None])
    rank = torch.cumsum(taken.flatten(), 0).reshape(taken.shape)
    table.copy_(torch.where(taken, free[(available - rank).clamp(0, pages - 1)], table))
    count.copy_(available - rank[-1, -1])
    lengths.copy_(base + new)
    cum = torch.cumsum(kept, 0)
    first = torch.cat((cum.new_zeros(1), cum))[end - rows]
    position = base[request] + cum - 1 - first[request]
    placed = kept & ~refused[request]
    at = table[request, (position // page).clamp(0, capacity - 1)].long() * page + position % page
    return tuple(torch.where(placed, x, -1).to(torch.int32) for x in (at, position, request))


def _rows_of(t, page):
    """Tokens of cache pages [pages, heads, .., ..., E]: keys' layout -> [pages, page, heads, D]."""
    return t.permute(0, 3, 1, 2, 4).flatten(3)


def _put(keys, slots, rows, page, values=False):
    e = keys.shape[-1]
    p, t = slots // page, slots % page
    if values:  # [pages, heads, page / E, D, E]
        keys.permute(0, 2, 4, 1, 3)[p, t // e, t % e] = rows
    else:       # [pages, heads, D / E, page, E]
        keys.permute(0, 3, 1, 2, 4)[p, t] = rows.unflatten(-1, (-1, e))


def _plain_codes(x):
    x = x.float()
    scale = x.abs().amax(-1) / 127.0
    code = torch.where(scale[..., None] > 0, torch.round(x / scale[..., None]), 0.0).clamp(-127, 127)
    return code.to(torch.int8), scale


def _plain_store(st):
    page = st["case"]["page"]
    at = (st["slots"] >= 0).nonzero()[:, 0]
    slots, k, v = st["slots"][at].long(), st["k"][at], st["v"][at]
    if st["case"]["bits"] == 8:
        (k, k_scale), (v, v_scale) = _plain_codes(k), _plain_codes(v)
        st["k_scales"].permute(0, 2, 1)[slots // page, slots % page] = k_scale
        st["v_scales"].permute(0, 2, 1)[slots // page, slots % page] = v_scale
    _put(st["keys"], slots, k, page)
    _put(st["values"], slots, v, page, values=True)


def _stored(st):
    """The cache's content: bf16 as it is, codes as the values that they stand for."""
    if st["case"]["bits"] == 16:
        return st["keys"], st["values"]
    page, e = st["case"]["page"], 16
    keys = (st["keys"] * st["k_scales"][:, :, None, :, None]).to(torch.bfloat16)
    values = (st["values"] * st["v_scales"].unflatten(2, (page // e, 1, e))).to(torch.bfloat16)
    return keys, values, st["k_scales"], st["v_scales"]


def _context(st, r, length, dtype):
    """(K, V) of a request's first `length` tokens, [heads, length, D]."""
    page = st["case"]["page"]
    at = st["table"][r, :(length + page - 1) // page].long()
    keys, values = st["keys"][at].to(dtype), st["values"][at].to(dtype)
    if st["k_scales"] is not None:
        keys *= st["k_scales"][at].to(dtype)[:, :, None, :, None]
        values *= st["v_scales"][at].to(dtype).unflatten(2, (-1, 1, values.shape[-1]))
    keys = keys.permute(1, 0, 3, 2, 4).flatten(3).flatten(1, 2)[:, :length]
    values = values.permute(1, 0, 2, 4, 3).flatten(1, 3)[:, :length]
    return keys, values


def _visible(st, first, n, cached):
    """Whether each of a request's n rows sees each of them, [n, n]."""
    i = torch.arange(n, device="cuda")
    if st["ancestors"] is None:
        return i[None, :] <= i[:, None]
    return (st["ancestors"][first:first + n, None] >> i) & 1 == 1


def _plain_attend(st):
    case = st["case"]
    hq, hk, d = case["q_heads"], case["k_heads"], case["dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float32, device="cuda")
    first = 0
    for r, (cached, n) in enumerate(zip(st["cached"], st["rows"])):
        if n == 0:
            continue
        keys, values = _context(st, r, cached + n, torch.float32)
        q = st["q"][first:first + n].float().reshape(n, hk, hq // hk, d).transpose(0, 1).reshape(hk, -1, d)
        s = (q @ keys.transpose(1, 2).contiguous() * st["scale"]).reshape(hk, n, hq // hk, cached + n)
        hidden = ~_visible(st, first, n, cached)
        s[..., cached:].masked_fill_(hidden[:, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
        p = (p / p.sum(-1, keepdim=True)).reshape(hk, -1, cached + n)
        out[first:first + n] = (p @ values.contiguous()).reshape(hk, n, hq // hk, d).transpose(0, 1).reshape(n, hq, d)
        first += n
    if st["gate"] is not None:
        out = out * torch.sigmoid(st["gate"].float())
    return out.to(torch.bfloat16)


def _package():
    path = os.path.join(_ROOT, "mlx-tree-spec_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mlx_tree_spec_amd as qmm

    return qmm


def _passes(case):
    """The calls that one pass over the tables makes, as (rows, total, keep): names in a state."""
    if case["kind"] == "decode":
        return [("rows", "total", None)]
    if case["kind"] == "verify":
        return [("rows", "total", None), ("rows", "total", "keep")]
    return [("rows", "total", None), ("none", 0, None)]


def _run_tables(st):
    case, out = st["case"], []
    for rows, total, keep in _passes(case):
        total, keep = st[total] if total else 0, st[keep] if keep else None
        if own:
            step = _package().step_tables_(st["lengths"], st["table"], st["free"], st["count"], st[rows], total, case["page"],
                                           32, 8, 128, base=st["base"], keep=keep, max_rows=case["rows"])
            out += [step.slots, step.positions, step.request]
        else:
            out += _plain_step(st, st[rows], total, case["page"], keep)
    return [*out, st["lengths"], st["table"], st["free"], st["count"]]


def run(state):
    case = state["case"]
    if case["op"] == "tables":
        return _run_tables(state)
    if not own:
        if case["op"] == "attend":
            return _plain_attend(state)
        _plain_store(state)
        return _stored(state)
    qmm = _package()
    cache = qmm.KVCache(state["keys"], state["values"], state["k_scales"], state["v_scales"])
    if case["op"] == "attend":
        return qmm.paged_attention(state["q"], cache, state["step"], scale=state["scale"], ancestors=state["ancestors"],
                                   gate=state["gate"])
    qmm.store_kv_(state["k"], state["v"], cache, state["slots"])
    return _stored(state)


def work(case):
    if case["op"] == "tables":
        cached, rows = _lengths(case)
        page, r = case["page"], case["requests"]
        pages = lambda n: (n + page - 1) // page  # noqa: E731
        moved = sum(pages(c + n) - pages(c) for c, n in zip(cached, rows))
        calls = len(_passes(case))
        nbytes = calls * 12 * r + (4 + 12) * sum(rows) + 8 * moved + 8
        if case["kind"] == "verify":
            nbytes += 13 * sum(rows) + 8 * moved
        if case["kind"] == "admit":
            nbytes += 8 * moved
        return {"bytes": nbytes, "flops": 10 * (sum(rows) + r) * calls}
    if case["op"] == "store":
        n = (case["m"] - case["dropped"]) * case["heads"]
        per = 4 * case["dim"] + (4 * case["dim"] if case["bits"] == 16 else 2 * case["dim"] + 8)
        return {"bytes": n * per + 4 * case["m"], "flops": n * case["dim"] * (2 if case["bits"] == 16 else 8)}
    cached, rows = _lengths(case)
    d, hq, hk = case["dim"], case["q_heads"], case["k_heads"]
    tokens = sum(c + n for c, n in zip(cached, rows) if n)
    per = 4 * d if case["bits"] == 16 else 2 * d + 8
    m = sum(rows)
    nbytes = tokens * hk * per + m * hq * d * (6 if case["gated"] else 4) + tokens // case["page"] * 4 + (8 * m if case["tree"] else 0)
    return {"bytes": nbytes, "flops": 4 * d * hq * sum(n * (c + n) for c, n in zip(cached, rows))}


# The definitions apart from the plain forms above, in 64 bits where they compute numbers.

def _exact_tables(st):
    case, page = st["case"], st["case"]["page"]
    lengths, count = st["lengths"].tolist(), int(st["count"])
    table, free = st["table"].cpu().numpy().copy(), st["free"].tolist()
    base, capacity, out = st["base"].tolist(), table.shape[1], []
    for rows, total, keep in _passes(case):
        total, keep = st[total] if total else 0, st[keep].tolist() if keep else [True] * st["total"]
        back = []
        for r, n in enumerate(lengths):
            base_r = min(base[r], n)
            for c in range(-(-base_r // page), -(-n // page)):
                back.append(int(table[r, c]))
                table[r, c] = -1
            lengths[r] = base_r
        free[count:count + len(back)] = back[::-1]
        count += len(back)
        got, row, short = [[-1] * total for _ in range(3)], 0, False
        for r, n in enumerate(st[rows].tolist()):
            mine = [m for m in range(row, row + n) if keep[m]]
            row += n
            have, want = -(-lengths[r] // page), -(-(lengths[r] + len(mine)) // page)
            if want > capacity:
                continue
            short = short or want - have > count
            if want > have and short:
                continue
            for c in range(have, want):
                count -= 1
                table[r, c] = free[count]
            for i, m in enumerate(mine):
                at = lengths[r] + i
                got[0][m], got[1][m], got[2][m] = int(table[r, at // page]) * page + at % page, at, r
            lengths[r] += len(mine)
        out += [_int(x) for x in got]
    return [*out, _int(lengths), torch.from_numpy(table).cuda(), _int(free), _int([count])]


def _exact_store(st):
    case, page = st["case"], st["case"]["page"]
    e = 8 if case["bits"] == 16 else 16
    slots = st["slots"].cpu().numpy()
    keys, values = st["keys"].double().cpu().numpy(), st["values"].double().cpu().numpy()
    scales = [s.cpu().numpy() for s in (st["k_scales"], st["v_scales"])] if e == 16 else None
    if scales:
        keys *= scales[0].astype(np.float64)[:, :, None, :, None]
        values *= scales[1].astype(np.float64).reshape(values.shape[:3] + (1, e))
    rows = [st["k"].double().cpu().numpy(), st["v"].double().cpu().numpy()]
    stored = list(rows)
    if scales:
        for i in range(2):
            scale = (np.abs(rows[i]).max(-1) / 127).astype(np.float32)  # (the format's scales are 32 bits)
            step = np.where(scale > 0, scale.astype(np.float64), 1.0)[..., None]
            stored[i] = np.rint(rows[i] / step) * step
            rows[i] = scale
    for m, slot in enumerate(slots):
        if slot < 0:
            continue
        p, t = divmod(int(slot), page)
        keys[p, :, :, t, :] = stored[0][m].reshape(keys.shape[1], -1, e)
        values[p, :, t // e, :, t % e] = stored[1][m]
        if scales:
            scales[0][p, :, t], scales[1][p, :, t] = rows[0][m], rows[1][m]
    out = [torch.from_numpy(x).cuda() for x in (keys, values)]
    return out + [torch.from_numpy(x.astype(np.float64)).cuda() for x in scales] if scales else out


def _exact_attend(st):
    case = st["case"]
    group = case["q_heads"] // case["k_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    page, d = case["page"], case["dim"]
    for r, (cached, n) in enumerate(zip(st["cached"], st["rows"])):
        if n == 0:
            continue
        rows = slice(first, first + n)
        token = torch.arange(cached + n, device="cuda")
        p, t = st["table"][r].long()[token // page], token % page
        e = st["keys"].shape[-1]
        sees = torch.ones(n, cached + n, dtype=torch.float64, device="cuda")
        for i in range(n):
            bits = (1 << i + 1) - 1 if st["ancestors"] is None else int(st["ancestors"][first + i])
            sees[i, cached:] = torch.tensor([float(bits >> j & 1) for j in range(n)], dtype=torch.float64)
        keys, values = [], []
        for h in range(case["k_heads"]):
            k = st["keys"][p, h, :, t].double().reshape(-1, d)
            v = st["values"][p, h, t // e, :, t % e].double()
            if st["k_scales"] is not None:
                k *= st["k_scales"][p, h, t].double()[:, None]
                v *= st["v_scales"][p, h, t].double()[:, None]
            keys.append(k)
            values.append(v)
        for h in range(case["q_heads"]):
            logits = st["q"][rows, h].double() @ keys[h // group].T * st["scale"]
            top = torch.where(sees > 0, logits, -math.inf).max(-1, keepdim=True).values
            w = sees * torch.exp(torch.minimum(logits - top, torch.zeros((), dtype=torch.float64, device="cuda")))
            out[rows, h] = (w @ values[h // group]) / w.sum(-1, keepdim=True)
        first += n
    if st["gate"] is not None:
        out /= 1 + torch.exp(-st["gate"].double())
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"tables": _exact_tables, "store": _exact_store, "attend": _exact_attend}[case["op"]](state)
