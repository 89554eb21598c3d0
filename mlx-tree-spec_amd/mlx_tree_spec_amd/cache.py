"""The paged key-value cache of a batched step, backed by libqmm4.so (gfx950 HIP).

Between a layer's attention inputs and its tail (src/mlx_tree_spec/tree_verify.py:311-402) lie the cache and the attention over
it. Requests' tokens live in pages that all layers number alike:

  step_tables_(lengths, block_table, free_pages, free_count, rows, total, page_size, heads, kv_heads, head_dim, ...)
      -> CacheStep: once a step, on the GPU: pages given back and taken, each new row's slot, position and request
  store_kv_(k, v, cache, slots): a layer's new keys and values into its cache, bf16 or 8-bit codes (kv8.py:244-288)
  paged_attention(q, cache, step, ...): its attention, split over the cache's length (tree_flash.py:117-196)
  KVCache, CacheTables: a layer's arrays, and the tables that all layers share

Everything works on lengths that only the GPU knows, so a step can be captured once and replayed. Tensors are on a HIP
device; there is no CPU path, and no gradient.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .heads import _head_rows, _strides
from .lora import no_gradient
from .qmm import _check_device

MAX_REQUESTS = 2048
MAX_ROWS = 1 << 22
MAX_KEEP = 1 << 16
MAX_CAPACITY = 1 << 22
MAX_TOKENS = 1 << 30
HEAD_DIMS = (64, 96, 128, 192, 256)


class KVCache(NamedTuple):
    """A layer's keys [pages, Hk, D / E, page, E] and values [pages, Hk, page / E, D, E], bf16 (E = 8) or int8 codes (E = 16)
    with their scales, fp32 [pages, Hk, page]: slot s is token s % page of page s // page."""
    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor | None = None
    value_scales: torch.Tensor | None = None

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 16, device="cuda") -> "KVCache":
        """A cache of `pages` pages; what it holds before it is stored to is never read into a result."""
        _check_page_size("KVCache", page_size)
        if bits not in (16, 8):
            raise NotImplementedError(f"[KVCache] bits={bits}: caches of 16 (bf16) or 8 bits are supported")
        _check_dim("KVCache", head_dim, bits == 8)
        e, dtype = (8, torch.bfloat16) if bits == 16 else (16, torch.int8)
        keys = torch.empty((pages, kv_heads, head_dim // e, page_size, e), dtype=dtype, device=device)
        values = torch.empty((pages, kv_heads, page_size // e, head_dim, e), dtype=dtype, device=device)
        if bits == 16:
            return cls(keys, values)
        scales = (torch.empty((pages, kv_heads, page_size), dtype=torch.float32, device=device) for _ in range(2))
        return cls(keys, values, *scales)


class CacheStep(NamedTuple):
    """A step's tables: slots, positions and request of each row, int32 [total] (-1: none), and what paged_attention needs
    (plan: None where rows were chosen by `keep`)."""
    slots: torch.Tensor
    positions: torch.Tensor
    request: torch.Tensor
    plan: torch.Tensor | None
    block_table: torch.Tensor
    page_size: int
    heads: int
    kv_heads: int
    head_dim: int
    max_rows: int


def _check_page_size(what: str, page_size: int) -> None:
    if page_size not in (16, 32, 64, 128, 256, 512, 1024):
        raise ValueError(f"[{what}] page_size={page_size} must be a power of two from 16 to 1024")


def _check_dim(what: str, head_dim: int, codes: bool) -> None:
    if head_dim not in HEAD_DIMS or codes and head_dim == 96:
        raise NotImplementedError(f"[{what}] heads of {head_dim} values{' in 8 bits' if codes else ''}: "
                                  f"{', '.join(map(str, HEAD_DIMS))} are supported (8 bits: not 96)")


def _check_heads(what: str, heads: int, kv_heads: int) -> None:
    if kv_heads < 1 or not 1 <= heads <= 1024 or heads % kv_heads:
        raise ValueError(f"[{what}] {heads} query heads and {kv_heads} key heads: the first must be a multiple of the second, "
                         "at most 1024")


def _table(what: str, name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype = torch.int32) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise ValueError(f"[{what}] {name} must be {dtype} of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _in_place(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
            raise ValueError(f"[{what}] {name} is written in place: it must be contiguous, on a 16-byte boundary")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def step_tables_(lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                 rows: torch.Tensor, total: int, page_size: int, heads: int, kv_heads: int, head_dim: int,
                 base: torch.Tensor | None = None, keep: torch.Tensor | None = None, max_rows: int | None = None) -> CacheStep:
    """One step of the tables, in place, and the new rows' places. `total` rows are packed one request behind the other,
    rows[r] of request r (none below 0, at most max_rows; those past `total` are cut off), padding behind the last. max_rows has to
    be at least the most rows of a request: a longer one is cut, and the next request's rows are taken to begin where it was cut.

    For each of R requests, with b = base[r] (by default its length; never more than that) and a = its rows, or with `keep`
    (bool [total]) those of them that are kept:
      its pages past ceil(b / page_size) go back to the free list, and their entries become -1; then, in the order of
      requests, it takes pages for b + a tokens from the list's end. The tokens get positions b, b + 1, .. and their slots.
    A request whose tokens would not fit its row of block_table is refused (no row of it gets a place, its length becomes b);
    so is every request that needs pages, from the first on for which too few are left. base 0 and rows 0 release a request;
    a tree verify stores all nodes, and then, with base the length before and `keep` the accepted nodes, these alone. A request
    that was refused for all nodes may fit with the kept ones, which have attended to nothing: keep & (step.request >= 0) leaves
    them out.

    lengths, rows, base int32 [R]; block_table int32 [R, capacity]; free_pages int32 [pages] (room for every page of the
    cache), the first free_count (int32 [1]) of which are free. Rows without a place (not kept, refused, padding) have -1 as
    slot, position and request. heads, kv_heads, head_dim: those of the layers whose attention takes this step. max_rows
    (total by default): the fewer, the better the attention's kernels fit (1 for a decode step). Up to 2048 requests, 2^22
    rows (2^16 with keep), 2^22 pages per request and 2^30 tokens.
    """
    what = "step_tables_"
    max_rows = total if max_rows is None else min(max_rows, total)
    out = None
    if lengths.is_cuda:
        out = _lib.native().cache_step(lengths, block_table, free_pages, free_count, rows, total, page_size, heads, kv_heads,
                                       head_dim, base, keep, max_rows)
        if type(out) is int:
            _lib.check(out, what)
    if out is None:
        out = _step_tables(what, lengths, block_table, free_pages, free_count, rows, total, page_size, heads, kv_heads,
                           head_dim, base, keep, max_rows)
    slots, positions, request, plan = out
    return CacheStep(slots, positions, request, plan, block_table, page_size, heads, kv_heads, head_dim, max_rows)


def _step_tables(what, lengths, block_table, free_pages, free_count, rows, total, page_size, heads, kv_heads, head_dim, base,
                 keep, max_rows):
    _check_page_size(what, page_size)
    _check_heads(what, heads, kv_heads)
    _check_dim(what, head_dim, False)
    if lengths.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError(f"[{what}] lengths, block_table and free_pages must have 1, 2 and 1 dimensions, got "
                         f"{tuple(lengths.shape)}, {tuple(block_table.shape)} and {tuple(free_pages.shape)}")
    r, capacity, pages = lengths.shape[0], block_table.shape[1], free_pages.shape[0]
    if r > MAX_REQUESTS or not 0 <= total <= MAX_ROWS or max_rows < 0:
        raise ValueError(f"[{what}] {r} requests, {total} rows, at most {max_rows} each: up to {MAX_REQUESTS} requests and "
                         f"{MAX_ROWS} rows are supported")
    if keep is not None and total > MAX_KEEP:
        raise ValueError(f"[{what}] {total} rows with keep: up to {MAX_KEEP} are supported")
    if capacity > MAX_CAPACITY:
        raise ValueError(f"[{what}] {capacity} pages per request: up to {MAX_CAPACITY} are supported")
    if max(capacity, pages) * page_size > MAX_TOKENS:
        raise ValueError(f"[{what}] {pages} pages, {capacity} per request, of {page_size} tokens: up to 2^30 tokens are supported")
    _table(what, "lengths", lengths, (r,))
    _table(what, "block_table", block_table, (r, capacity))
    _table(what, "free_pages", free_pages, (pages,))
    _table(what, "free_count", free_count, (1,))
    _table(what, "rows", rows, (r,))
    if base is not None:
        _table(what, "base", base, (r,))
    if keep is not None:
        _table(what, "keep", keep, (total,), torch.bool)
    dev = _check_device(what, lengths, block_table, free_pages, free_count, rows, *(t for t in (base, keep) if t is not None))
    for name, t in (("lengths", lengths), ("block_table", block_table), ("free_pages", free_pages), ("free_count", free_count)):
        if not t.is_contiguous():
            raise ValueError(f"[{what}] {name} is written in place: it must be contiguous")
    rows = rows.contiguous()
    base, keep = (t if t is None else t.contiguous() for t in (base, keep))
    lib = _lib.load()
    with torch.cuda.device(dev):
        words = lib.qmm4_cache_plan_words(r, heads, kv_heads, head_dim, max_rows)
        _lib.check(min(words, 0), what)
        slots, positions, request = (torch.empty(total, dtype=torch.int32, device=dev) for _ in range(3))
        plan = torch.empty(words, dtype=torch.int32, device=dev) if keep is None else None
        rc = lib.qmm4_cache_step(lengths.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
                                 rows.data_ptr(), _ptr(base), _ptr(keep), slots.data_ptr(), positions.data_ptr(),
                                 request.data_ptr(), _ptr(plan), r, capacity, pages, total, max_rows, page_size, heads,
                                 kv_heads, head_dim, torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, what)
    return slots, positions, request, plan


def _check_cache(what: str, cache: KVCache) -> tuple[int, int, int, int, int]:
    """(pages, kv_heads, head_dim, page_size, bits) of a layer's arrays."""
    keys, values, scales = cache.keys, cache.values, (cache.key_scales, cache.value_scales)
    if keys.dtype not in (torch.bfloat16, torch.int8) or values.dtype != keys.dtype:
        raise ValueError(f"[{what}] keys and values must both be bfloat16 or int8, got {keys.dtype} and {values.dtype}")
    bits, e = (16, 8) if keys.dtype == torch.bfloat16 else (8, 16)
    if keys.dim() != 5 or values.dim() != 5 or keys.shape[4] != e:
        raise ValueError(f"[{what}] keys and values must be [pages, heads, D / {e}, page, {e}] and [pages, heads, page / {e}, D, "
                         f"{e}], got {tuple(keys.shape)} and {tuple(values.shape)}")
    pages, heads, pieces, page_size, _ = keys.shape
    dim = pieces * e
    _check_page_size(what, page_size)
    _check_dim(what, dim, bits == 8)
    _check_heads(what, heads, heads)
    _table(what, "values", values, (pages, heads, page_size // e, dim, e), keys.dtype)
    for name, t in zip(("key_scales", "value_scales"), scales):
        if (t is not None) != (bits == 8):
            raise ValueError(f"[{what}] {name}: a cache of int8 has scales, one of bfloat16 has none")
        if t is not None:
            _table(what, name, t, (pages, heads, page_size), torch.float32)
    if pages * page_size > MAX_TOKENS:
        raise ValueError(f"[{what}] {pages} pages of {page_size} tokens: up to 2^30 tokens are supported")
    _in_place(what, keys=keys, values=values, key_scales=scales[0], value_scales=scales[1])
    return pages, heads, dim, page_size, bits


def store_kv_(k: torch.Tensor, v: torch.Tensor, cache: KVCache, slots: torch.Tensor) -> None:
    """k, v bf16 (M, Hk, D) into the cache, row m at slots[m] (int32 [M], different ones); rows whose slot is not one of the
    cache's, -1 by convention, are skipped. Strided rows and heads are read in place.

    In 8 bits each row's head has the scale max|x| / 127 and codes x / scale, rounded to the nearest; a head that is not finite
    stands for NaN.
    """
    what = "store_kv_"
    if k.is_cuda:
        out = _lib.native().store_kv(k, v, cache.keys, cache.values, cache.key_scales, cache.value_scales, slots)
        if type(out) is int:
            _lib.check(out, what)
            return
    no_gradient(what, k=k, v=v, keys=cache.keys, values=cache.values, key_scales=cache.key_scales,
                value_scales=cache.value_scales)
    pages, heads, dim, page_size, bits = _check_cache(what, cache)
    for name, t in (("k", k), ("v", v)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"[{what}] {name} must be bfloat16, got {t.dtype}")
        if t.dim() != 3 or tuple(t.shape[1:]) != (heads, dim) or t.shape[0] != k.shape[0]:
            raise ValueError(f"[{what}] {name} must be (rows, {heads}, {dim}), got {tuple(t.shape)}")
    m = k.shape[0]
    if m > MAX_ROWS:
        raise ValueError(f"[{what}] {m} rows: up to {MAX_ROWS} are supported")
    _table(what, "slots", slots, (m,))
    dev = _check_device(what, k, v, slots, *(t for t in cache if t is not None))
    k3, v3, slots = _head_rows(k), _head_rows(v), slots.contiguous()
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.qmm4_store_kv_bf16(k3.data_ptr(), *_strides(k3), v3.data_ptr(), *_strides(v3), slots.data_ptr(),
                                    cache.keys.data_ptr(), cache.values.data_ptr(), _ptr(cache.key_scales),
                                    _ptr(cache.value_scales), m, heads, dim, pages, page_size, bits,
                                    torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, what)


def _check_step(what: str, cache: KVCache, step: CacheStep, scale: float, ancestors: torch.Tensor | None) -> tuple[int, int]:
    """(pages, bits) of a cache that a step's rows can attend to."""
    pages, kv_heads, dim, page_size, bits = _check_cache(what, cache)
    if (kv_heads, dim, page_size) != (step.kv_heads, step.head_dim, step.page_size):
        raise ValueError(f"[{what}] a cache of {kv_heads} heads of {dim} in pages of {page_size}, but the step was made for "
                         f"{step.kv_heads} heads of {step.head_dim} in pages of {step.page_size}")
    m = step.request.shape[0]
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"[{what}] scale={scale} must be finite")
    if ancestors is not None:
        _table(what, "ancestors", ancestors, (m,), torch.int64)
    if step.block_table.dim() != 2:
        raise ValueError(f"[{what}] the step's block_table must have 2 dimensions, got {tuple(step.block_table.shape)}")
    for name, t, shape in (("block_table", step.block_table, tuple(step.block_table.shape)), ("request", step.request, (m,)),
                           ("plan", step.plan, tuple(step.plan.shape))):
        _table(what, f"the step's {name}", t, shape)
        if not t.is_contiguous():
            raise ValueError(f"[{what}] the step's {name} must be contiguous")
    if m > 0 and (pages == 0 or step.block_table.shape[1] == 0):
        raise ValueError(f"[{what}] a cache without pages has nothing to attend to")
    return pages, bits


def _check_plan(what: str, cache: KVCache, step: CacheStep, *others: torch.Tensor | None) -> torch.device:
    """The device of all of them, where the step's plan has the size of one for its requests and heads."""
    dev = _check_device(what, step.block_table, step.request, step.plan, *(t for t in (*cache, *others) if t is not None))
    with torch.cuda.device(dev):
        words = _lib.load().qmm4_cache_plan_words(step.block_table.shape[0], step.heads, step.kv_heads, step.head_dim, step.max_rows)
    _lib.check(min(words, 0), what)
    _table(what, "the step's plan", step.plan, (words,))
    return dev


def check_attention(what: str, cache: KVCache, step: CacheStep, scale: float | None, ancestors: torch.Tensor | None) -> None:
    """Raises where paged_attention would, whatever its rows are."""
    if step.plan is None:
        raise ValueError(f"[{what}] the step has no plan: it was made with keep")
    scale = 1.0 if scale is None else scale
    if cache.keys.is_cuda and _lib.native().paged(None, *cache, step.block_table, step.request, step.plan, step.heads, step.kv_heads,
                                                  step.head_dim, step.max_rows, step.page_size, float(scale), ancestors, None) is True:
        return
    _check_step(what, cache, step, scale, ancestors)
    _check_plan(what, cache, step, ancestors)


def paged_attention(q: torch.Tensor, cache: KVCache, step: CacheStep, scale: float | None = None,
                    ancestors: torch.Tensor | None = None, gate: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's rows over their requests' cached tokens, their own among them (stored before): bf16 (M, Hq, D)

        out[m, h] = softmax(scale * q[m, h] . keys of what the row sees) values  (* sigmoid(gate[m, h])),

    query head h over key head h // (Hq // Hk). A row sees every token before the step's, and of its request's rows those up
    to its own; with `ancestors` (int64 [M], a tree's masks) row j of its request where bit j is set, itself included (the
    64 rows that have a bit: those behind them are seen by none). Rows that see nothing, and rows without a request, give zeros.

    q and gate bf16 (M, Hq, D): projections, or views of one (strided rows and heads are read in place). scale: D ** -0.5 by
    default. step: of step_tables_ with as many rows, these heads and this cache's page size, without `keep`.
    """
    what = "paged_attention"
    if step.plan is None:
        raise ValueError(f"[{what}] the step has no plan: it was made with keep")
    if scale is None:
        scale = step.head_dim ** -0.5
    if q.is_cuda:
        out = _lib.native().paged(q, cache.keys, cache.values, cache.key_scales, cache.value_scales, step.block_table,
                                  step.request, step.plan, step.heads, step.kv_heads, step.head_dim, step.max_rows,
                                  step.page_size, float(scale), ancestors, gate)
        if type(out) is int:
            _lib.check(out, what)
        if out is not None:
            return out
    no_gradient(what, q=q, gate=gate, keys=cache.keys, values=cache.values, key_scales=cache.key_scales,
                value_scales=cache.value_scales)
    pages, bits = _check_step(what, cache, step, scale, ancestors)
    m, r, capacity, kv_heads, dim = step.request.shape[0], *step.block_table.shape, step.kv_heads, step.head_dim
    for name, t in (("q", q), ("gate", gate)):
        if t is None:
            continue
        if t.dtype != torch.bfloat16:
            raise ValueError(f"[{what}] {name} must be bfloat16, got {t.dtype}")
        if tuple(t.shape) != (m, step.heads, dim):
            raise ValueError(f"[{what}] {name} must be the step's ({m}, {step.heads}, {dim}), got {tuple(t.shape)}")
    dev = _check_plan(what, cache, step, ancestors, q, gate)
    q3 = _head_rows(q)
    g3 = None if gate is None else _head_rows(gate)
    ancestors = ancestors if ancestors is None else ancestors.contiguous()
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        size = lib.qmm4_paged_workspace(m, r, step.heads, kv_heads, dim, step.max_rows)
        _lib.check(min(size, 0), what)
        workspace = torch.empty(size, dtype=torch.uint8, device=dev)
        rc = lib.qmm4_paged_attention_bf16(q3.data_ptr(), *_strides(q3), cache.keys.data_ptr(), cache.values.data_ptr(),
                                           _ptr(cache.key_scales), _ptr(cache.value_scales), step.block_table.data_ptr(),
                                           step.request.data_ptr(), step.plan.data_ptr(), _ptr(ancestors), _ptr(g3),
                                           *((0, 0) if g3 is None else _strides(g3)), out.data_ptr(), workspace.data_ptr(),
                                           float(scale), m, r, step.heads, kv_heads, dim, pages, step.page_size, capacity,
                                           step.max_rows, bits, torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, what)
    return out


class CacheTables:
    """The tables that a batch's layers share: lengths, block_table, free_pages and free_count, as step_tables_ takes them,
    with all pages free."""

    def __init__(self, requests: int, capacity: int, pages: int, page_size: int, heads: int, kv_heads: int, head_dim: int,
                 device="cuda"):
        _check_page_size("CacheTables", page_size)
        _check_heads("CacheTables", heads, kv_heads)
        _check_dim("CacheTables", head_dim, False)
        self.page_size, self.heads, self.kv_heads, self.head_dim = page_size, heads, kv_heads, head_dim
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.block_table = torch.full((requests, capacity), -1, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)

    def cache(self, bits: int = 16) -> KVCache:
        """A layer's cache over these pages."""
        return KVCache.empty(self.free_pages.shape[0], self.page_size, self.kv_heads, self.head_dim, bits, self.lengths.device)

    def step(self, rows: torch.Tensor, total: int, base: torch.Tensor | None = None, keep: torch.Tensor | None = None,
             max_rows: int | None = None) -> CacheStep:
        """step_tables_ of these tables."""
        return step_tables_(self.lengths, self.block_table, self.free_pages, self.free_count, rows, total, self.page_size,
                            self.heads, self.kv_heads, self.head_dim, base=base, keep=keep, max_rows=max_rows)
