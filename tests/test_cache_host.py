"""The paged cache's refusals, in Python and at the C ABI (CPU only: every call here ends before any GPU work)."""

import os
import re
import types

import pytest
import torch

from mlx_tree_spec_amd import CacheStep, CacheTables, KVCache, _lib, cached_attention, paged_attention, step_tables_, store_kv_

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, I32 = torch.bfloat16, torch.int32


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def test_library_exports_what_the_header_declares():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "qmm_cache.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(\w+)\s*\(", src, flags=re.M)))
    assert names == sorted(["qmm4_cache_plan_words", "qmm4_cache_step", "qmm4_store_kv_bf16", "qmm4_paged_workspace",
                            "qmm4_paged_attention_bf16"])
    lib = _lib.load()
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES


def table_args(r=3, capacity=4, pages=8, total=5):
    return dict(lengths=z(r, dtype=I32), block_table=z(r, capacity, dtype=I32), free_pages=z(pages, dtype=I32),
                free_count=z(1, dtype=I32), rows=z(r, dtype=I32), total=total, page_size=16, heads=8, kv_heads=2, head_dim=64)


@pytest.mark.parametrize("change,error,msg", [
    (dict(page_size=24), ValueError, "page_size=24"),
    (dict(page_size=8), ValueError, "page_size=8"),
    (dict(page_size=2048), ValueError, "page_size=2048"),
    (dict(heads=7), ValueError, "7 query heads"),
    (dict(heads=2048, kv_heads=2048), ValueError, "2048 query heads"),
    (dict(kv_heads=0), ValueError, "0 key heads"),
    (dict(head_dim=80), NotImplementedError, "heads of 80"),
    (dict(total=-1), ValueError, "-1 rows"),
    (dict(total=(1 << 22) + 1), ValueError, "up to 2048 requests and 4194304 rows"),
    (dict(max_rows=-1), ValueError, "at most -1"),
    (dict(lengths=z(3)), ValueError, "lengths must be torch.int32"),
    (dict(lengths=z(3, 1, dtype=I32)), ValueError, "1, 2 and 1 dimensions"),
    (dict(block_table=z(2, 4, dtype=I32)), ValueError, "block_table must be"),
    (dict(block_table=z(12, dtype=I32)), ValueError, "dimensions"),
    (dict(free_pages=z(8, dtype=torch.int64)), ValueError, "free_pages must be"),
    (dict(free_count=z(2, dtype=I32)), ValueError, "free_count must be"),
    (dict(rows=z(4, dtype=I32)), ValueError, "rows must be"),
    (dict(base=z(3, dtype=torch.int64)), ValueError, "base must be"),
    (dict(keep=z(4, dtype=torch.bool)), ValueError, "keep must be"),
    (dict(keep=z(5, dtype=I32)), ValueError, "keep must be"),
    (dict(lengths=z(2049, dtype=I32), block_table=z(2049, 4, dtype=I32), rows=z(2049, dtype=I32)), ValueError, "2049 requests"),
    (dict(), ValueError, "HIP device"),
])
def test_table_refusals(change, error, msg):
    with pytest.raises(error, match=msg):
        step_tables_(**{**table_args(), **change})


def test_tables_of_too_many_tokens():
    args = table_args()
    args["block_table"] = torch.empty(3, (1 << 22) + 1, dtype=I32, device="meta")
    with pytest.raises(ValueError, match="4194305 pages per request"):
        step_tables_(**args)
    args["block_table"], args["page_size"] = torch.empty(3, (1 << 20) + 1, dtype=I32, device="meta"), 1024
    with pytest.raises(ValueError, match="up to 2\\^30 tokens"):
        step_tables_(**args)
    with pytest.raises(ValueError, match="65537 rows with keep"):
        step_tables_(**{**table_args(total=65537), "keep": z(65537, dtype=torch.bool)})


def cache(pages=4, page=16, heads=2, dim=64, bits=16):
    return KVCache.empty(pages, page, heads, dim, bits, "cpu")


def test_empty_caches():
    c = cache(heads=3, dim=96, page=32)
    assert c.keys.shape == (4, 3, 12, 32, 8) and c.values.shape == (4, 3, 4, 96, 8) and c.keys.dtype == BF and c.key_scales is None
    c = cache(dim=128, bits=8)
    assert c.keys.shape == (4, 2, 8, 16, 16) and c.values.shape == (4, 2, 1, 128, 16) and c.values.dtype == torch.int8
    assert c.key_scales.shape == c.value_scales.shape == (4, 2, 16) and c.key_scales.dtype == torch.float32
    for kw, error in ((dict(dim=80), NotImplementedError), (dict(dim=96, bits=8), NotImplementedError),
                      (dict(bits=4), NotImplementedError), (dict(page=20), ValueError)):
        with pytest.raises(error):
            cache(**kw)
    t = CacheTables(3, 5, 7, 16, 8, 2, 64, "cpu")
    assert t.free_pages.tolist() == [6, 5, 4, 3, 2, 1, 0] and t.free_count.item() == 7 and (t.block_table == -1).all()
    assert t.cache(8).keys.shape == (7, 2, 4, 16, 16)


def bad_caches():
    c, c8 = cache(), cache(bits=8)
    odd = torch.empty(c.keys.numel() + 1, dtype=BF)[1:].reshape(c.keys.shape)
    return [
        (c._replace(keys=c.keys.float()), "both be bfloat16 or int8"),
        (c._replace(values=c8.values), "both be bfloat16 or int8"),
        (c._replace(keys=c.keys[0]), "must be \\[pages"),
        (KVCache(c8.keys.to(BF), c8.values.to(BF)), "must be \\[pages"),
        (c._replace(values=z(4, 2, 2, 128, 8)), "values must be"),
        (c._replace(key_scales=c8.key_scales), "scales"),
        (c8._replace(value_scales=None), "scales"),
        (c8._replace(key_scales=c8.key_scales[:3]), "key_scales must be"),
        (c8._replace(key_scales=c8.key_scales.double()), "key_scales must be"),
        (c._replace(keys=odd), "in place"),
        (c._replace(keys=c.keys.transpose(0, 1).contiguous().transpose(0, 1)), "in place"),
    ]


def step(m=5, heads=8, kv_heads=2, dim=64, page=16, plan=True):
    i = z(m, dtype=I32)
    return CacheStep(i, i, i, z(40, dtype=I32) if plan else None, z(3, 4, dtype=I32), page, heads, kv_heads, dim, m)


def test_cache_refusals():
    for bad, msg in bad_caches():
        with pytest.raises(ValueError, match=msg):
            store_kv_(z(5, 2, 64), z(5, 2, 64), bad, z(5, dtype=I32))
        with pytest.raises(ValueError, match=msg):
            paged_attention(z(5, 8, 64), bad, step())


@pytest.mark.parametrize("change,msg", [
    (dict(k=z(5, 2, 64, dtype=torch.float16)), "k must be bfloat16"),
    (dict(v=z(5, 2, 64, dtype=torch.float32)), "v must be bfloat16"),
    (dict(k=z(5, 3, 64)), "k must be \\(rows, 2, 64\\)"),
    (dict(v=z(4, 2, 64)), "v must be"),
    (dict(k=z(5, 128)), "k must be"),
    (dict(slots=z(4, dtype=I32)), "slots must be"),
    (dict(slots=z(5, dtype=torch.int64)), "slots must be"),
    (dict(k=z(5, 2, 64).requires_grad_()), "requires a gradient"),
    (dict(), "HIP device"),
])
def test_store_refusals(change, msg):
    args = {**dict(k=z(5, 2, 64), v=z(5, 2, 64), cache=cache(), slots=z(5, dtype=I32)), **change}
    with pytest.raises(ValueError, match=msg):
        store_kv_(**args)


@pytest.mark.parametrize("change,msg", [
    (dict(q=z(5, 8, 64, dtype=torch.float16)), "q must be bfloat16"),
    (dict(q=z(4, 8, 64)), "q must be the step's"),
    (dict(q=z(5, 6, 64)), "q must be the step's"),
    (dict(gate=z(5, 8, 32)), "gate must be the step's"),
    (dict(gate=z(5, 8, 64, dtype=torch.float32)), "gate must be bfloat16"),
    (dict(step=step(page=32)), "the step was made for"),
    (dict(step=step(kv_heads=4)), "the step was made for"),
    (dict(step=step(dim=128)), "the step was made for"),
    (dict(step=step(plan=False)), "made with keep"),
    (dict(scale=float("inf")), "must be finite"),
    (dict(ancestors=z(5, dtype=I32)), "ancestors must be"),
    (dict(ancestors=z(4, dtype=torch.int64)), "ancestors must be"),
    (dict(q=z(5, 8, 64).requires_grad_()), "requires a gradient"),
    (dict(gate=z(5, 8, 64).requires_grad_()), "requires a gradient"),
    (dict(), "HIP device"),
])
def test_attention_refusals(change, msg):
    args = {**dict(q=z(5, 8, 64), cache=cache(), step=step()), **change}
    with pytest.raises(ValueError, match=msg):
        paged_attention(**args)


@pytest.mark.parametrize("change,msg", [
    (dict(block_table=z(12, dtype=I32)), "block_table must have 2 dimensions"),
    (dict(block_table=z(3, 4, dtype=torch.int64)), "block_table must be"),
    (dict(block_table=z(3, 8, dtype=I32)[:, :4]), "block_table must be contiguous"),
    (dict(request=z(10, dtype=I32)[::2]), "request must be contiguous"),
    (dict(request=z(5, dtype=torch.int64)), "request must be"),
    (dict(plan=z(40)), "plan must be"),
    (dict(plan=z(80, dtype=I32)[::2]), "plan must be contiguous"),
])
def test_attention_of_a_changed_step(change, msg):
    with pytest.raises(ValueError, match=msg):
        paged_attention(z(5, 8, 64), cache(), step()._replace(**change))


def test_cached_attention_wants_a_plan():
    """A step of kept rows is refused before anything is computed or stored."""
    layer = types.SimpleNamespace(heads=8, kv_heads=2, head_dim=64)
    with pytest.raises(ValueError, match="no plan"):
        cached_attention(z(5, 32), layer, cache(), step(plan=False))


P = 0x10000


def c_step(**kw):
    a = dict(lengths=P, table=P, free=P, count=P, rows=P, base=None, keep=None, slots=P, positions=P, request=P, plan=P, R=3,
             capacity=4, pages=8, total=5, max_rows=5, page=16, heads=8, kv=2, dim=64)
    a.update(kw)
    return _lib.load().qmm4_cache_step(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(page=17), "page_size=17"), (dict(page=0), "page_size=0"), (dict(pages=-1), "-1 pages"),
    (dict(capacity=1 << 40), "up to 2^30"), (dict(capacity=(1 << 22) + 1), "up to 2^22"),
    (dict(keep=P, total=65537), "65537 rows with keep"),
    (dict(pages=(1 << 26) + 1), "up to 2^30"), (dict(heads=9), "9 query heads"),
    (dict(R=2049), "2049 requests"), (dict(total=-2), "-2 rows"), (dict(max_rows=-1), "at most -1"), (dict(lengths=None), "null"),
    (dict(table=None), "null"), (dict(count=None), "null"), (dict(free=None), "null"), (dict(slots=None), "null"),
    (dict(rows=P + 2), "aligned"), (dict(plan=P + 1), "aligned")])
def test_c_step_refusals(kw, msg):
    assert c_step(**kw) == _lib.QMM4_ERR_INVALID and msg in _lib.last_error()


def c_store(**kw):
    a = dict(k=P, kr=128, kh=64, v=P, vr=128, vh=64, slots=P, keys=P, values=P, ks=None, vs=None, M=5, H=2, D=64, pages=4, page=16,
             bits=16)
    a.update(kw)
    return _lib.load().qmm4_store_kv_bf16(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(bits=4), _lib.QMM4_ERR_UNSUPPORTED, "bits=4"), (dict(D=80), _lib.QMM4_ERR_UNSUPPORTED, "heads of 80"),
    (dict(D=96, bits=8, ks=P, vs=P), _lib.QMM4_ERR_UNSUPPORTED, "heads of 96"),
    (dict(bits=8), _lib.QMM4_ERR_INVALID, "scales"), (dict(ks=P, vs=P), _lib.QMM4_ERR_INVALID, "scales"),
    (dict(H=0), _lib.QMM4_ERR_INVALID, "0 key heads"), (dict(M=-1), _lib.QMM4_ERR_INVALID, "-1 rows"),
    (dict(k=None), _lib.QMM4_ERR_INVALID, "null"), (dict(slots=None), _lib.QMM4_ERR_INVALID, "null"),
    (dict(k=P + 2), _lib.QMM4_ERR_INVALID, "k must be 16-byte"), (dict(vr=12), _lib.QMM4_ERR_INVALID, "v must be 16-byte"),
    (dict(keys=P + 8), _lib.QMM4_ERR_INVALID, "16-byte"), (dict(M=0, k=None), _lib.QMM4_OK, ""), (dict(pages=0), _lib.QMM4_OK, "")])
def test_c_store_refusals(kw, code, msg):
    assert c_store(**kw) == code and msg in _lib.last_error()


def c_attention(**kw):
    a = dict(q=P, qr=512, qh=64, keys=P, values=P, ks=None, vs=None, table=P, request=P, plan=P, ancestors=None, gate=None, gr=0, gh=0,
             out=P, ws=P, scale=1.0, M=5, R=3, Hq=8, Hk=2, D=64, pages=4, page=16, capacity=4, max_rows=5, bits=16)
    a.update(kw)
    return _lib.load().qmm4_paged_attention_bf16(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(bits=32), _lib.QMM4_ERR_UNSUPPORTED, "bits=32"), (dict(D=512), _lib.QMM4_ERR_UNSUPPORTED, "heads of 512"),
    (dict(Hk=3), _lib.QMM4_ERR_INVALID, "multiple"), (dict(scale=float("nan")), _lib.QMM4_ERR_INVALID, "finite"),
    (dict(plan=None), _lib.QMM4_ERR_INVALID, "null"), (dict(out=None), _lib.QMM4_ERR_INVALID, "null"),
    (dict(q=P + 4), _lib.QMM4_ERR_INVALID, "q must be"), (dict(gate=P, gh=4), _lib.QMM4_ERR_INVALID, "gate must be"),
    (dict(ws=P + 8), _lib.QMM4_ERR_INVALID, "16-byte"), (dict(ancestors=P + 4), _lib.QMM4_ERR_INVALID, "aligned"),
    (dict(pages=0), _lib.QMM4_ERR_INVALID, "without pages"), (dict(capacity=0), _lib.QMM4_ERR_INVALID, "without pages"),
    (dict(M=0, q=None), _lib.QMM4_OK, "")])
def test_c_attention_refusals(kw, code, msg):
    assert c_attention(**kw) == code and msg in _lib.last_error()
