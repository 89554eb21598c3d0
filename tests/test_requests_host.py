"""The per-request operators' refusals, in Python and at the C ABI (CPU only: every call here ends before any GPU
work)."""

import os
import re

import pytest
import torch

from mlx_tree_spec_amd import _lib, qk_norm_rope, quantized_matmul_lora, sample, stack_adapters

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16


def test_library_exports_what_the_header_declares():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "qmm_requests.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(\w+)\s*\(", src, flags=re.M)))
    assert names == sorted(["qmm4_lora_workspace", "qmm4_lora_add_bf16", "qmm4_affine_lora_bf16", "qmm4_qk_norm_rope_bf16",
                            "qmm4_sample_workspace", "qmm4_sample_bf16"])
    lib = _lib.load()
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES


def lora_args(m=4, k=128, n=32, rank=8, count=2):
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)  # noqa: E731
    return dict(x=z(m, k), w=z(n, k // 8, dtype=torch.int32), scales=z(n, k // 64), biases=z(n, k // 64),
                lora_a=z(count, rank, k), lora_b=z(count, n, rank), lora_scale=z(count, dtype=torch.float32),
                adapters=z(m, dtype=torch.int32))


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("change,error,msg", [
    (dict(x=z(4, 128, dtype=torch.float16)), ValueError, "x must be bfloat16"),
    (dict(x=z(4, 64)), ValueError, "does not match"),
    (dict(lora_a=z(2, 8, 64)), ValueError, "do not match"),
    (dict(lora_a=z(8, 128)), ValueError, "must be"),
    (dict(lora_b=z(2, 32, 16)), ValueError, "do not match"),
    (dict(lora_b=z(3, 32, 8)), ValueError, "do not match"),
    (dict(lora_a=z(2, 4, 128), lora_b=z(2, 32, 4)), ValueError, "rank 4"),
    (dict(lora_a=z(2, 264, 128), lora_b=z(2, 32, 264)), ValueError, "rank 264"),
    (dict(lora_a=z(2, 0, 128), lora_b=z(2, 32, 0)), ValueError, "rank 0"),
    (dict(lora_a=z(2, 8, 128, dtype=torch.float32)), ValueError, "lora_a must be bfloat16"),
    (dict(lora_scale=z(2)), ValueError, "lora_scale"),
    (dict(lora_scale=z(3, dtype=torch.float32)), ValueError, "lora_scale"),
    (dict(adapters=z(4, dtype=torch.int16)), ValueError, "int32 or int64"),
    (dict(adapters=z(5, dtype=torch.int32)), ValueError, "one value per row"),
    (dict(adapters=z(4, 1, dtype=torch.int32)), ValueError, "one value per row"),
    (dict(scales=None), ValueError, "scales and biases"),
    (dict(bits=3), NotImplementedError, "bits=3"),
    (dict(transpose=False), NotImplementedError, "transpose"),
    (dict(mode="other"), NotImplementedError, "mode"),
    (dict(), ValueError, "no CPU path"),
])
def test_lora_refuses(change, error, msg):
    with pytest.raises(error, match=msg):
        quantized_matmul_lora(**{**lora_args(), **change})


@pytest.mark.parametrize("name", ["x", "lora_a", "lora_b", "lora_scale"])
def test_lora_refuses_gradients(name):
    args = lora_args()
    args[name].requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        quantized_matmul_lora(**args)
    with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
        quantized_matmul_lora(**args)


def test_stack_adapters_refuses():
    with pytest.raises(ValueError, match="no adapters"):
        stack_adapters([])
    with pytest.raises(ValueError, match="adapter 1"):
        stack_adapters([(z(4, 64), z(32, 4), 1.0), (z(4, 64), z(32, 5), 1.0)])
    with pytest.raises(ValueError, match="largest rank"):
        stack_adapters([(z(257, 64), z(32, 257), 1.0)])


def rope_args(m=3, hq=4, hk=2, d=64, p=32):
    return dict(q=z(m, hq, d), k=z(m, hk, d), q_weight=z(d), k_weight=z(d), eps=1e-6,
                positions=z(m, dtype=torch.int32), inv_freq=z(p, dtype=torch.float32))


@pytest.mark.parametrize("change,msg", [
    (dict(q=z(3, 4, 64, dtype=torch.float32)), "q must be bfloat16"),
    (dict(k_weight=z(64, dtype=torch.float32)), "k_weight must be bfloat16"),
    (dict(k=z(2, 2, 64)), "one leading shape"),
    (dict(k=z(3, 2, 128)), "one leading shape"),
    (dict(q=z(64), k=z(64)), "one leading shape"),
    (dict(q=z(3, 4, 60), k=z(3, 2, 60)), "multiple of 8"),
    (dict(q=z(3, 4, 520), k=z(3, 2, 520)), "at most 512"),
    (dict(q_weight=z(32)), "q_weight must have shape"),
    (dict(inv_freq=z(33, dtype=torch.float32)), "at most 32"),
    (dict(inv_freq=z(32)), "float32 or float64"),
    (dict(inv_freq=z(4, 8, dtype=torch.float32)), "inv_freq"),
    (dict(positions=z(4, dtype=torch.int32)), "one value per row"),
    (dict(positions=z(3, dtype=torch.float32)), "int32 or int64"),
    (dict(), "no CPU path"),
])
def test_rope_refuses(change, msg):
    with pytest.raises(ValueError, match=msg):
        qk_norm_rope(**{**rope_args(), **change})


def test_rope_refuses_gradients_of_its_heads():
    args = rope_args()
    args["q_weight"].requires_grad_(True)  # a norm module's weight: no gradient flows, as in add_rms_norm
    with pytest.raises(ValueError, match="no CPU path"):
        qk_norm_rope(**args)
    args["k"].requires_grad_(True)
    with pytest.raises(ValueError, match="k requires a gradient"):
        qk_norm_rope(**args)


@pytest.mark.parametrize("change,msg", [
    (dict(logits=z(4, 100, dtype=torch.float32)), "logits must be bfloat16"),
    (dict(logits=z(4, 0)), "1 <= V"),
    (dict(uniform=z(4)), "uniform must be float32"),
    (dict(uniform=z(5, dtype=torch.float32)), "uniform must be float32 of shape"),
    (dict(temperature=-0.5), "temperature=-0.5"),
    (dict(temperature=float("nan")), "temperature=nan"),
    (dict(temperature=float("inf")), "temperature=inf"),
    (dict(top_k=-1), "top_k=-1"),
    (dict(top_p=0.0), "top_p=0.0"),
    (dict(top_p=1.5), "top_p=1.5"),
    (dict(min_p=-0.1), "min_p=-0.1"),
    (dict(min_p=1.5), "min_p=1.5"),
    (dict(temperature=z(4)), "temperature must be a number or torch.float32"),
    (dict(top_k=z(4, dtype=torch.int64)), "top_k must be a number or torch.int32"),
    (dict(top_p=z(5, dtype=torch.float32)), "top_p must be"),
    (dict(), "no CPU path"),
])
def test_sample_refuses(change, msg):
    args = dict(logits=z(4, 100), uniform=z(4, dtype=torch.float32))
    with pytest.raises(ValueError, match=msg):
        sample(**{**args, **change})


def test_sample_refuses_gradients():
    with pytest.raises(ValueError, match="gradient"):
        sample(z(4, 100).requires_grad_(True), z(4, dtype=torch.float32))


P = 0x10000


@pytest.mark.parametrize("kw,code,msg", [
    (dict(ab=16), _lib.QMM4_ERR_UNSUPPORTED, "16 bits"),
    (dict(M=-1), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(K=12), _lib.QMM4_ERR_INVALID, "multiple of 8"),
    (dict(L=1 << 31), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(R=4), _lib.QMM4_ERR_INVALID, "R=4"),
    (dict(R=264), _lib.QMM4_ERR_INVALID, "R=264"),
    (dict(x=0), _lib.QMM4_ERR_INVALID, "null pointer"),
    (dict(x=P + 2), _lib.QMM4_ERR_INVALID, "16-byte aligned"),
    (dict(ws=P + 4), _lib.QMM4_ERR_INVALID, "16-byte aligned"),
    (dict(y=P + 1), _lib.QMM4_ERR_INVALID, "aligned to their elements"),
    (dict(M=(1 << 26) + 1), _lib.QMM4_ERR_INVALID, "2^26 rows"),
    (dict(M=0, x=0), _lib.QMM4_OK, ""),
    (dict(L=0, x=0), _lib.QMM4_OK, ""),
    (dict(N=0, x=0), _lib.QMM4_OK, ""),
])
def test_lora_add_at_the_c_abi(kw, code, msg):
    a = dict(x=P, ab=32, y=P, ws=P, M=4, N=32, K=128, L=2, R=8)
    a.update(kw)
    rc = _lib.load().qmm4_lora_add_bf16(a["x"], P, P, P, P, a["ab"], a["y"], a["ws"], a["M"], a["N"], a["K"], a["L"],
                                        a["R"], None)
    assert rc == code and msg in _lib.last_error()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(bits=3), _lib.QMM4_ERR_UNSUPPORTED, "bits=3"),
    (dict(gs=48), _lib.QMM4_ERR_UNSUPPORTED, "group_size=48"),
    (dict(K=96), _lib.QMM4_ERR_INVALID, "K=96"),
    (dict(M=1 << 26), _lib.QMM4_ERR_INVALID, "exceeds 4 GiB"),
    (dict(R=12), _lib.QMM4_ERR_INVALID, "R=12"),
    (dict(M=0), _lib.QMM4_OK, ""),
])
def test_affine_lora_at_the_c_abi(kw, code, msg):
    a = dict(M=4, N=32, K=128, L=2, R=8, gs=64, bits=4)
    a.update(kw)
    rc = _lib.load().qmm4_affine_lora_bf16(P, P, P, P, P, P, P, P, 32, P, P, a["M"], a["N"], a["K"], a["L"], a["R"],
                                           a["gs"], a["bits"], 1, None)
    assert rc == code and msg in _lib.last_error()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(pb=16), _lib.QMM4_ERR_UNSUPPORTED, "positions of 16 bits"),
    (dict(fb=16), _lib.QMM4_ERR_UNSUPPORTED, "inv_freq of 16 bits"),
    (dict(M=-1), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(Hq=70000), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(D=60), _lib.QMM4_ERR_INVALID, "D=60"),
    (dict(D=520), _lib.QMM4_ERR_INVALID, "D=520"),
    (dict(P=33), _lib.QMM4_ERR_INVALID, "P=33"),
    (dict(P=-1), _lib.QMM4_ERR_INVALID, "P=-1"),
    (dict(eps=-1.0), _lib.QMM4_ERR_INVALID, "eps"),
    (dict(eps=float("nan")), _lib.QMM4_ERR_INVALID, "eps"),
    (dict(eps=float("inf")), _lib.QMM4_ERR_INVALID, "eps"),
    (dict(q=0), _lib.QMM4_ERR_INVALID, "null pointer"),
    (dict(q=P + 8), _lib.QMM4_ERR_INVALID, "16-byte aligned"),
    (dict(row=100), _lib.QMM4_ERR_INVALID, "multiples of 8"),
    (dict(pos=P + 2), _lib.QMM4_ERR_INVALID, "aligned to their elements"),
    (dict(M=0, q=0), _lib.QMM4_OK, ""),
    (dict(Hq=0, Hk=0, q=0), _lib.QMM4_OK, ""),
])
def test_rope_at_the_c_abi(kw, code, msg):
    a = dict(q=P, row=256, pos=P, pb=32, fb=32, M=4, Hq=4, Hk=2, D=64, P=32, eps=1e-6)
    a.update(kw)
    rc = _lib.load().qmm4_qk_norm_rope_bf16(a["q"], a["row"], 64, P, 128, 64, P, P, a["eps"], a["pos"], a["pb"], P, a["fb"],
                                            P, P, a["M"], a["Hq"], a["Hk"], a["D"], a["P"], 0, None)
    assert rc == code and msg in _lib.last_error()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(M=-1), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(M=(1 << 20) + 1), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(V=0), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(V=(1 << 24) + 1), _lib.QMM4_ERR_INVALID, "invalid shape"),
    (dict(stride=99), _lib.QMM4_ERR_INVALID, "row_stride=99"),
    (dict(logits=0), _lib.QMM4_ERR_INVALID, "null pointer"),
    (dict(logits=P + 1), _lib.QMM4_ERR_INVALID, "aligned"),
    (dict(ws=P + 8), _lib.QMM4_ERR_INVALID, "aligned"),
    (dict(M=0, logits=0), _lib.QMM4_OK, ""),
])
def test_sample_at_the_c_abi(kw, code, msg):
    a = dict(logits=P, M=2, V=100, stride=100, ws=P)
    a.update(kw)
    rc = _lib.load().qmm4_sample_bf16(a["logits"], a["M"], a["V"], a["stride"], P, None, 1.0, None, 0, None, 1.0, None, 0.0,
                                      P, P, a["ws"], None)
    assert rc == code and msg in _lib.last_error()
