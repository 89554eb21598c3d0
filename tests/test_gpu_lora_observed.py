"""Adapters under autocast, function and dispatch modes, on every form of the projection (needs an MI355X): the result is
bf16 with the bits of the plain call, and where a library product computes the projection, what would see that product
and not the adapters' is refused."""

import contextlib

import pytest
import torch
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from mlx_tree_spec_amd import quantized_matmul_lora
from test_gpu_lora import check, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# (m, k, n, bits, group, whether a library product computes the projection)
FORMS = [(7, 256, 96, 4, 64, False), (9, 512, 96, 8, 32, False), (7, 96, 40, 4, 32, True), (300, 128, 77, 8, 64, False)]


class Functions(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class Operations(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class Wrapped(torch.Tensor):
    pass


def call(form):
    m, k, n, bits, group, _ = form
    args = inputs(m, k, n, 16, 3, m + n, bits, group)
    return args, lambda x=args[0]: quantized_matmul_lora(x, *args[1:], group_size=group, bits=bits)


@pytest.mark.parametrize("context", [lambda: torch.autocast("cuda", dtype=torch.float16), lambda: torch.autocast("cuda"),
                                     lambda: torch.autocast("cuda", dtype=torch.bfloat16), lambda: torch.device(DEV)],
                         ids=["float16", "default", "bfloat16", "device"])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_autocast_and_default_device(form, context):
    args, f = call(form)
    want = f()
    check(args, want, form[4], form[3], twice=form[5])
    with context():
        got = f()
    assert got.dtype == torch.bfloat16 and torch.equal(got, want)


@pytest.mark.parametrize("mode", [Functions, Operations])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_modes(form, mode):
    _, f = call(form)
    want = f()
    with mode(), (pytest.raises(ValueError, match="mode") if form[5] else contextlib.nullcontext()):
        got = f()
    assert form[5] or torch.equal(got, want)


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_subclasses(form):
    args, f = call(form)
    want = f()
    x = args[0].as_subclass(Wrapped)
    if form[5]:
        with pytest.raises(ValueError, match="subclass"):
            f(x)
    else:
        assert torch.equal(f(x).as_subclass(torch.Tensor), want)


class Counts(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(func.overloadpacket.__name__)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("form", [f for f in FORMS if not f[5]], ids=str)
def test_nothing_is_seen_in_part(form):
    _, f = call(form)
    with Counts() as mode:
        f()
    assert not {"linear", "mm", "addmm", "matmul"} & set(mode.seen)


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_modes_where_there_is_nothing_to_add(form):
    m, k, n, bits, group, _ = form
    x, w, s, b, la, lb, scale, ids = inputs(m, k, n, 16, 3, m + n, bits, group)
    with Operations():
        no_rows = quantized_matmul_lora(x[:0], w, s, b, la, lb, scale, ids[:0], group_size=group, bits=bits)
        no_adapters = quantized_matmul_lora(x, w, s, b, la[:0], lb[:0], scale[:0], ids, group_size=group, bits=bits)
    assert no_rows.shape == (0, n) and no_adapters.shape == (m, n)
