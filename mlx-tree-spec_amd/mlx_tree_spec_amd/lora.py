"""Low-rank adapters of many requests beside a shared quantized projection, backed by libqmm4.so.

A batched step concatenates several requests' rows (src/mlx_tree_spec/tree_verify.py:414-447) and runs each
projection once over all of them; requests may carry adapters of their own:

  quantized_matmul_lora(x, w, scales, biases, lora_a, lora_b, lora_scale, adapters, ...)
      y[m] = x[m] @ dequant(w).T + lora_scale[a] * (x[m] @ lora_a[a].T) @ lora_b[a].T,  a = adapters[m]
  stack_adapters([(A, B, scale), ...]) -> (lora_a, lora_b, lora_scale), the tables it reads
  LoRALinear(base, lora_a, lora_b, lora_scale): a QuantizedLinear with such tables, called with (x, adapters)

The reference has no adapters; the projection is packed_linear._call's (packed_linear.py:83-104). Tensors are
bfloat16 on a HIP device; there is no CPU path, and no gradient.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib
from .packed_linear import STATS, QuantizedLinear
from .qmm import (GENERAL_BITS, GENERAL_GROUP_SIZES, _check_device, _check_format, _check_weights,
                  _general_shape_ok, _watched, aligned_contiguous, quantized_matmul)

MAX_RANK = 256
_INDEX_DTYPES = (torch.int32, torch.int64)


def no_tangent(what: str, **inputs) -> None:
    """Raises where an input carries a tangent of forward mode, which the kernels would drop unseen."""
    if forward_ad._current_level >= 0:
        for name, t in inputs.items():
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"[{what}] {name} carries a tangent, which this operator does not have; detach the tensor")


def no_gradient(what: str, **inputs) -> None:
    """Raises where a gradient of an input is asked for, in either mode: the kernels have none, and would cut it
    unseen. (What is no tensor is passed over.)"""
    no_tangent(what, **inputs)
    if torch.is_grad_enabled():
        for name, t in inputs.items():
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise ValueError(f"[{what}] {name} requires a gradient, which this operator does not have; "
                                 "call it under torch.no_grad() or detach the tensor")


def check_index(what: str, name: str, t: torch.Tensor, shape: torch.Size) -> torch.Tensor:
    """An int32 / int64 tensor of one value per row, contiguous."""
    if t.dtype not in _INDEX_DTYPES:
        raise ValueError(f"[{what}] {name} must be int32 or int64, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"[{what}] {name} must have one value per row, shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _check_adapters(what: str, lora_a: torch.Tensor, lora_b: torch.Tensor, lora_scale: torch.Tensor, n: int,
                    k: int) -> None:
    if lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError(f"[{what}] lora_a and lora_b must be [adapters, rank, {k}] and [adapters, {n}, rank], got "
                         f"{tuple(lora_a.shape)} and {tuple(lora_b.shape)}")
    count, rank, _ = lora_a.shape
    if tuple(lora_a.shape) != (count, rank, k) or tuple(lora_b.shape) != (count, n, rank):
        raise ValueError(f"[{what}] lora_a {tuple(lora_a.shape)} and lora_b {tuple(lora_b.shape)} do not match "
                         f"[adapters, rank, {k}] and [adapters, {n}, rank]")
    if rank % 8 or not 8 <= rank <= MAX_RANK:
        raise ValueError(f"[{what}] rank {rank} must be a multiple of 8 from 8 to {MAX_RANK} (stack_adapters pads)")
    for name, t in (("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"[{what}] {name} must be bfloat16, got {t.dtype}")
    if lora_scale.dtype != torch.float32 or tuple(lora_scale.shape) != (count,):
        raise ValueError(f"[{what}] lora_scale must be float32 of shape ({count},), got {lora_scale.dtype} "
                         f"{tuple(lora_scale.shape)}")


def _native_lora(x, w, scales, biases, lora_a, lora_b, lora_scale, adapters, transpose, group_size, bits, mode):
    """The usual call in native code (the output), or None for the general form below."""
    if transpose is not True or mode != "affine" or not x.is_cuda or x.dim() < 1 or w.dim() != 2:
        return None
    k, n = x.shape[-1], w.shape[0]
    general = bits != 4 or group_size != 64 or k % 128 != 0 or n % 16 != 0
    if general and (bits not in GENERAL_BITS or group_size not in GENERAL_GROUP_SIZES or k == 0
                    or not _general_shape_ok(x, x.numel() // k, n, k, bits)):
        return None
    y = _lib.native().lora(x, w, scales, biases, lora_a, lora_b, lora_scale, adapters, group_size, bits)
    if type(y) is int:
        _lib.check(y, "quantized_matmul_lora")
    return y


def _library_product(x2: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, group_size: int,
                     bits: int) -> torch.Tensor:
    """The projection at the sizes at which quantized_matmul dequantizes and multiplies, in bf16 under autocast too: the
    adapters are added to its words."""
    if not torch.is_autocast_enabled("cuda"):
        return quantized_matmul(x2, w, scales, biases, group_size=group_size, bits=bits)
    with torch.autocast("cuda", enabled=False):
        return quantized_matmul(x2, w, scales, biases, group_size=group_size, bits=bits)


def quantized_matmul_lora(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                          lora_a: torch.Tensor, lora_b: torch.Tensor, lora_scale: torch.Tensor,
                          adapters: torch.Tensor, transpose: bool = True, group_size: int = 64, bits: int = 4,
                          mode: str = "affine") -> torch.Tensor:
    """quantized_matmul with each row's low-rank adapter: bf16 (..., N), under autocast to another type too,

        y[m] = x[m] @ dequant(w).T + lora_scale[a] * (x[m] @ lora_a[a].T) @ lora_b[a].T,   a = adapters[m].

    x bf16 (..., K); w, scales, biases as in quantized_matmul, in any format that takes; lora_a bf16 [L, R, K],
    lora_b bf16 [L, N, R], lora_scale fp32 [L] (R a multiple of 8, up to 256); adapters int32 or int64 of x's
    leading shape. A row whose adapter lies outside 0 .. L - 1 (-1, say) has the projection alone, with its bits.
    Both products are summed in fp32 and rounded once (twice at the sizes and formats for which quantized_matmul
    dequantizes and multiplies); x @ lora_a.T is kept to 2^-18 of its value in between. What is not finite in an
    adapter reaches the rows that use it, as the formula has it, and no other. Nothing sees the call as torch operations;
    where a library product computes the projection it is refused under a function or dispatch mode or for a tensor
    subclass, which would see that product alone.
    """
    what = "quantized_matmul_lora"
    y = _native_lora(x, w, scales, biases, lora_a, lora_b, lora_scale, adapters, transpose, group_size, bits, mode)
    if y is not None:
        return y
    _check_format(group_size, bits, transpose, mode, general=True)
    no_gradient(what, x=x, scales=scales, biases=biases, lora_a=lora_a, lora_b=lora_b, lora_scale=lora_scale)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"[{what}] x must be bfloat16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"[{what}] x must have at least one dimension")
    k = x.shape[-1]
    if k % group_size:
        raise ValueError(f"[{what}] x.shape[-1]={k} must be a multiple of group_size={group_size}")
    n, _ = _check_weights(w, scales, biases, k, group_size, bits, what)
    _check_adapters(what, lora_a, lora_b, lora_scale, n, k)
    adapters = check_index(what, "adapters", adapters, x.shape[:-1])
    dev = _check_device(what, x, w, scales, biases, lora_a, lora_b, lora_scale, adapters)
    x2 = aligned_contiguous(x.reshape(-1, k))
    lora_a, lora_b, lora_scale = aligned_contiguous(lora_a), aligned_contiguous(lora_b), lora_scale.contiguous()
    m, (count, rank) = x2.shape[0], lora_a.shape[:2]
    lib = _lib.load()
    workspace = torch.empty((m, rank), dtype=torch.int32, device=dev)
    packed = bits == 4 and group_size == 64 and k % 128 == 0 and n % 16 == 0
    fused = packed or _general_shape_ok(x, m, n, k, bits)
    w, scales, biases = aligned_contiguous(w), aligned_contiguous(scales), aligned_contiguous(biases)
    if fused:
        y = torch.empty((*x.shape[:-1], n), dtype=torch.bfloat16, device=dev)
    else:
        if m * n * count > 0 and _watched(x):
            raise ValueError(f"[{what}] at this size and format a library product computes the projection: a tensor "
                             "subclass, a function mode or a dispatch mode would see it without the adapters' part")
        y = _library_product(x2, w, scales, biases, group_size, bits).reshape(*x.shape[:-1], n)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        lora = (lora_a.data_ptr(), lora_b.data_ptr(), lora_scale.data_ptr(), adapters.data_ptr(),
                adapters.element_size() * 8, y.data_ptr(), workspace.data_ptr(), m, n, k, count, rank)
        if fused:
            rc = lib.qmm4_affine_lora_bf16(x2.data_ptr(), w.data_ptr(), scales.data_ptr(), biases.data_ptr(), *lora,
                                           group_size, bits, 1, stream)
        else:
            rc = lib.qmm4_lora_add_bf16(x2.data_ptr(), *lora, stream)
    _lib.check(rc, what)
    return y


def stack_adapters(adapters, device=None):
    """(lora_a [L, R, K], lora_b [L, N, R], lora_scale [L]) of a list of (A [r, K], B [N, r], scale): the ranks
    padded with zeros to the largest, rounded up to a multiple of 8."""
    if not adapters:
        raise ValueError("[stack_adapters] no adapters")
    k, n = adapters[0][0].shape[1], adapters[0][1].shape[0]
    for i, (a, b, _) in enumerate(adapters):
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != k or b.shape[0] != n or a.shape[0] != b.shape[1]:
            raise ValueError(f"[stack_adapters] adapter {i}: A {tuple(a.shape)} and B {tuple(b.shape)} do not match "
                             f"[r, {k}] and [{n}, r]")
    rank = (max(a.shape[0] for a, _, _ in adapters) + 7) // 8 * 8
    if not 8 <= rank <= MAX_RANK:
        raise ValueError(f"[stack_adapters] the largest rank must be from 1 to {MAX_RANK}")
    device = adapters[0][0].device if device is None else device
    lora_a = torch.zeros((len(adapters), rank, k), dtype=torch.bfloat16, device=device)
    lora_b = torch.zeros((len(adapters), n, rank), dtype=torch.bfloat16, device=device)
    with torch.no_grad():
        for i, (a, b, _) in enumerate(adapters):
            lora_a[i, :a.shape[0]].copy_(a)
            lora_b[i, :, :b.shape[1]].copy_(b)
    return lora_a, lora_b, torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=device)


class LoRALinear(torch.nn.Module):
    """A QuantizedLinear with the adapters of several requests: forward(x, adapters) = quantized_matmul_lora on
    its weights (+ its bias); adapters None: the base layer alone."""

    def __init__(self, base: QuantizedLinear, lora_a: torch.Tensor, lora_b: torch.Tensor, lora_scale: torch.Tensor):
        super().__init__()
        _check_adapters("LoRALinear", lora_a, lora_b, lora_scale, base.output_dims, base.input_dims)
        self.base = base
        self.register_buffer("lora_a", lora_a)
        self.register_buffer("lora_b", lora_b)
        self.register_buffer("lora_scale", lora_scale)

    def forward(self, x: torch.Tensor, adapters: torch.Tensor | None = None) -> torch.Tensor:
        base = self.base
        if adapters is None:
            return base(x)
        STATS["lora"] += 1
        y = quantized_matmul_lora(x, base.weight, base.scales, base.biases, self.lora_a, self.lora_b,
                                  self.lora_scale, adapters, group_size=base.group_size, bits=base.bits,
                                  mode=base.mode)
        return y + base.bias if base.bias is not None else y
