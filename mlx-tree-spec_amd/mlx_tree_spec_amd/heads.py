"""The step between the query / key projections and attention, backed by libqmm4.so (gfx950 HIP).

Mirrors the head norms and the rotation of src/mlx_tree_spec/tree_verify.py:311-328 (batch_attention), where a
batch's rows are tree nodes of several requests, each at a position of its own:

  qk_norm_rope(q, k, q_weight, k_weight, eps, positions, inv_freq, interleaved=False) -> (q', k')

one launch in place of two norms and two rotations. Tensors are bfloat16 on a HIP device; there is no CPU path,
and no gradient.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .lora import check_index, no_gradient, no_tangent
from .qmm import _check_device, aligned_contiguous

MAX_DIM = 512


def _head_rows(t: torch.Tensor) -> torch.Tensor:
    """t (..., heads, D) as [M, heads, D] with 16-byte aligned heads: a view where its strides allow, else a copy."""
    t3 = t.reshape(math.prod(t.shape[:-2]), *t.shape[-2:])
    ok = (t3.stride(2) == 1 or t3.shape[2] == 1) and t3.data_ptr() % 16 == 0
    for d in (0, 1):
        ok = ok and (t3.shape[d] == 1 or t3.stride(d) % 8 == 0 and t3.stride(d) >= 0)
    return t3 if ok else aligned_contiguous(t3.contiguous())


def _strides(t3: torch.Tensor) -> tuple[int, int]:
    return tuple(t3.stride(d) if t3.shape[d] > 1 else 0 for d in (0, 1))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                 positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False):
    """(q', k'): the RMS norm of every head of q and k (over its D values, with the weight of its side) and its
    rotation by the row's position, bf16, shaped like q and k.

    q bf16 (..., Hq, D), k bf16 (..., Hk, D) of one leading shape: projections, or views of one (strided rows and
    heads are read in place); q_weight, k_weight bf16 [D]; positions int32 or int64 of the leading shape; inv_freq
    fp32 or fp64 [P], 2 P <= D: pair i turns by positions * inv_freq[i]. Pairs are (i, i + P), or (2 i, 2 i + 1)
    when `interleaved` (MLX's traditional=True); values past 2 P are normed only. Norm and rotation are fp32 with
    angles reduced in fp64, so far positions turn by what inv_freq says, and the result is rounded once. q, k and
    inv_freq may not ask for a gradient; the weights, which a norm module holds as parameters, may and get none, as in
    add_rms_norm.
    """
    what = "qk_norm_rope"
    if q.is_cuda:
        out = _lib.native().rope(q, k, q_weight, k_weight, float(eps), positions, inv_freq, bool(interleaved))
        if type(out) is int:
            _lib.check(out, what)
        if out is not None:
            return out
    no_gradient(what, q=q, k=k, inv_freq=inv_freq)
    no_tangent(what, q_weight=q_weight, k_weight=k_weight)
    for name, t in (("q", q), ("k", k), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"[{what}] {name} must be bfloat16, got {t.dtype}")
    if q.dim() < 2 or k.dim() < 2 or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"[{what}] q {tuple(q.shape)} and k {tuple(k.shape)} must be (..., heads, D) of one leading "
                         "shape and D")
    d = q.shape[-1]
    if d % 8 or not 8 <= d <= MAX_DIM:
        raise ValueError(f"[{what}] heads of {d} values: D must be a multiple of 8, at most {MAX_DIM}")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if tuple(t.shape) != (d,):
            raise ValueError(f"[{what}] {name} must have shape ({d},), got {tuple(t.shape)}")
    if inv_freq.dtype not in (torch.float32, torch.float64) or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > d:
        raise ValueError(f"[{what}] inv_freq must be float32 or float64 of at most {d // 2} frequencies, got "
                         f"{inv_freq.dtype} {tuple(inv_freq.shape)}")
    positions = check_index(what, "positions", positions, q.shape[:-2])
    dev = _check_device(what, q, k, q_weight, k_weight, positions, inv_freq)
    q3, k3 = _head_rows(q), _head_rows(k)
    q_weight, k_weight, inv_freq = aligned_contiguous(q_weight), aligned_contiguous(k_weight), inv_freq.contiguous()
    q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
    k_out = torch.empty(k.shape, dtype=torch.bfloat16, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = lib.qmm4_qk_norm_rope_bf16(q3.data_ptr(), *_strides(q3), k3.data_ptr(), *_strides(k3), q_weight.data_ptr(),
                                        k_weight.data_ptr(), float(eps), positions.data_ptr(),
                                        positions.element_size() * 8, inv_freq.data_ptr(), inv_freq.element_size() * 8,
                                        q_out.data_ptr(), k_out.data_ptr(), q3.shape[0], q3.shape[1], k3.shape[1], d,
                                        inv_freq.shape[0], int(bool(interleaved)), stream)
    _lib.check(rc, what)
    return q_out, k_out
