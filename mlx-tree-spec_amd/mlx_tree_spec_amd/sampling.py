"""Tokens from the vocabulary head's logits, backed by libqmm4.so (gfx950 HIP).

  sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> (tokens, logprobs)

The step behind the vocabulary head of a batched forward (src/mlx_tree_spec/tree_verify.py:447, whose tokens the
reference takes by argmax or mlx-lm's samplers), each row with the settings of its request. The random numbers are
an input: the same inputs give the same tokens. Logits are bfloat16 on a HIP device, as quantized_matmul writes
them; there is no CPU path, and no gradient.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .lora import no_gradient
from .qmm import _check_device

MAX_VOCAB = 1 << 24


def _setting(what: str, name: str, value, dtype: torch.dtype, shape: torch.Size, valid):
    """(tensor or None, value): one value per row, or one for all."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.shape != shape:
            raise ValueError(f"[{what}] {name} must be a number or {dtype} of shape {tuple(shape)}, got {value.dtype} "
                             f"{tuple(value.shape)}")
        return value.contiguous(), 0
    if not valid(value):
        raise ValueError(f"[{what}] {name}={value} is out of range")
    return None, value


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens int64, logprobs fp32) of the leading shape of logits (..., V).

    With w = exp((l - max l) / temperature), in the order of falling logits (equal ones by index): kept are the
    first top_k; of them the shortest prefix whose mass reaches top_p of theirs; of them those with w >= min_p; at
    least the first. The token is the first kept one whose cumulative mass exceeds uniform * the kept mass, and its
    log probability log(w / kept mass).

    uniform fp32 of the leading shape, in [0, 1). Each setting is a number for all rows (taken as fp32) or a tensor
    of the leading shape (fp32; top_k int32). temperature 0: the first of the order; top_k 0, top_p 1, min_p 0:
    off. NaN logits count as -infinity; a row without anything above it gives token -1 and log probability
    -infinity. Masses are summed in fp64.
    """
    what = "sample"
    if logits.is_cuda:
        out = _lib.native().sample(logits, uniform, temperature, top_k, top_p, min_p)
        if type(out) is int:
            _lib.check(out, what)
        if out is not None:
            return out
    no_gradient(what, logits=logits, uniform=uniform, temperature=temperature, top_p=top_p, min_p=min_p)
    if logits.dtype != torch.bfloat16:
        raise ValueError(f"[{what}] logits must be bfloat16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"[{what}] logits must be (..., V) with 1 <= V <= {MAX_VOCAB}, got {tuple(logits.shape)}")
    lead, v = logits.shape[:-1], logits.shape[-1]
    if uniform.dtype != torch.float32 or uniform.shape != lead:
        raise ValueError(f"[{what}] uniform must be float32 of shape {tuple(lead)}, got {uniform.dtype} "
                         f"{tuple(uniform.shape)}")
    temps, temp = _setting(what, "temperature", temperature, torch.float32, lead, lambda t: 0 <= t < math.inf)
    ks, k = _setting(what, "top_k", top_k, torch.int32, lead, lambda t: t >= 0)
    ps, p = _setting(what, "top_p", top_p, torch.float32, lead, lambda t: 0 < t <= 1)
    mins, mn = _setting(what, "min_p", min_p, torch.float32, lead, lambda t: 0 <= t <= 1)
    dev = _check_device(what, logits, uniform, *(t for t in (temps, ks, ps, mins) if t is not None))
    rows = logits.reshape(-1, v)
    if v > 1 and rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < v:
        rows = rows.contiguous()
    m = rows.shape[0]
    uniform = uniform.contiguous()
    tokens = torch.empty(lead, dtype=torch.int64, device=dev)
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev)
    lib = _lib.load()
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    with torch.cuda.device(dev):
        size = lib.qmm4_sample_workspace(m, v)
        _lib.check(min(size, 0), what)
        workspace = torch.empty(size, dtype=torch.uint8, device=dev)
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = lib.qmm4_sample_bf16(rows.data_ptr(), m, v, rows.stride(0), uniform.data_ptr(), ptr(temps), float(temp),
                                  ptr(ks), min(int(k), 2**31 - 1), ptr(ps), float(p), ptr(mins), float(mn),
                                  tokens.data_ptr(), logprobs.data_ptr(), workspace.data_ptr(), stream)
    _lib.check(rc, what)
    return tokens, logprobs
