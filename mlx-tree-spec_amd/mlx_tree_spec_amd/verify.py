"""The quantized layers inside a batched tree-verify forward, and their capture into a HIP graph.

Mirrors the MLP half of each layer of src/mlx_tree_spec/tree_verify.py batch_forward (414-447):
every request's tree nodes are concatenated into one batch of rows, the matmuls, norms and MLPs run
once over all rows, and each residual add is fused with the RMS norm that follows it:

    h, x = add_rms_norm(h, r, layer.post_attention_layernorm)     # tree_verify.py:444
    nxt  = next layer's input_layernorm, or the model's final norm # 445
    h, x = add_rms_norm(h, layer.mlp(x), nxt)                      # 446

`r` is the attention (or GatedDeltaNet) output of the layer. What lies before it, attention over a paged cache, and what
lies behind the last layer are here as well:

    q, k, v, gate = attention_inputs(x, layer, positions, adapters)  # tree_verify.py:311-328: projections (with each
                                                                     # row's adapter), head norms, rotation
    a, k, v = cached_attention(x, layer, cache, step, ...)           # tree_verify.py:311-402: the same, the rows stored, and
                                                                     # attention over all that their requests hold
    tokens, logprobs = next_tokens(x, lm_head, uniform, ...)         # tree_verify.py:447: vocabulary head, sampling

When the MLP is a QuantizedMLP, the first norm is folded into its gate+up projection
(add_rms_norm_gate_up: the same bits, one launch fewer for up to 4 rows).
The row count M = the sum of the requests' tree nodes decides the kernel inside libqmm4 (row-split
for M <= 4, verify kernels up to 64, the GEMM above), as packed_linear._call's routing does.

The reference prebinds one launcher per module to keep the ~400 calls of a forward cheap on the
host (packed_linear.py:61-69, 136-171). Here the same end is reached with a HIP graph: the layers of
a forward are captured once for a fixed row count and replayed, so a replay costs one launch on
the host whatever the number of kernels. Every entry point used here is capturable: none allocates
or clears memory with a memset once its first call has set up its buffers.
"""

from __future__ import annotations

import torch

from .cache import CacheStep, KVCache, check_attention, paged_attention, store_kv_
from .fused_ops import _norm_eps, add_rms_norm, add_rms_norm_gate_up
from .heads import qk_norm_rope
from .lora import LoRALinear
from .packed_linear import STATS, QuantizedMLP
from .sampling import sample


class MLPLayer(torch.nn.Module):
    """The parts of one decoder layer the MLP half uses: post_attention_layernorm and mlp."""

    def __init__(self, post_attention_layernorm: torch.nn.Module, mlp: torch.nn.Module):
        super().__init__()
        self.post_attention_layernorm = post_attention_layernorm
        self.mlp = mlp


def layer_tail(h: torch.Tensor, r: torch.Tensor, layer: MLPLayer, next_norm: torch.nn.Module):
    """(h, x) after one layer's residual adds, norms and MLP (tree_verify.py:444-446)."""
    mlp = layer.mlp
    if isinstance(mlp, QuantizedMLP):
        STATS["gate_up_silu"] += 1
        h, _, t = add_rms_norm_gate_up(h, r, layer.post_attention_layernorm, mlp)
        return add_rms_norm(h, mlp.down_proj(t), next_norm)
    h, x = add_rms_norm(h, r, layer.post_attention_layernorm)
    return add_rms_norm(h, mlp(x), next_norm)


def stack_tail(h: torch.Tensor, rs: list[torch.Tensor], layers: list[MLPLayer], final_norm: torch.nn.Module):
    """layer_tail over a stack of layers; rs[i] is layer i's attention output. Returns (h, x)."""
    if len(rs) != len(layers):
        raise ValueError(f"[stack_tail] {len(rs)} attention outputs for {len(layers)} layers")
    x = None
    for i, layer in enumerate(layers):
        nxt = layers[i + 1].post_attention_layernorm if i + 1 < len(layers) else final_norm
        h, x = layer_tail(h, rs[i], layer, nxt)
    return h, x


class AttentionInputs(torch.nn.Module):
    """The parts of one decoder layer in front of its attention: q_proj, k_proj, v_proj (QuantizedLinear or LoRALinear),
    q_norm and k_norm (RMSNorm modules over a head), the head counts and width, and inv_freq [P]. gated: q_proj gives
    each query head followed by a gate of its width (tree_verify.py:318-321); interleaved as in qk_norm_rope."""

    def __init__(self, q_proj: torch.nn.Module, k_proj: torch.nn.Module, v_proj: torch.nn.Module, q_norm: torch.nn.Module,
                 k_norm: torch.nn.Module, heads: int, kv_heads: int, head_dim: int, inv_freq: torch.Tensor,
                 gated: bool = False, interleaved: bool = False):
        super().__init__()
        self.q_proj, self.k_proj, self.v_proj, self.q_norm, self.k_norm = q_proj, k_proj, v_proj, q_norm, k_norm
        self.heads, self.kv_heads, self.head_dim, self.gated, self.interleaved = heads, kv_heads, head_dim, gated, interleaved
        if _norm_eps(q_norm) != _norm_eps(k_norm):
            raise ValueError(f"[AttentionInputs] q_norm and k_norm differ in eps: {_norm_eps(q_norm)}, {_norm_eps(k_norm)}")
        self.register_buffer("inv_freq", inv_freq)


def _project(proj: torch.nn.Module, x: torch.Tensor, adapters: torch.Tensor | None) -> torch.Tensor:
    return proj(x, adapters) if isinstance(proj, LoRALinear) else proj(x)


def attention_inputs(x: torch.Tensor, layer: AttentionInputs, positions: torch.Tensor, adapters: torch.Tensor | None = None):
    """(q, k, v, gate) of rows x (..., K): q (..., heads, D) and k (..., kv_heads, D) normed and rotated at each row's
    position, v (..., kv_heads, D), gate (..., heads, D) or None. `adapters` (one per row) goes to the projections that
    are LoRALinear."""
    lead, d = x.shape[:-1], layer.head_dim
    width = 2 * d if layer.gated else d
    q = _project(layer.q_proj, x, adapters)
    if q.shape[-1] != layer.heads * width:
        raise ValueError(f"[attention_inputs] q_proj gives {q.shape[-1]} values, expected {layer.heads} heads of {width}")
    q = q.reshape(*lead, layer.heads, width)
    k = _project(layer.k_proj, x, adapters).reshape(*lead, layer.kv_heads, d)
    v = _project(layer.v_proj, x, adapters).reshape(*lead, layer.kv_heads, d)
    gate = q[..., d:] if layer.gated else None
    q, k = qk_norm_rope(q[..., :d] if layer.gated else q, k, layer.q_norm.weight, layer.k_norm.weight,
                        _norm_eps(layer.q_norm), positions, layer.inv_freq, interleaved=layer.interleaved)
    return q, k, v, gate


def cached_attention(x: torch.Tensor, layer: AttentionInputs, cache: KVCache, step: CacheStep,
                     positions: torch.Tensor | None = None, adapters: torch.Tensor | None = None,
                     ancestors: torch.Tensor | None = None, scale: float | None = None):
    """(a, k, v) of a step's rows x (M, K): attention_inputs at `positions`, their keys and values stored into the layer's cache at
    the step's places, and their attention a (M, heads * D) over it, times sigmoid(gate) where the layer is gated: what its
    output projection takes.

    positions: the step's by default (rows in a line); a tree's rows have that of their depth. ancestors as in
    paged_attention. k and v (M, kv_heads, D) are what was stored: once a tree's accepted nodes are known, a step of the
    tables with base and keep gives their places in a line, and store_kv_(k, v, cache, step.slots) puts them there. Rows of a
    request that the step refused (step.request < 0) are not stored and have an attention of zeros: they are not to be kept.
    """
    if x.dim() != 2:
        raise ValueError(f"[cached_attention] x must be (rows, K), got {tuple(x.shape)}")
    if (layer.heads, layer.kv_heads, layer.head_dim) != (step.heads, step.kv_heads, step.head_dim):
        raise ValueError(f"[cached_attention] a layer of {layer.heads} and {layer.kv_heads} heads of {layer.head_dim}, but the step "
                         f"was made for {step.heads} and {step.kv_heads} heads of {step.head_dim}")
    check_attention("cached_attention", cache, step, scale, ancestors)  # (nothing is stored for a step that is refused)
    q, k, v, gate = attention_inputs(x, layer, step.positions if positions is None else positions, adapters)
    store_kv_(k, v, cache, step.slots)
    return paged_attention(q, cache, step, scale=scale, ancestors=ancestors, gate=gate).reshape(len(x), layer.heads * layer.head_dim), k, v


def next_tokens(x: torch.Tensor, head: torch.nn.Module, uniform: torch.Tensor, adapters: torch.Tensor | None = None,
                **settings):
    """(tokens, logprobs) drawn from the vocabulary head's logits of rows x (tree_verify.py:447), with `sample`'s
    settings."""
    return sample(_project(head, x, adapters), uniform, **settings)


class GraphedTail:
    """stack_tail captured into a HIP graph for a fixed batch of rows.

    The inputs are copied into static buffers, the graph replays every kernel of the stack, and
    the outputs are views of static buffers that the next replay overwrites.
    """

    def __init__(self, layers: list[MLPLayer], final_norm: torch.nn.Module, rows: int, dim: int, device):
        self.layers, self.final_norm = layers, final_norm
        self.h_in = torch.zeros((rows, dim), dtype=torch.bfloat16, device=device)
        self.r_in = [torch.zeros((rows, dim), dtype=torch.bfloat16, device=device) for _ in layers]
        # The library keeps its split-K workspace and scratch per (device, stream): warm up on a
        # private stream (first calls allocate them), then capture on that same stream, so the
        # captured kernels use buffers that exist and that no later call on another stream regrows.
        self.stream = torch.cuda.Stream(device)
        self.stream.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(self.stream):
            stack_tail(self.h_in, self.r_in, layers, final_norm)
        torch.cuda.current_stream(device).wait_stream(self.stream)
        torch.cuda.synchronize(device)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.stream):
            self.h_out, self.x_out = stack_tail(self.h_in, self.r_in, layers, final_norm)

    def __call__(self, h: torch.Tensor, rs: list[torch.Tensor]):
        # One launch for all inputs (where their types and layouts allow) instead of one each: 5 inputs of
        # 2 rows 16.9 -> 6.0 us (back to back, host included); 2 rows through 4 layers 206 -> 199 us a pass.
        dst, src = zip((self.h_in, h), *zip(self.r_in, rs))
        torch._foreach_copy_(dst, src)
        self.graph.replay()
        return self.h_out, self.x_out
