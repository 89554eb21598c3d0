"""MI355X (gfx950) packed 4-bit affine quantized matmul in MLX's format.

    from mlx_tree_spec_amd import quantized_matmul, dequantize, QuantizedLinear, install
    from mlx_tree_spec_amd import quantized_matmul_lora, qk_norm_rope, sample    # what differs per request

All compute runs in libqmm4.so (hand-written HIP kernels, C ABI in include/); importing
this package does not load it, the first call does, and fails loudly if it is not built.
"""

from .fused_ops import add_rms_norm, add_rms_norm_, add_rms_norm_gate_up, add_rms_norm_qmm_
from .heads import qk_norm_rope
from .lora import LoRALinear, quantized_matmul_lora, stack_adapters
from .packed_linear import STATS, QuantizedLinear, QuantizedMLP, eligible, install
from .qmm import dequantize, gate_up_silu, pack_nax, quantized_matmul, unpack_nax
from .sampling import sample
from .verify import AttentionInputs, GraphedTail, MLPLayer, attention_inputs, layer_tail, next_tokens, stack_tail

__all__ = [
    "quantized_matmul", "gate_up_silu", "dequantize", "pack_nax", "unpack_nax", "add_rms_norm",
    "add_rms_norm_", "add_rms_norm_qmm_", "add_rms_norm_gate_up", "QuantizedLinear", "QuantizedMLP",
    "quantized_matmul_lora", "stack_adapters", "LoRALinear", "qk_norm_rope", "sample", "eligible", "install",
    "STATS", "MLPLayer", "layer_tail", "stack_tail", "GraphedTail", "AttentionInputs", "attention_inputs", "next_tokens",
]
__version__ = "0.1.0"
