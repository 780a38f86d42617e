"""B200 (sm_100a) kernels behind the reference engine's ``kernels`` API.

Same exports as the reference package (``kernels/__init__.py:3-14``), plus
the int8 weight-only variants, the ``o`` / ``down`` projections and the GQA
decode attention op, and for decoding in little memory the projections with
4-bit weights, the 8-bit KV cache with its attention, and log probabilities.
"""

from .decode_attn import apply_decode_attn, b200_decode_attn
from .fused_ffn import TritonFFN, triton_fused_gate_up_silu
from .fused_qkv import TritonAttention, triton_fused_qkv
from .int4 import (
    Int4Attention,
    Int4FFN,
    Int4Linear,
    dequantize_grouped,
    int4_fused_gate_up_silu,
    int4_fused_qkv,
    int4_linear,
    quantize_grouped,
)
from .kv8 import Int8KV, Int8KVCache, int8_kv_append, int8_kv_decode_attn, int8_kv_expand, int8_kv_step
from .linear import B200Linear, Int8Linear, b200_linear, int8_linear
from .logprobs import TokenLogprobs, b200_token_logprobs
from .quant import (
    Int8Attention,
    Int8FFN,
    dequantize_per_row,
    int8_fused_gate_up_silu,
    int8_fused_qkv,
    quantize_per_row,
)
from .swap import (
    apply_int4_kernels,
    apply_int8_kernels,
    apply_linear_kernels,
    apply_triton_kernels,
    prewarm_triton_kernels,
)

__all__ = [
    "Int4Attention",
    "Int4FFN",
    "Int4Linear",
    "apply_int4_kernels",
    "dequantize_grouped",
    "int4_fused_gate_up_silu",
    "int4_fused_qkv",
    "int4_linear",
    "quantize_grouped",
    "Int8KV",
    "Int8KVCache",
    "int8_kv_append",
    "int8_kv_decode_attn",
    "int8_kv_expand",
    "int8_kv_step",
    "TokenLogprobs",
    "b200_token_logprobs",
    "apply_decode_attn",
    "b200_decode_attn",
    "B200Linear",
    "Int8Linear",
    "apply_linear_kernels",
    "b200_linear",
    "int8_linear",
    "Int8Attention",
    "Int8FFN",
    "TritonAttention",
    "TritonFFN",
    "apply_int8_kernels",
    "apply_triton_kernels",
    "dequantize_per_row",
    "int8_fused_gate_up_silu",
    "int8_fused_qkv",
    "prewarm_triton_kernels",
    "quantize_per_row",
    "triton_fused_gate_up_silu",
    "triton_fused_qkv",
]
