"""INT8 W8A8 (+ Hadamard) quantisation (quantization/__init__.py of the reference), and block-scaled
8-bit floating-point products."""

from .fp8_linear import (
    Fp8BlockLinear,
    fp8_block_linear,
    fp8_block_matmul,
    fp8_block_quantize,
    fp8_block_quantize_weight,
    fp8_block_transpose,
)
from .int8_linear import apply_int8_quantization, refresh_int8_weights, restore_int8_quantization

__all__ = ["apply_int8_quantization", "restore_int8_quantization", "refresh_int8_weights",
           "fp8_block_quantize", "fp8_block_quantize_weight", "fp8_block_transpose", "fp8_block_matmul",
           "fp8_block_linear", "Fp8BlockLinear"]
