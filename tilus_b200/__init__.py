"""B200-native weight-only quantized matmul (drop-in for the reference's
examples/quantization/matmul_a16wx.py operator surface), and what a decoder needs around it."""
from .dtypes import *  # noqa: F401,F403
from .int8 import Int8Linear  # noqa: E402,F401
from .linear import QuantizedLinear  # noqa: E402,F401
from .norm import BlockNorm, block_norm  # noqa: E402,F401
from .ops import (block_norm_backward, block_norm_cast_int8, dequantize, int8_gate_up,  # noqa: E402,F401
                  int8_matmul, per_token_cast_int8, quantized_matmul)
