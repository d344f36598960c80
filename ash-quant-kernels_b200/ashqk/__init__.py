"""ashqk on B200: AWQ-format W4A16 linear layers with hand-written sm_100a kernels, and microscaled
4-bit floating point (``ashqk.fp4``: MXFP4 / NVFP4 tensors, their quantiser and W4A4 products).

Same public names as MMMchou/ash-quant-kernels (ashqk/__init__.py:1-24): the
dispatcher ``w4a16_linear`` and the format helpers of ``ashqk.ref``.
"""

from .fp4 import (
    FP4Linear,
    FP4Tensor,
    dequantize_fp4,
    fp4_global_scale,
    fp4_matmul,
    quantize_fp4,
    silu_mul_quantize_fp4,
    w4a4_linear,
)
from .ops import GEMV_MAX_M, w4a16_linear
from .ref import (
    AWQ_ORDER,
    AWQ_REVERSE_ORDER,
    dequantize_awq,
    pack_awq,
    quantize_awq,
    unpack_awq,
    w4a16_gemm_fp32,
    w4a16_gemm_ref,
)

__all__ = [
    "w4a16_linear",
    "GEMV_MAX_M",
    "AWQ_ORDER",
    "AWQ_REVERSE_ORDER",
    "dequantize_awq",
    "pack_awq",
    "quantize_awq",
    "unpack_awq",
    "w4a16_gemm_fp32",
    "w4a16_gemm_ref",
    "FP4Linear",
    "FP4Tensor",
    "quantize_fp4",
    "silu_mul_quantize_fp4",
    "dequantize_fp4",
    "fp4_global_scale",
    "fp4_matmul",
    "w4a4_linear",
]
__version__ = "0.1.0"
