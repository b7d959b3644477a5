"""sm_100a kernel wrappers with the export list of triton_moe.kernels
(triton_moe/kernels/__init__.py:18-40), and the few-token (decode) and 4-bit
kernels beside it."""

from ._ops import check_device_status
from .few_tokens import FEW_TOKENS_MAX, moe_few_tokens
from .fused_cumsum import fused_route
from .gather import padded_gather, padded_gather_autograd
from .grouped_gemm import (
    GroupedGemmDown,
    GroupedGemmUp,
    grouped_gemm_down,
    grouped_gemm_down_autograd,
    grouped_gemm_down_backward,
    grouped_gemm_up,
    grouped_gemm_up_autograd,
    grouped_gemm_up_backward,
    precompute_gather_map,
)
from .int4 import (
    Int4Weight,
    dequantize_int4,
    grouped_gemv_down_int4,
    grouped_gemv_up_int4,
    pack_int4,
    quantize_int4,
)
from .scatter import padded_scatter, padded_scatter_autograd

__all__ = [
    # Gather/Scatter
    "padded_gather",
    "padded_gather_autograd",
    "padded_scatter",
    "padded_scatter_autograd",
    # Forward kernels
    "grouped_gemm_up",
    "grouped_gemm_down",
    # Backward kernels
    "grouped_gemm_up_backward",
    "grouped_gemm_down_backward",
    # Autograd wrappers
    "grouped_gemm_up_autograd",
    "grouped_gemm_down_autograd",
    # Gather map for fused gather
    "precompute_gather_map",
    # Autograd Function classes
    "GroupedGemmUp",
    "GroupedGemmDown",
    # Routing
    "fused_route",
    # The whole layer for a few tokens (decode)
    "moe_few_tokens",
    "FEW_TOKENS_MAX",
    # 4-bit expert weights
    "Int4Weight",
    "quantize_int4",
    "pack_int4",
    "dequantize_int4",
    "grouped_gemv_up_int4",
    "grouped_gemv_down_int4",
    # Device status word (bounded waits, bad expert ids, capacity)
    "check_device_status",
]
