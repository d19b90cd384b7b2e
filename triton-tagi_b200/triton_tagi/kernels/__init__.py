"""Moment-contraction kernels (sm_100a CUDA through the C ABI).

Function names and signatures follow triton_tagi/kernels/__init__.py of the
reference so existing callers work unchanged; there is no Triton underneath.
"""

from .attention import bmm_shared_left, bmm_shared_right, bmm_tagi_var
from .common import triton_fused_backward_delta, triton_fused_var_forward, triton_fused_weight_grad
from .embedding import embedding_grad, embedding_lookup, embedding_update
from .int8 import Int8Moments, int8_moments_matmul, quantize_moments, quantize_weights
from .norm import add_rmsnorm, add_rmsnorm_backward, add_rmsnorm_int8

__all__ = [
    "Int8Moments",
    "add_rmsnorm",
    "add_rmsnorm_backward",
    "add_rmsnorm_int8",
    "bmm_shared_left",
    "bmm_shared_right",
    "bmm_tagi_var",
    "embedding_grad",
    "embedding_lookup",
    "embedding_update",
    "int8_moments_matmul",
    "quantize_moments",
    "quantize_weights",
    "triton_fused_backward_delta",
    "triton_fused_var_forward",
    "triton_fused_weight_grad",
]
