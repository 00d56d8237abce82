"""mlxcel_amd — MI355X (gfx950) quantized-matmul hot path for mlxcel / MLX.

The product is the C-ABI library ``libmlxq.so`` (``include/mlxq.h``); this
package holds its HIP sources (``csrc/``), the build script, and a Python
mirror of the reference operator interface (``ops``).
"""
from .ops import (cache_append, cache_compact, cache_fork, cache_free, cache_reserve, clear_cache,  # noqa: F401
                  dequantize, fused_moe_expert, fused_moe_geglu, gather_qmm, get_cache_memory, paged_attention,
                  quantize, quantized_linear, quantized_matmul, quantized_matmul_matches_dense_gemm,
                  quantized_matmul_multi, residual_norm, token_logprobs, workspace_reserve)
from ._lib import LIB_PATH, load as load_library  # noqa: F401
from . import loader  # noqa: F401,E402  (MLX-quantized safetensors -> device planes)

__all__ = ["quantized_matmul", "quantized_matmul_multi", "quantized_linear",
           "quantized_matmul_matches_dense_gemm", "gather_qmm", "dequantize", "quantize",
           "paged_attention", "cache_reserve", "cache_append", "cache_fork", "cache_free", "cache_compact",
           "residual_norm", "token_logprobs", "fused_moe_expert", "fused_moe_geglu", "workspace_reserve", "get_cache_memory", "clear_cache",
           "loader", "load_library", "LIB_PATH"]
