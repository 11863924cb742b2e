"""Public quantization API, same names as cublade.quantization
(reference: quantization/__init__.py:1-17)."""
from .utils import *  # noqa: F401,F403  (replace_linear_layers, as in the reference)
from .tensor import QuantizedTensor
from .dequantizers import dequantize_tensor
from .kv_cache import QuantizedKVCache, append_kv, attend_kv, dequantize_kv
from .linear import cuBladeW8A16LinearLayer, cubladeW8A16LinearLayer
from .norms import norm_tensor, residual_norm
from .quantizers import quantize_tensor, quantize_model
from .w8a8 import cuBladeW8A8GatedMLP, cuBladeW8A8LinearLayer, gated_w8a8, linear_w8a8
from .outlier_utils import (detect_activation_outlier_columns, detect_outlier_columns,
                            separate_outliers, split_weights_by_outliers)

__all__ = [
    "quantize_model",
    "quantize_tensor",
    "dequantize_tensor",
    "QuantizedTensor",
    "cuBladeW8A16LinearLayer",
    "cubladeW8A16LinearLayer",
    "detect_outlier_columns",
    "detect_activation_outlier_columns",
    "QuantizedKVCache",
    "append_kv",
    "attend_kv",
    "dequantize_kv",
    "linear_w8a8",
    "gated_w8a8",
    "norm_tensor",
    "residual_norm",
    "cuBladeW8A8LinearLayer",
    "cuBladeW8A8GatedMLP",
    "separate_outliers",
    "split_weights_by_outliers",
]
