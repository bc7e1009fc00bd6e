"""CUDA platform implementations (the reference ships this package empty:
ejkernel/kernels/_cuda/__init__.py:1-15)."""

from .page_attention import page_attention
from .quantized_kv import build_page_tables, quantized_kv_read, quantized_kv_write, quantized_ragged_page_attention
from .ragged_page_attention import ragged_page_attention
from .ragged_page_attention_v3 import ragged_page_attention_v3

__all__ = [
    "build_page_tables",
    "page_attention",
    "quantized_kv_read",
    "quantized_kv_write",
    "quantized_ragged_page_attention",
    "ragged_page_attention",
    "ragged_page_attention_v3",
]
