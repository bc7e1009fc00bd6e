"""B200-native (sm_100a) ragged paged attention behind the ejkernel operator API.

Importing the package does not touch CUDA; the compiled library is loaded on the first call and
its absence is an error, never a silent fallback.
"""

__version__ = "0.1.0"

from . import kernels, modules  # noqa: F401
from .kernels import Backend, Platform, kernel_registry, serving_registry
from .modules import (
    allocate_quantized_kv,
    build_page_tables,
    page_attention,
    quantized_kv_read,
    quantized_kv_write,
    quantized_ragged_page_attention,
    RaggedPageAttention,
    RaggedPageAttentionConfig,
    ragged_page_attention,
    ragged_page_attention_v3,
)

__all__ = [
    "Backend",
    "Platform",
    "RaggedPageAttention",
    "RaggedPageAttentionConfig",
    "allocate_quantized_kv",
    "build_page_tables",
    "kernel_registry",
    "page_attention",
    "quantized_kv_read",
    "quantized_kv_write",
    "quantized_ragged_page_attention",
    "ragged_page_attention",
    "ragged_page_attention_v3",
    "serving_registry",
]
