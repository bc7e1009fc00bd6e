"""Public operator API, mirroring ``ejkernel.modules`` for the operators this package covers, and
the serving step over an 8-bit cache, which the reference does not have."""

from .operations import (
    PageAttentionConfig,
    page_attention,
    RaggedPageAttention,
    RaggedPageAttentionConfig,
    RaggedPageAttentionv3Config,
    allocate_quantized_kv,
    build_page_tables,
    quantized_kv_read,
    quantized_kv_write,
    quantized_ragged_page_attention,
    ragged_page_attention,
    ragged_page_attention_v3,
)

__all__ = [
    "PageAttentionConfig",
    "page_attention",
    "RaggedPageAttention",
    "RaggedPageAttentionConfig",
    "RaggedPageAttentionv3Config",
    "allocate_quantized_kv",
    "build_page_tables",
    "quantized_kv_read",
    "quantized_kv_write",
    "quantized_ragged_page_attention",
    "ragged_page_attention",
    "ragged_page_attention_v3",
]
