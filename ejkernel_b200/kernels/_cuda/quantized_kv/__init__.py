from ._interface import (
    build_page_tables,
    quantized_kv_read,
    quantized_kv_write,
    quantized_ragged_page_attention,
    read_status,
)

__all__ = [
    "build_page_tables",
    "quantized_kv_read",
    "quantized_kv_write",
    "quantized_ragged_page_attention",
    "read_status",
]
