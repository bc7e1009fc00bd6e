"""Public operators of a serving step over a paged KV cache held in 8 bits.

    lens, start, slots, num_free = build_page_tables(query_lens, context_lens, block_tables, free_pages, num_free, n,
                                                     page_size=page, total_tokens=T)
    quantized_kv_write(keys, values, kv_pages, kv_scales, slots)
    out = quantized_ragged_page_attention(queries, kv_pages, kv_scales, lens, block_tables, start, n)

None of the three reads anything back to the host, so a step can be captured into a CUDA graph.  Sharding by KV heads works
as for ``ragged_page_attention``: every rank holds its heads of q/k/v, ``kv_pages`` and ``kv_scales`` (their axis 1) and the
same page tables.  There is one implementation (CUDA); any other ``platform`` raises.
"""

from __future__ import annotations

from typing import Literal

import torch

from ...kernels._registry import Backend, serving_registry
from ...sharding import Mesh1D, PartitionSpec, all_gather_heads
from .configs import RaggedPageAttentionConfig
from .ragged_page_attention import _resolve_platform

Array = torch.Tensor
PlatformName = Literal["triton", "pallas", "cuda", "xla", "auto"]


def _impl(name: str, platform):
    return serving_registry.get(name, platform=_resolve_platform(platform), backend=Backend.GPU)


# the registry is asked once for the usual case
_attention, _write, _read, _tables = (
    _impl(name, None) for name in ("quantized_ragged_page_attention", "quantized_kv_write", "quantized_kv_read", "build_page_tables")
)


def allocate_quantized_kv(
    num_pages: int,
    num_kv_heads: int,
    page_size: int,
    head_dim: int,
    *,
    dtype: torch.dtype = torch.float8_e4m3fn,
    scale_block: int | None = None,
    device: torch.device | str = "cuda",
) -> tuple[Array, Array]:
    """An empty 8-bit cache ``(kv_pages, kv_scales)``: e4m3 or int8 codes, one scale per ``scale_block`` tokens of a head
    (a power of two that divides ``page_size``; default the largest)."""
    if scale_block is None:
        scale_block = page_size & -page_size
    if scale_block < 1 or scale_block & (scale_block - 1) or page_size % scale_block:
        raise ValueError(f"{scale_block=} must be a power of two that divides {page_size=}")
    if dtype not in (torch.float8_e4m3fn, torch.int8):
        raise NotImplementedError(f"dtype {dtype} is not supported (float8_e4m3fn, int8)")
    pages = torch.zeros((num_pages, num_kv_heads, 2, page_size, head_dim), dtype=torch.int8, device=device).view(dtype)
    scales = torch.ones((num_pages, num_kv_heads, 2, page_size // scale_block), dtype=torch.float32, device=device)
    return pages, scales


def build_page_tables(
    query_lens: Array,
    context_lens: Array,
    block_tables: Array,
    free_pages: Array,
    num_free: Array,
    num_seqs: Array | int,
    /,
    *,
    page_size: int,
    total_tokens: int,
    finished: Array | None = None,
    platform: PlatformName | None = None,
) -> tuple[Array, Array, Array, Array]:
    """``(context_lens, query_start_loc, slot_mapping, num_free)`` of this step; tables and free list in place."""
    impl = _tables if platform is None else _impl("build_page_tables", platform)
    return impl(query_lens, context_lens, block_tables, free_pages, num_free, num_seqs, page_size=page_size,
                total_tokens=total_tokens, finished=finished)


def quantized_kv_write(
    keys: Array, values: Array, kv_pages: Array, kv_scales: Array, slot_mapping: Array, /, *, platform: PlatformName | None = None
) -> tuple[Array, Array]:
    """Write a step's rows to the cache in place; returns ``(kv_pages, kv_scales)``."""
    impl = _write if platform is None else _impl("quantized_kv_write", platform)
    return impl(keys, values, kv_pages, kv_scales, slot_mapping)


def quantized_kv_read(
    kv_pages: Array,
    kv_scales: Array,
    slot_mapping: Array,
    /,
    *,
    dtype: torch.dtype = torch.bfloat16,
    platform: PlatformName | None = None,
) -> tuple[Array, Array]:
    """``(keys, values)`` of the cache's rows at ``slot_mapping``, in 16 bits."""
    impl = _read if platform is None else _impl("quantized_kv_read", platform)
    return impl(kv_pages, kv_scales, slot_mapping, dtype=dtype)


def quantized_ragged_page_attention(
    queries: Array,
    kv_pages: Array,
    kv_scales: Array,
    context_lens: Array,
    block_tables: Array,
    query_start_loc: Array,
    num_seqs: Array | int,
    /,
    *,
    softmax_scale: float | None = None,
    logits_soft_cap: float | None = None,
    sliding_window: int | None = None,
    softmax_aux: Array | None = None,
    platform: PlatformName | None = None,
    cfg: RaggedPageAttentionConfig | None = None,
    mesh: Mesh1D | None = None,
    in_specs: tuple[PartitionSpec | None, ...] | None = None,
    out_specs: PartitionSpec | None = None,
) -> Array:
    """Mixed decode / chunked-prefill attention over the 8-bit cache."""
    impl = _attention if platform is None else _impl("quantized_ragged_page_attention", platform)
    out = impl(
        queries, kv_pages, kv_scales, context_lens, block_tables, query_start_loc, num_seqs,
        softmax_scale=softmax_scale, logits_soft_cap=logits_soft_cap, sliding_window=sliding_window, softmax_aux=softmax_aux,
        num_kv_pages_per_block=None if cfg is None else cfg.num_kv_pages_per_block,
        num_queries_per_block=None if cfg is None else cfg.num_queries_per_block,
    )
    if mesh is not None and in_specs is not None and out_specs is not None and mesh.size > 1:
        if PartitionSpec(*out_specs).sharded_dim(mesh.axis_name) is None:
            out = all_gather_heads(out, mesh)
    return out
