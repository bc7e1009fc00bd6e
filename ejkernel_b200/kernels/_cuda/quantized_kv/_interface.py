"""CUDA (sm_100a) implementations of the serving step around a paged KV cache held in 8 bits.

``build_page_tables`` -> ``quantized_kv_write`` -> ``quantized_ragged_page_attention`` (and ``quantized_kv_read``, the
cache's values back in 16 bits), registered in ``serving_registry``; the reference has none of them.  The work is done by
hand-written kernels behind the C ABI of ``include/ejk_q8.h``, which also defines the operators; there is no other code
path.

The cache is ``kv_pages [num_pages, num_kv_heads, 2, page_size, head_dim]`` (``torch.float8_e4m3fn`` or ``torch.int8``;
index 2 = K, V) with ``kv_scales [num_pages, num_kv_heads, 2, blocks_per_page]`` in float32: the value of a code is the
code times the scale of its block of ``page_size / blocks_per_page`` tokens.

What a call may look like depends only on shapes, strides, dtypes and keywords: it is checked in full the first time and
remembered under that signature with the structs of the C call, so that a serving loop pays for a dictionary look-up.
What depends on values (lengths, page ids) is checked on the device and reported through ``read_status``.

Streams and graphs: a call runs on the current stream.  Scratch is kept per stream; a call that is being captured takes
its own from the graph's memory pool instead, so that two graphs never share it and no later call can free it.
"""

from __future__ import annotations

import ctypes
import math
import os

import jaxtyping
import torch
from beartype import beartype
from jaxtyping import Bool, Float, Int32, Shaped
from torch import Tensor as Array

from .... import _cabi
from ..._registry import Backend, Platform, serving_registry
from ..ragged_page_attention._interface import _DTYPE_CODE, FP8, _num_seqs_tensor

CODE_DTYPES = {FP8: _cabi.E4M3, torch.int8: _cabi.I8}

_MAX_REMEMBERED = 4096
_MAX_FACTOR, _MAX_CAP = 2.0**126, 2.0**100
_MAX_INT = 0x7FFFFFFF
_plans: dict[tuple, object] = {}
_status: dict[int, int] = {}  # address of the device's word, in the library's image: bits are only OR-ed in, so streams can share it
_scratch: dict[tuple[int, int], torch.Tensor] = {}  # (device, stream) -> workspace; a stream's calls are ordered
_MAX_STREAMS = 16

_checked = jaxtyping.jaxtyped(typechecker=beartype)


_capturing = torch._C._cuda_isCurrentStreamCapturing
_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without a Stream object around it
_current_device = torch._C._cuda_getDevice


def _template(shape, dtype, device) -> torch.Tensor:
    """What ``torch.empty_like`` takes to make a dense tensor of this shape, in half the time of ``torch.empty``; one element."""
    return torch.empty(1, dtype=dtype, device=device).expand(shape)


_functions = {}


def _function(name: str):
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_cabi.load(), name)
    return fn


def _remember(key, plan):
    if key is not None:
        if len(_plans) >= _MAX_REMEMBERED:
            _plans.clear()
        _plans[key] = plan
    return plan


def _on_one_device(first: str, device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, {first} on {device}")


def _contiguous(**tensors) -> None:
    for name, t in tensors.items():
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous (dense row-major)")


def _need_cuda(what: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what}[cuda]: tensors must live on a CUDA device (no CPU fallback)")


def _check_cache(kv_pages, kv_scales) -> int:
    """The tokens of a scale block."""
    if kv_pages.dtype not in CODE_DTYPES:
        raise NotImplementedError(f"kv_pages dtype {kv_pages.dtype} is not supported (float8_e4m3fn, int8)")
    pages, heads, two, page_size, head_dim = kv_pages.shape
    if two != 2:
        raise ValueError(f"kv_pages must be [num_pages, num_kv_heads, 2, page_size, head_dim], got {tuple(kv_pages.shape)}")
    if head_dim not in (64, 128, 256):
        raise NotImplementedError(f"{head_dim=} is not supported by the CUDA path (64, 128, 256)")
    if min(pages, heads, page_size) < 1 or pages * page_size > 0x7FFFFFFF:
        raise ValueError(f"kv_pages of shape {tuple(kv_pages.shape)}: empty, or more than 2^31 - 1 token slots")
    blocks = kv_scales.shape[3]
    if blocks < 1 or page_size % blocks or (page_size // blocks) & (page_size // blocks - 1):
        raise ValueError(f"kv_scales: {blocks} scales for a page of {page_size} tokens; a block must be a power of two of tokens")
    _contiguous(kv_pages=kv_pages, kv_scales=kv_scales)
    return page_size // blocks


def _status_word(device: torch.device) -> int:
    """Address of the status word of a device, which is the current one.  Memory of the allocator would not do: a word that is
    made while a stream is captured would be the graph's, and zeroed by every replay."""
    at = _status.get(device.index)
    if at is None:
        word = ctypes.c_void_p()
        _cabi.check(_function("ejk_q8_status_word")(ctypes.byref(word)), "ejk_q8_status_word")
        at = _status[device.index] = word.value
    return at


class _Word:
    def __init__(self, at: int):
        self.__cuda_array_interface__ = dict(shape=(1,), typestr="<i4", data=(at, False), version=3)


def _status_tensor(index: int) -> torch.Tensor:
    return torch.as_tensor(_Word(_status[index]), device=torch.device("cuda", index))


def read_status(device: torch.device | str | int | None = None, clear: bool = True) -> int:
    """The status word of these operators on a device (forces a synchronisation): bits of ``_cabi.STATUS_TEXT``."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    if index not in _status:
        return 0
    torch.cuda.synchronize(index)
    word = _status_tensor(index)
    value = int(word.item())
    if clear:
        word.zero_()
        torch.cuda.current_stream(index).synchronize()
    return value


def _after(device: torch.device, what: str) -> None:
    """Opt-in (``EJKERNEL_B200_CHECK_STATUS=1``): read the status word after the call and raise when an output is invalid."""
    if os.environ.get("EJKERNEL_B200_CHECK_STATUS", "0") in ("", "0") or device.index not in _status or _capturing():
        return
    tensor = _status_tensor(device.index)
    word = int(tensor.item())
    if word & (_cabi.ST_TIMEOUT | _cabi.ST_INTERNAL):
        tensor.zero_()
        raise _cabi.RpaLibraryError(f"{what}: status word {word:#x}: " + "; ".join(_cabi.decode_status(word)))


def _workspace(nbytes: int, device: torch.device, stream: int) -> torch.Tensor:
    if _capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[: _cabi.Q8_TICKET_BYTES].zero_()  # a step of the graph: its memory may have had other uses
        return ws
    key = (device.index, stream)
    ws = _scratch.pop(key, None)
    if ws is None or ws.shape[0] < nbytes:
        ws = torch.empty(1 << max(16, (nbytes - 1).bit_length()), dtype=torch.uint8, device=device)
        ws[: _cabi.Q8_TICKET_BYTES].zero_()
    _scratch[key] = ws  # the most recently used stands last
    if len(_scratch) > _MAX_STREAMS:
        del _scratch[next(iter(_scratch))]
    return ws


def _count(num_seqs, device: torch.device) -> torch.Tensor:
    """The number of sequences as an int32 on the device."""
    if isinstance(num_seqs, torch.Tensor) and num_seqs.dtype is torch.int32 and num_seqs.device == device and num_seqs.numel() == 1:
        return num_seqs
    if _capturing() and not (isinstance(num_seqs, torch.Tensor) and num_seqs.is_cuda):
        # a step of the graph: copying from the host cannot be captured, and a constant that is kept for eager calls can be
        # dropped while the graph lives
        return torch.full((1,), int(num_seqs), dtype=torch.int32, device=device)
    return _num_seqs_tensor(num_seqs, device)


# ---------------------------------------------------------------------------------------- attention


@_checked
def _plan_attention(
    queries: Float[Array, "total_tokens num_q_heads head_dim"],
    kv_pages: Shaped[Array, "num_pages num_kv_heads two page_size head_dim"],
    kv_scales: Float[Array, "num_pages num_kv_heads two blocks_per_page"],
    context_lens: Int32[Array, "num_seqs"],
    block_tables: Int32[Array, "num_seqs pages_per_seq"],
    query_start_loc: Int32[Array, "num_seqs_plus_one"],
    softmax_aux: Float[Array, "rows num_sinks"] | Float[Array, "num_sinks"] | None,
    softmax_scale: float | int | None,
    logits_soft_cap: float | int | None,
    sliding_window: int | None,
    num_kv_pages_per_block: int | None,
    num_queries_per_block: int | None,
):
    block = _check_cache(kv_pages, kv_scales)
    if queries.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"queries dtype {queries.dtype} is not supported by the CUDA path (bf16/f16 only)")
    if kv_scales.dtype != torch.float32:
        raise ValueError(f"kv_scales must be float32, got {kv_scales.dtype}")
    T, Hq, D = queries.shape
    P, Hkv, _, page_size, _ = kv_pages.shape
    S, pps = block_tables.shape
    if Hq % Hkv != 0 or Hq == 0:
        raise ValueError(f"num_q_heads={Hq} must be divisible by num_kv_heads={Hkv}")
    if S < 1 or pps < 1:
        raise ValueError(f"block_tables of shape {tuple(block_tables.shape)} holds no page")
    if query_start_loc.shape != (S + 1,):
        raise ValueError(f"Expected {query_start_loc.shape=} to be ({S + 1},) where `num_seqs` is `block_tables.shape[0]`.")
    if sliding_window is not None and sliding_window <= 0:
        raise ValueError(f"{sliding_window=} must be positive.")
    if logits_soft_cap is not None and (logits_soft_cap == 0.0 or not math.isfinite(logits_soft_cap)):
        raise ValueError(f"{logits_soft_cap=} must be finite and not 0.0.")
    scale = D**-0.5 if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale):
        raise ValueError(f"{softmax_scale=} must be finite")
    # the kernels hold these numbers in float32, times 2 log2(e) at most
    if abs(scale) > _MAX_FACTOR:
        raise ValueError(f"{softmax_scale=} is beyond the range of float32")
    if logits_soft_cap is not None and not (1 / _MAX_CAP <= abs(logits_soft_cap) <= _MAX_CAP and abs(scale) / abs(logits_soft_cap) <= _MAX_CAP):
        raise ValueError(f"{logits_soft_cap=} or its quotient with the softmax scale is beyond the range of float32")
    if num_kv_pages_per_block is not None and not 0 < num_kv_pages_per_block <= pps:
        raise ValueError(f"{num_kv_pages_per_block=} must be in range (0, {pps}].")
    if num_queries_per_block is not None and num_queries_per_block <= 0:
        raise ValueError(f"{num_queries_per_block=} must be positive.")
    sinks = rows = 0
    if softmax_aux is not None:
        sinks, rows = softmax_aux.shape[-1], 1 if softmax_aux.ndim == 1 else softmax_aux.shape[0]
        if softmax_aux.ndim == 2 and rows not in (Hq, Hkv):
            raise ValueError(f"softmax_aux first dim must be num_q_heads ({Hq}) or num_kv_heads ({Hkv}), got {tuple(softmax_aux.shape)}")
    _contiguous(queries=queries, context_lens=context_lens, block_tables=block_tables, query_start_loc=query_start_loc)
    _on_one_device("queries", queries.device, kv_pages=kv_pages, kv_scales=kv_scales, context_lens=context_lens,
                   block_tables=block_tables, query_start_loc=query_start_loc, softmax_aux=softmax_aux)
    _need_cuda("quantized_ragged_page_attention", queries)
    shape = _cabi.Q8Shape(T, S, pps, P, page_size, Hq, Hkv, D, _DTYPE_CODE[queries.dtype], CODE_DTYPES[kv_pages.dtype], block)
    # a window, or a threshold, beyond 32 bits is beyond every length
    attrs = _cabi.Attrs(scale, float(logits_soft_cap or 0.0), min(int(sliding_window or 0), _MAX_INT), sinks, rows,
                        int(num_kv_pages_per_block or 0), min(int(num_queries_per_block or 0), _MAX_INT), 0.0, 0.0)
    nbytes = 0
    if T:
        with torch.cuda.device(queries.device):
            nbytes = int(_cabi.load().ejk_q8_attention_workspace_bytes(ctypes.byref(shape), ctypes.byref(attrs)))
        if nbytes == 0:
            raise ValueError("ejk_q8_attention_workspace_bytes rejected the shape")
    return shape, attrs, nbytes, ctypes.byref(shape), ctypes.byref(attrs), queries.device


@serving_registry.register("quantized_ragged_page_attention", Platform.CUDA, Backend.GPU)
def quantized_ragged_page_attention(
    queries: Float[Array, "total_tokens num_q_heads head_dim"],
    kv_pages: Shaped[Array, "num_pages num_kv_heads 2 page_size head_dim"],
    kv_scales: Float[Array, "num_pages num_kv_heads 2 blocks_per_page"],
    context_lens: Int32[Array, "num_seqs"],
    block_tables: Int32[Array, "num_seqs pages_per_seq"],
    query_start_loc: Int32[Array, "num_seqs_plus_one"],
    num_seqs: Array | int,
    *,
    softmax_scale: float | None = None,
    logits_soft_cap: float | None = None,
    sliding_window: int | None = None,
    softmax_aux: Float[Array, "rows num_sinks"] | Float[Array, "num_sinks"] | None = None,
    num_kv_pages_per_block: int | None = None,
    num_queries_per_block: int | None = None,
) -> Float[Array, "total_tokens num_q_heads head_dim"]:
    """``ragged_page_attention`` over the 8-bit cache: the same batch description, masks, soft cap, sinks and zero rows.

    Products run on the codes as 16-bit floats (exact) and accumulate in float32; ``softmax_scale`` defaults to
    ``head_dim ** -0.5``.  Returns a tensor of the shape and dtype of ``queries``.

    ``num_queries_per_block``: from how many query tokens on a sequence is served by tensor tiles (head_dim 64 and 128).  Without
    it that is decided for batches with more tokens than ``block_tables`` has rows; a table padded with idle rows hides from the
    host whether there is a prompt in the batch, so give it where chunks of prompts come in such tables.
    """
    try:
        key = (queries.shape, queries.dtype, queries.is_contiguous(), queries.get_device(),
               kv_pages.shape, kv_pages.dtype, kv_pages.is_contiguous(), kv_pages.get_device(),
               kv_scales.shape, kv_scales.dtype, kv_scales.is_contiguous(), kv_scales.get_device(),
               context_lens.shape, context_lens.dtype, context_lens.is_contiguous(), context_lens.get_device(),
               block_tables.shape, block_tables.dtype, block_tables.is_contiguous(), block_tables.get_device(),
               query_start_loc.shape, query_start_loc.dtype, query_start_loc.is_contiguous(), query_start_loc.get_device(),
               None if softmax_aux is None else (softmax_aux.shape, softmax_aux.dtype, softmax_aux.get_device()),
               softmax_scale, logits_soft_cap, sliding_window, num_kv_pages_per_block, num_queries_per_block, "attention")
        plan = _plans.get(key)
    except (AttributeError, TypeError):  # not tensors, not hashable: the full check says what is wrong
        key = plan = None
    if plan is None:
        plan = _plan_attention(queries, kv_pages, kv_scales, context_lens, block_tables, query_start_loc, softmax_aux,
                               softmax_scale, logits_soft_cap, sliding_window, num_kv_pages_per_block, num_queries_per_block)
        _remember(key, plan)
    shape, attrs, nbytes, shape_ref, attrs_ref, device = plan
    if shape.total_tokens == 0:
        return torch.empty_like(queries)
    index = device.index
    if index != _current_device():
        with torch.cuda.device(device):
            return quantized_ragged_page_attention(
                queries, kv_pages, kv_scales, context_lens, block_tables, query_start_loc, num_seqs, softmax_scale=softmax_scale,
                logits_soft_cap=logits_soft_cap, sliding_window=sliding_window, softmax_aux=softmax_aux,
                num_kv_pages_per_block=num_kv_pages_per_block, num_queries_per_block=num_queries_per_block)
    out = torch.empty_like(queries)  # every row is written: sequences by their tiles, rows of no sequence or of a refused one with zeros
    aux = None
    if softmax_aux is not None and attrs.num_sinks:
        aux = softmax_aux.to(torch.float32).contiguous()
    num_seqs = _count(num_seqs, device)
    stream = _raw_stream(index)
    ws = _workspace(nbytes, device, stream)
    rc = _function("ejk_q8_attention_launch")(
        queries.data_ptr(), kv_pages.data_ptr(), kv_scales.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(),
        query_start_loc.data_ptr(), num_seqs.data_ptr(), None if aux is None else aux.data_ptr(), out.data_ptr(),
        ws.data_ptr(), nbytes, _status_word(device), shape_ref, attrs_ref, stream)
    if rc:
        _cabi.check(rc, "ejk_q8_attention_launch")
    _after(device, "quantized_ragged_page_attention")
    return out


# ------------------------------------------------------------------------------------ write and read


@_checked
def _plan_write(
    keys: Float[Array, "total_tokens num_kv_heads head_dim"],
    values: Float[Array, "total_tokens num_kv_heads head_dim"],
    kv_pages: Shaped[Array, "num_pages num_kv_heads two page_size head_dim"],
    kv_scales: Float[Array, "num_pages num_kv_heads two blocks_per_page"],
    slot_mapping: Int32[Array, "total_tokens"],
):
    block = _check_cache(kv_pages, kv_scales)
    if keys.dtype not in _DTYPE_CODE or values.dtype != keys.dtype:
        raise NotImplementedError(f"keys and values must share one 16-bit float dtype (bf16/f16), got {keys.dtype} and {values.dtype}")
    if kv_scales.dtype != torch.float32:
        raise ValueError(f"kv_scales must be float32, got {kv_scales.dtype}")
    T, Hkv, D = keys.shape
    strides = []
    for name, t in (("keys", keys), ("values", values)):
        # rows may be apart, as in a view of a fused projection; a row itself is dense
        row = t.stride(0) if T > 1 else Hkv * D
        if t.stride(2) != 1 or (Hkv > 1 and t.stride(1) != D) or row < Hkv * D or row % 8:
            raise ValueError(f"{name}: rows must be dense and a multiple of 8 elements apart, got strides {t.stride()}")
        strides.append(row)
    _contiguous(slot_mapping=slot_mapping)
    _on_one_device("keys", keys.device, values=values, kv_pages=kv_pages, kv_scales=kv_scales, slot_mapping=slot_mapping)
    _need_cuda("quantized_kv_write", keys)
    P, _, _, page_size, _ = kv_pages.shape
    shape = _cabi.Q8Shape(T, 1, 1, P, page_size, Hkv, Hkv, D, _DTYPE_CODE[keys.dtype], CODE_DTYPES[kv_pages.dtype], block)
    return shape, ctypes.byref(shape), strides[0], strides[1], keys.device


@serving_registry.register("quantized_kv_write", Platform.CUDA, Backend.GPU)
def quantized_kv_write(
    keys: Float[Array, "total_tokens num_kv_heads head_dim"],
    values: Float[Array, "total_tokens num_kv_heads head_dim"],
    kv_pages: Shaped[Array, "num_pages num_kv_heads 2 page_size head_dim"],
    kv_scales: Float[Array, "num_pages num_kv_heads 2 blocks_per_page"],
    slot_mapping: Int32[Array, "total_tokens"],
) -> tuple[Array, Array]:
    """Write a step's rows to the 8-bit cache IN PLACE; returns ``(kv_pages, kv_scales)``, the same tensors.

    ``slot_mapping`` is that of ``build_page_tables``: negative slots are skipped, the rows of one scale block are
    neighbours with ascending slots, and no slot occurs twice.  The scale of a block is the smallest power of two under
    which its largest value is still a code; when a later row needs a larger one, the rows that the block holds already
    move to it (exactly for e4m3 above its subnormal range, by rounding once more otherwise).  ``read_status`` reports
    NaN and infinities among the rows.
    """
    try:
        key = (keys.shape, keys.dtype, keys.stride(), keys.get_device(), values.shape, values.dtype, values.stride(), values.get_device(),
               kv_pages.shape, kv_pages.dtype, kv_pages.is_contiguous(), kv_pages.get_device(),
               kv_scales.shape, kv_scales.dtype, kv_scales.is_contiguous(), kv_scales.get_device(),
               slot_mapping.shape, slot_mapping.dtype, slot_mapping.is_contiguous(), slot_mapping.get_device(), "write")
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        plan = _remember(key, _plan_write(keys, values, kv_pages, kv_scales, slot_mapping))
    shape, shape_ref, key_stride, value_stride, device = plan
    if shape.total_tokens == 0:
        return kv_pages, kv_scales
    if device.index != _current_device():
        with torch.cuda.device(device):
            return quantized_kv_write(keys, values, kv_pages, kv_scales, slot_mapping)
    rc = _function("ejk_q8_write_launch")(
        keys.data_ptr(), values.data_ptr(), key_stride, value_stride, kv_pages.data_ptr(), kv_scales.data_ptr(),
        slot_mapping.data_ptr(), _status_word(device), shape_ref, _raw_stream(device.index))
    if rc:
        _cabi.check(rc, "ejk_q8_write_launch")
    return kv_pages, kv_scales


@_checked
def _plan_read(
    kv_pages: Shaped[Array, "num_pages num_kv_heads two page_size head_dim"],
    kv_scales: Float[Array, "num_pages num_kv_heads two blocks_per_page"],
    slot_mapping: Int32[Array, "rows"],
    dtype: torch.dtype,
):
    block = _check_cache(kv_pages, kv_scales)
    if dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"dtype {dtype} is not supported by the CUDA path (bf16/f16 only)")
    if kv_scales.dtype != torch.float32:
        raise ValueError(f"kv_scales must be float32, got {kv_scales.dtype}")
    _contiguous(slot_mapping=slot_mapping)
    _on_one_device("kv_pages", kv_pages.device, kv_scales=kv_scales, slot_mapping=slot_mapping)
    _need_cuda("quantized_kv_read", kv_pages)
    P, Hkv, _, page_size, D = kv_pages.shape
    rows = slot_mapping.shape[0]
    shape = _cabi.Q8Shape(rows, 1, 1, P, page_size, Hkv, Hkv, D, _DTYPE_CODE[dtype], CODE_DTYPES[kv_pages.dtype], block)
    return shape, ctypes.byref(shape), _template((rows, Hkv, D), dtype, kv_pages.device)


@serving_registry.register("quantized_kv_read", Platform.CUDA, Backend.GPU)
def quantized_kv_read(
    kv_pages: Shaped[Array, "num_pages num_kv_heads 2 page_size head_dim"],
    kv_scales: Float[Array, "num_pages num_kv_heads 2 blocks_per_page"],
    slot_mapping: Int32[Array, "rows"],
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[Array, Array]:
    """The cache's rows at ``slot_mapping`` in 16 bits: ``(keys, values)``, each ``[rows, num_kv_heads, head_dim]``.

    A value beyond the range of ``dtype`` saturates, a code that is a NaN gives a NaN; a negative slot gives a row of zeros.
    """
    try:
        key = (kv_pages.shape, kv_pages.dtype, kv_pages.is_contiguous(), kv_pages.get_device(),
               kv_scales.shape, kv_scales.dtype, kv_scales.is_contiguous(), kv_scales.get_device(),
               slot_mapping.shape, slot_mapping.dtype, slot_mapping.is_contiguous(), slot_mapping.get_device(), dtype, "read")
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        plan = _remember(key, _plan_read(kv_pages, kv_scales, slot_mapping, dtype))
    shape, shape_ref, like = plan
    device = like.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return quantized_kv_read(kv_pages, kv_scales, slot_mapping, dtype=dtype)
    keys, values = torch.empty_like(like), torch.empty_like(like)
    if shape.total_tokens:
        rc = _function("ejk_q8_read_launch")(
            kv_pages.data_ptr(), kv_scales.data_ptr(), slot_mapping.data_ptr(), keys.data_ptr(), values.data_ptr(),
            _status_word(device), shape_ref, _raw_stream(device.index))
        if rc:
            _cabi.check(rc, "ejk_q8_read_launch")
    return keys, values


# ------------------------------------------------------------------------------------------- page tables


@_checked
def _plan_tables(
    query_lens: Int32[Array, "num_seqs"],
    context_lens: Int32[Array, "num_seqs"],
    block_tables: Int32[Array, "num_seqs pages_per_seq"],
    free_pages: Int32[Array, "capacity"],
    num_free: Int32[Array, "1"],
    finished: Bool[Array, "num_seqs"] | None,
    page_size: int,
    total_tokens: int,
):
    S, pps = block_tables.shape
    if S < 1 or pps < 1 or free_pages.shape[0] < 1:
        raise ValueError(f"block_tables {tuple(block_tables.shape)} and free_pages {tuple(free_pages.shape)} must not be empty")
    if S > 16384:
        raise NotImplementedError(f"{S} sequences: the CUDA path holds the sums of 16384 rows")
    if page_size < 1 or pps * page_size > 0x3FFFFFFF:
        raise ValueError(f"{page_size=} with {pps} pages per sequence: must be positive, and below 2^30 tokens in all")
    if not 0 <= total_tokens <= 0x3FFFFFFF:
        raise ValueError(f"{total_tokens=} must be in [0, 2^30)")
    _contiguous(query_lens=query_lens, context_lens=context_lens, block_tables=block_tables, free_pages=free_pages,
                num_free=num_free, finished=finished)
    _on_one_device("block_tables", block_tables.device, query_lens=query_lens, context_lens=context_lens,
                   free_pages=free_pages, num_free=num_free, finished=finished)
    _need_cuda("build_page_tables", block_tables)
    like = _template((2 * S + 2 + total_tokens,), torch.int32, block_tables.device)
    return S, pps, free_pages.shape[0], like, (S, S + 1, total_tokens, 1)


@serving_registry.register("build_page_tables", Platform.CUDA, Backend.GPU)
def build_page_tables(
    query_lens: Int32[Array, "num_seqs"],
    context_lens: Int32[Array, "num_seqs"],
    block_tables: Int32[Array, "num_seqs pages_per_seq"],
    free_pages: Int32[Array, "capacity"],
    num_free: Int32[Array, "1"],
    num_seqs: Array | int,
    *,
    page_size: int,
    total_tokens: int,
    finished: Bool[Array, "num_seqs"] | None = None,
) -> tuple[Array, Array, Array, Array]:
    """Page tables and slot maps of one step, on the device: ``(context_lens, query_start_loc, slot_mapping, num_free)``.

    ``context_lens`` goes in as the tokens that a request has cached and comes out with this step's ``query_lens`` added:
    the lengths that attention takes.  ``block_tables`` and the stack ``free_pages`` (its first ``num_free`` entries are
    free) are updated IN PLACE: the pages of ``finished`` rows go on top, then each row in order takes from the top what
    its new tokens need.  A finished row takes no tokens in this call and comes out with length 0; its slot of the batch
    can be given to a new request with the next call.  ``slot_mapping`` has ``total_tokens`` entries,
    ``page * page_size + offset`` each, -1 behind the last sequence and for rows that could not be served (the stack ran
    out, the row's table is too short, the batch exceeds ``total_tokens``): such a row keeps its length and takes no page,
    and ``read_status`` says so.  What attention returns for its query rows is to be dropped (they count in
    ``query_start_loc``, and are taken as the last tokens of the old length); its new length is its old one.  Nothing is read
    back by the host, so the call can be captured into a graph.
    """
    try:
        key = (query_lens.shape, query_lens.dtype, query_lens.is_contiguous(), query_lens.get_device(),
               context_lens.shape, context_lens.dtype, context_lens.is_contiguous(), context_lens.get_device(),
               block_tables.shape, block_tables.dtype, block_tables.is_contiguous(), block_tables.get_device(),
               free_pages.shape, free_pages.dtype, free_pages.is_contiguous(), free_pages.get_device(),
               num_free.shape, num_free.dtype, num_free.get_device(),
               None if finished is None else (finished.shape, finished.dtype, finished.is_contiguous(), finished.get_device()),
               page_size, total_tokens, "tables")
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        plan = _remember(key, _plan_tables(query_lens, context_lens, block_tables, free_pages, num_free, finished, page_size, total_tokens))
    S, pps, capacity, like, sizes = plan
    device = like.device
    index = device.index
    if index != _current_device():
        with torch.cuda.device(device):
            return build_page_tables(query_lens, context_lens, block_tables, free_pages, num_free, num_seqs, page_size=page_size,
                                     total_tokens=total_tokens, finished=finished)
    num_seqs = _count(num_seqs, device)
    out = torch.empty_like(like)  # one allocation for the four results
    base = out.data_ptr()
    at_slots = base + 4 * (2 * S + 1)
    rc = _function("ejk_page_tables_launch")(
        query_lens.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(),
        num_free.data_ptr(), num_seqs.data_ptr(), None if finished is None else finished.data_ptr(), base, base + 4 * S,
        at_slots if total_tokens else None, at_slots + 4 * total_tokens, _status_word(device), S, pps, page_size, capacity,
        total_tokens, _raw_stream(index))
    if rc:
        _cabi.check(rc, "ejk_page_tables_launch")
    return out.split_with_sizes(sizes)
