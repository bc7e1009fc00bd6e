"""The serving step over an 8-bit cache, on the CPU: refusals, the plain forms against their definitions, the C entry points'
argument checks.  Numbers of the kernels are checked in test_quantized_kv_gpu.py."""

import ctypes
import inspect
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import ejkernel_b200 as ej
from ejkernel_b200 import _cabi
from oracle import q8_oracle
from oracle.rpa_oracle import dense_reference

ROOT = Path(__file__).resolve().parent.parent


def make(pages=4, heads=2, page=16, dim=64, block=16, code=torch.int8, T=3, Hq=4, S=2, pps=2):
    kv, scales = ej.modules.operations.allocate_quantized_kv(pages, heads, page, dim, dtype=code, scale_block=block, device="cpu")
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    return dict(queries=torch.zeros(T, Hq, dim, dtype=torch.bfloat16), kv_pages=kv, kv_scales=scales, context_lens=i32(S),
                block_tables=i32(S, pps), query_start_loc=i32(S + 1), num_seqs=1)


def attend(c, **kw):
    return ej.quantized_ragged_page_attention(c["queries"], c["kv_pages"], c["kv_scales"], c["context_lens"], c["block_tables"],
                                              c["query_start_loc"], c["num_seqs"], **kw)


def test_registered_apart_from_the_reference_algorithms():
    names = ["build_page_tables", "quantized_kv_read", "quantized_kv_write", "quantized_ragged_page_attention"]
    assert ej.serving_registry.list_algorithms() == names
    assert not set(names) & set(ej.kernel_registry.list_algorithms())
    assert ej.serving_registry.validate_signatures()
    for name in names:
        public = inspect.signature(getattr(ej, name)).parameters
        for p in inspect.signature(ej.serving_registry.get(name, "cuda", "gpu")).parameters.values():
            if not p.name.startswith("num_kv_pages") and not p.name.startswith("num_queries"):
                assert public[p.name].default == p.default, (name, p.name)
        with pytest.raises(ValueError, match="only the CUDA"):
            getattr(ej, name)(*[None] * sum(p.kind.name == "POSITIONAL_ONLY" for p in public.values()), platform="triton",
                              **{p.name: 1 for p in public.values() if p.default is p.empty and p.kind.name == "KEYWORD_ONLY"})


def test_no_cpu_fallback():
    c = make()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attend(c)
    kv = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ej.quantized_kv_write(kv, kv, c["kv_pages"], c["kv_scales"], slots)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ej.quantized_kv_read(c["kv_pages"], c["kv_scales"], slots)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ej.build_page_tables(i, i, c["block_tables"], i, i[:1], 2, page_size=16, total_tokens=4)


@pytest.mark.parametrize("change, error", [
    (dict(queries=torch.zeros(3, 4, 64)), NotImplementedError),                               # float32 queries
    (dict(queries=torch.zeros(3, 3, 64, dtype=torch.float16)), ValueError),                   # 3 heads over 2
    (dict(queries=torch.zeros(3, 8, 64, dtype=torch.float16)[:, ::2]), ValueError),           # not dense
    (dict(kv_pages=torch.zeros(4, 2, 2, 16, 64, dtype=torch.float8_e5m2)), NotImplementedError),
    (dict(kv_pages=torch.zeros(4, 2, 3, 16, 64, dtype=torch.int8), kv_scales=torch.ones(4, 2, 3, 1)), ValueError),
    (dict(kv_scales=torch.ones(4, 2, 2, 3)), ValueError),                                     # 3 does not divide 16
    (dict(kv_scales=torch.ones(4, 2, 2, 1, dtype=torch.float16)), ValueError),
    (dict(kv_scales=torch.ones(4, 2, 2, 0)), ValueError),
    (dict(query_start_loc=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(block_tables=torch.zeros(2, 0, dtype=torch.int32)), ValueError),
    (dict(sliding_window=0), ValueError),
    (dict(logits_soft_cap=0.0), ValueError),
    (dict(logits_soft_cap=float("inf")), ValueError),
    (dict(softmax_scale=float("nan")), ValueError),
    (dict(softmax_aux=torch.zeros(3, 1)), ValueError),
])
def test_attention_refuses(change, error):
    c = make()
    kw = {k: v for k, v in change.items() if k not in c}
    c.update({k: v for k, v in change.items() if k in c})
    with pytest.raises(error):
        attend(c, **kw)


@pytest.mark.parametrize("change", [
    dict(context_lens=torch.zeros(2, dtype=torch.int64)), dict(block_tables=torch.zeros(3, 2, dtype=torch.int32)),
    dict(queries=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), dict(kv_scales=torch.ones(4, 1, 2, 1)), dict(softmax_scale="1"),
])
def test_attention_checks_shapes_and_types_together(change):
    c = make()
    kw = {k: v for k, v in change.items() if k not in c}
    c.update({k: v for k, v in change.items() if k in c})
    with pytest.raises(Exception) as e:
        attend(c, **kw)
    assert "TypeCheck" in type(e.value).__name__ or "Beartype" in type(e.value).__name__


def test_a_block_of_tokens_is_a_power_of_two():
    c = make(page=24, block=8)
    c["kv_scales"] = torch.ones(4, 2, 2, 2)  # 12 tokens
    with pytest.raises(ValueError, match="power of two"):
        attend(c)
    with pytest.raises(ValueError, match="power of two"):
        ej.modules.operations.allocate_quantized_kv(1, 1, 24, 64, scale_block=12, device="cpu")
    kv, s = ej.modules.operations.allocate_quantized_kv(3, 2, 24, 64, device="cpu")
    assert kv.dtype == torch.float8_e4m3fn and s.shape == (3, 2, 2, 3)


def test_write_and_read_refuse():
    c = make()
    slots = torch.zeros(3, dtype=torch.int32)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for keys, values, error in ((rows.float(), rows.float(), NotImplementedError), (rows, rows.half(), NotImplementedError),
                                (torch.zeros(3, 4, 64, dtype=torch.bfloat16)[:, ::2], rows, ValueError),
                                (torch.zeros(3, 132, dtype=torch.bfloat16)[:, :128].unflatten(1, (2, 64)), rows, ValueError)):
        with pytest.raises(error):
            ej.quantized_kv_write(keys, values, c["kv_pages"], c["kv_scales"], slots)
    with pytest.raises(ValueError, match="contiguous"):
        ej.quantized_kv_write(rows, rows, c["kv_pages"], c["kv_scales"], torch.zeros(6, dtype=torch.int32)[::2])
    with pytest.raises(NotImplementedError):
        ej.quantized_kv_read(c["kv_pages"], c["kv_scales"], slots, dtype=torch.float32)


def test_page_tables_refuse_more_rows_than_their_sums_hold():
    i = torch.zeros(16385, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        ej.build_page_tables(i, i, torch.zeros(16385, 1, dtype=torch.int32), i, i[:1], 2, page_size=16, total_tokens=4)


@pytest.mark.parametrize("kw", [dict(page_size=0), dict(total_tokens=-1), dict(page_size=1 << 30), dict(total_tokens=1 << 30)])
def test_page_tables_refuse(kw):
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ej.build_page_tables(i, i, torch.zeros(2, 2, dtype=torch.int32), i, i[:1], 2, **(dict(page_size=16, total_tokens=4) | kw))


def test_library_exports_every_declared_symbol(rpa_lib):
    header = (ROOT / "include" / "ejk_q8.h").read_text()
    declared = set(re.findall(r"EJK_RPA_API\s+[\w\s\*]+?\b(ejk_\w+)\s*\(", header))
    assert declared == set(_cabi.Q8_EXPORTS)
    for name in declared:
        assert getattr(rpa_lib, name) is not None
    body = re.search(r"typedef struct ejk_q8_shape \{(.*?)\} ejk_q8_shape;", header, re.S).group(1)
    fields = re.findall(r"int32_t\s+(\w+);", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
    assert fields == [n for n, _ in _cabi.Q8Shape._fields_]


def test_c_entries_refuse_before_they_touch_anything(rpa_lib):
    """Every refusal answers with its code; the pointers are never followed (they are not memory)."""
    one = 1 << 20
    good = dict(total_tokens=4, max_num_seqs=2, pages_per_seq=2, num_pages=4, page_size=16, num_q_heads=4, num_kv_heads=2,
                head_dim=64, dtype=0, code_dtype=3, scale_block=16)
    attrs = _cabi.Attrs(1.0, 0.0, 0, 0, 0, 0, 0, 0.0, 0.0)

    def attention(shape=good, attrs=attrs, q=one, ws=one):
        return rpa_lib.ejk_q8_attention_launch(q, one, one, one, one, one, one, None, one, ws, 1 << 30, None,
                                               ctypes.byref(_cabi.Q8Shape(**shape)), ctypes.byref(attrs), None)

    def write(shape=good, stride=128, keys=one):
        return rpa_lib.ejk_q8_write_launch(keys, one, stride, 128, one, one, one, None, ctypes.byref(_cabi.Q8Shape(**shape)), None)

    def read(shape=good, keys=one):
        return rpa_lib.ejk_q8_read_launch(one, one, one, keys, one, None, ctypes.byref(_cabi.Q8Shape(**shape)), None)

    def tables(S=2, pps=2, page=16, cap=8, T=4, q=one):
        return rpa_lib.ejk_page_tables_launch(q, one, one, one, one, one, None, one, one, one, one, None, S, pps, page, cap, T, None)

    for call in (attention, write, read):
        for field, value, code in (("head_dim", 96, -3), ("dtype", 2, -4), ("code_dtype", 0, -4), ("scale_block", 12, -2),
                                   ("scale_block", 32, -2), ("scale_block", 0, -2), ("page_size", 0, -2), ("num_pages", 1 << 28, -2),
                                   ("num_kv_heads", 0, -2), ("total_tokens", 0, -2)):
            assert call(shape=good | {field: value}) == code, (call.__name__, field, value)
        assert call(**({"q": None} if call is attention else {"keys": None})) == -1
        assert call(**({"q": one + 8} if call is attention else {"keys": one + 8})) == -8
    assert attention(good | {"num_q_heads": 3}) == -2
    assert attention(ws=None) == -1
    for bad in (_cabi.Attrs(float("nan")), _cabi.Attrs(1.0, float("inf")), _cabi.Attrs(1.0, 0.0, 0, 2, 4), _cabi.Attrs(1.0, 0.0, 0, -1),
                _cabi.Attrs(1.0, 0.0, 0, 0, 0, 0, 0, 2.0), _cabi.Attrs(1.0, 0.0, 0, 0, 0, 0, 0, 0.0, 2.0)):
        assert attention(attrs=bad) == -6
    assert write(stride=64) == -2 and write(stride=132) == -8
    assert tables(q=None) == -1
    for kw in (dict(S=0), dict(S=16385), dict(pps=0), dict(page=0), dict(cap=0), dict(T=-1), dict(page=1 << 30), dict(T=1 << 30)):
        assert tables(**kw) == -2, kw
    assert rpa_lib.ejk_q8_workspace_bytes(None) == 0


# ------------------------------------------------------------------------------------- the plain forms themselves


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_oracle_codes_are_the_nearest_ones(code):
    x = np.concatenate([np.linspace(-q8_oracle.QMAX[code], q8_oracle.QMAX[code], 4001), 2.0 ** np.arange(-12, 8.0), [0.0, 0.0009765625 * 1.5]])
    x = np.clip(x, -q8_oracle.QMAX[code], q8_oracle.QMAX[code])  # 2^7 is no int8: values arrive clamped
    got = q8_oracle.round_to_code(x, code)
    t = torch.from_numpy(x)
    want = t.round().to(torch.int8).double() if code == torch.int8 else t.float().to(code).double()
    assert np.array_equal(got, want.numpy())
    for amax in (0.0, 1e-45, 1.0, 447.9, 448.0, 448.1, 127.0, 127.1, 3.0e38):
        s = q8_oracle.scale_for(amax, code)
        assert amax <= q8_oracle.QMAX[code] * s and (s == 2.0**-126 or amax > q8_oracle.QMAX[code] * s / 2)


def test_oracle_attention_agrees_with_the_dense_reference_of_the_16_bit_operator():
    g = torch.Generator().manual_seed(1)
    P, Hkv, page, D, Hq = 12, 2, 8, 64, 4
    kv16 = torch.randint(-30, 31, (P, page, 2 * Hkv, D), generator=g).float() / 16
    codes = (kv16 * 16).to(torch.int8).view(P, page, Hkv, 2, D).permute(0, 2, 3, 1, 4).contiguous()
    scales = torch.full((P, Hkv, 2, 2), 1 / 16)
    lens, starts = torch.tensor([20, 37, 5], dtype=torch.int32), torch.tensor([0, 4, 5, 10], dtype=torch.int32)
    tab = torch.randperm(P, generator=g)[:12].view(3, 4).to(torch.int32)
    tab = torch.cat([tab, tab[:, :1]], 1)
    q = torch.randn(10, Hq, D, generator=g)
    sinks = torch.randn(Hq, 2, generator=g)
    kw = dict(softmax_scale=0.3, sliding_window=9, logits_soft_cap=5.0, softmax_aux=sinks)
    want = dense_reference(q, kv16, lens, tab, starts, torch.tensor([3]), precision="fp64", **kw)
    got = q8_oracle.attention(q, codes, scales, lens, tab, starts, 3, softmax_scale=0.3, window=9, cap=5.0, sinks=sinks)
    assert np.abs(got - want).max() < 1e-6
