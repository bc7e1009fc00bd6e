"""Calls of the operators around the 8-bit cache that are refused on the host: pointers that a kernel would read at a misaligned
address, numbers that float32 or int32 do not hold.  None of them reaches a GPU."""

import ctypes

import pytest
import torch

from ejkernel_b200 import _cabi

from .test_quantized_kv import attend, make

ONE = 1 << 20  # not memory: a refusal never follows a pointer
SHAPE = dict(total_tokens=4, max_num_seqs=2, pages_per_seq=2, num_pages=4, page_size=16, num_q_heads=4, num_kv_heads=2,
             head_dim=64, dtype=0, code_dtype=3, scale_block=16)


@pytest.mark.parametrize("which", ["kv_scales", "context_lens", "block_tables", "query_start_loc", "num_seqs", "softmax_aux", "status"])
@pytest.mark.parametrize("by", [1, 2])
def test_attention_refuses_four_byte_operands_off_their_boundary(rpa_lib, which, by):
    at = dict(kv_scales=ONE, context_lens=ONE, block_tables=ONE, query_start_loc=ONE, num_seqs=ONE, softmax_aux=ONE, status=ONE)
    at[which] += by
    attrs = _cabi.Attrs(1.0, 0.0, 0, 2, 4, 0, 0, 0.0, 0.0)
    rc = rpa_lib.ejk_q8_attention_launch(ONE, ONE, at["kv_scales"], at["context_lens"], at["block_tables"], at["query_start_loc"], at["num_seqs"],
                                         at["softmax_aux"], ONE, ONE, 1 << 30, at["status"], ctypes.byref(_cabi.Q8Shape(**SHAPE)), ctypes.byref(attrs), None)
    assert rc == -8


@pytest.mark.parametrize("which", ["kv_scales", "slots", "status"])
def test_write_and_read_refuse_four_byte_operands_off_their_boundary(rpa_lib, which):
    at = dict(kv_scales=ONE, slots=ONE, status=ONE)
    at[which] += 2
    shape = ctypes.byref(_cabi.Q8Shape(**SHAPE))
    assert rpa_lib.ejk_q8_write_launch(ONE, ONE, 128, 128, ONE, at["kv_scales"], at["slots"], at["status"], shape, None) == -8
    assert rpa_lib.ejk_q8_read_launch(ONE, at["kv_scales"], at["slots"], ONE, ONE, at["status"], shape, None) == -8


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4, 5, 7, 8, 9, 10, 11])  # 6 is `finished`, of bytes
def test_page_tables_refuse_operands_off_their_boundary(rpa_lib, which):
    at = [ONE] * 12
    at[which] += 2
    assert rpa_lib.ejk_page_tables_launch(*at, 2, 2, 16, 8, 4, None) == -8


@pytest.mark.parametrize("kw", [dict(logits_soft_cap=1e-60), dict(logits_soft_cap=-1e-44), dict(logits_soft_cap=1e60), dict(logits_soft_cap=3e30),
                                dict(softmax_scale=1e60), dict(softmax_scale=-3e38), dict(logits_soft_cap=1e-30, softmax_scale=1e30)])
def test_attention_refuses_numbers_that_float32_does_not_hold(kw):
    """A cap that rounds to zero would be no cap; one whose quotient overflows makes NaN of a logit of zero."""
    with pytest.raises(ValueError, match="float32"):
        attend(make(), **kw)


@pytest.mark.parametrize("scale, cap", [(3e38, 0.0), (1.0, 3e30), (1.0, 1e-44), (1e30, 1e-30)])
def test_the_c_entry_refuses_factors_that_overflow(rpa_lib, scale, cap):
    attrs = _cabi.Attrs(scale, cap, 0, 0, 0, 0, 0, 0.0, 0.0)
    rc = rpa_lib.ejk_q8_attention_launch(*[ONE] * 7, None, ONE, ONE, 1 << 30, None, ctypes.byref(_cabi.Q8Shape(**SHAPE)), ctypes.byref(attrs), None)
    assert rc == -6
