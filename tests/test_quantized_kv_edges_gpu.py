"""The operators around the 8-bit cache at the edges of what a call may hold: scales far apart under a mask, offsets that
describe no batch, NaN, the largest scale, table sizes around the shared-memory limit, a first call under capture.

Attention is checked row by row: with the bounds of test_quantized_kv_gpu.py, but the last term, what underflows, is taken of the
largest |V| among the keys that the ROW sees, so that a key which the mask hides from a row cannot excuse an error in it.
"""

import subprocess
import sys
import textwrap
from pathlib import Path

import numpy as np
import pytest
import torch

import ejkernel_b200 as ej
from ejkernel_b200 import _cabi
from ejkernel_b200.kernels._cuda.quantized_kv import read_status
from oracle import q8_oracle

from .test_quantized_kv_gpu import CODES, HALVES, clean_status, make_batch, make_cache, make_requests, check_tables, option, oracle, run  # noqa: F401

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def visible_top(b, window=None):
    """[T, Hq, 1]: the largest |V| among the keys that a row sees."""
    v = np.abs(q8_oracle.values_of(b["codes"], b["scales"])[:, :, 1]).max(-1)  # [P, Hkv, page]
    T, Hq, _ = b["q"].shape
    Hkv = v.shape[1]
    out = np.zeros((T, Hq, 1))
    start, tab = b["start"].tolist(), b["tab"].numpy()
    for s in range(b["n"]):
        n, kv = start[s + 1] - start[s], int(b["ctx"][s])
        keys = v[tab[s, : -(-kv // v.shape[2])]].transpose(1, 0, 2).reshape(Hkv, -1)[:, :kv]
        for r in range(n):
            pos = kv - n + r
            seen = keys[:, max(0, pos - window + 1) if window else 0: pos + 1]
            if seen.shape[1]:
                out[start[s] + r, :, 0] = np.repeat(seen.max(1), Hq // Hkv)
    return out


def check_rows(b, out, **kw):
    want, bound = oracle(b, **kw)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    exact_scales = bool((torch.frexp(b["scales"]).mantissa == 0.5).all())
    room = (2.0**-10 if exact_scales else 2.0**-9) * bound + torch.finfo(out.dtype).eps / 2 * (1 + 2.0**-6) * np.abs(want) \
        + 2.0**-24 * visible_top(b, kw.get("sliding_window")) + torch.finfo(out.dtype).tiny
    worst = (np.abs(got - want) / room).max()
    assert worst <= 1.0, worst


def launches():
    return _cabi.load().ejk_rpa_last_launch_count()


def set_v_scales(b, of):
    """V scale of the block that token j of every sequence lies in: of(sequence, first token of the block)."""
    page, per = b["codes"].shape[3], b["scales"].shape[3]
    block = page // per
    for s in range(b["n"]):
        for j in range(0, int(b["ctx"][s]), block):
            b["scales"][int(b["tab"][s, j // page]), :, 1, j % page // block] = of(s, j)


# ------------------------------------------------------------------- a row's result and the scales that it does not see


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim, Hq", [(64, 2), (128, 2), (256, 2), (64, 9), (128, 9), (256, 9)])
@pytest.mark.parametrize("window", [None, 40])
def test_split_kv_rows_do_not_feel_scales_that_their_mask_hides(code, dim, Hq, window):
    """Few tokens share a row tile.  Causally the first ones must not lose what later tokens' large values push out of f16; with
    a window the last ones must not feel the large values that have left their window."""
    b = make_batch([(3, 200), (2, 33), (3, 3), (1, 90)], Hq=Hq, Hkv=1, dim=dim, page=16, block=1, code=code, half=torch.bfloat16, seed=dim + Hq)
    ctx = b["ctx"].tolist()
    set_v_scales(b, lambda s, j: 2.0**-40 if (j < ctx[s] - 2 if window is None else j > ctx[s] - 42) else 1.0)
    kw = {} if window is None else dict(sliding_window=window)
    check_rows(b, run(b, **kw), **kw)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block, kw", [(1, {}), (8, {}), (16, {}), (8, dict(logits_soft_cap=5.0)), (2, dict(softmax_scale=-0.1))])
def test_prompt_rows_do_not_feel_scales_that_the_causal_mask_hides(code, dim, block, kw):
    """A prefix of small values, then large ones in the same 64-token stage and in later ones."""
    b = make_batch([(200, 200), (90, 333), (40, 40)], Hq=4, Hkv=2, dim=dim, page=16, block=block, code=code, half=torch.bfloat16, seed=dim + block)
    ctx = b["ctx"].tolist()
    set_v_scales(b, lambda s, j: 2.0**-40 if j < (48, ctx[1] - 48, 16)[s] else 1.0)
    check_rows(b, run(b, **kw), **kw)


@pytest.mark.parametrize("split", [0, 2])
@pytest.mark.parametrize("dim, block", [(64, 4), (128, 16)])
def test_prompt_rows_do_not_feel_scales_that_left_their_window(option, dim, block, split):
    """Large values first: rows whose window has passed them see small ones alone, in the same stage and in later ones."""
    option("prefill_split", split)
    b = make_batch([(300, 700), (250, 250)], Hq=4, Hkv=2, dim=dim, page=16, block=block, code=torch.int8, half=torch.bfloat16, seed=dim)
    first = [400, 0]
    set_v_scales(b, lambda s, j: 1.0 if j < first[s] + 16 else 2.0**-40)
    check_rows(b, run(b, sliding_window=50), sliding_window=50)


@pytest.mark.parametrize("rows", [3, 100])
@pytest.mark.parametrize("half", HALVES)
@pytest.mark.parametrize("any_scale", [False, True])
def test_scales_far_apart_row_by_row(rows, half, any_scale):
    far = 30 if half == torch.bfloat16 else 6
    b = make_batch([(rows, 260), (1, 150), (rows, rows)], Hq=4, Hkv=1, dim=64, page=16, block=8, code=torch.float8_e4m3fn, half=half, seed=rows, any_scale=any_scale)
    b["scales"][:, :, 1] *= torch.exp2(torch.randint(-far, far - 2, b["scales"][:, :, 1].shape, generator=torch.Generator().manual_seed(2)).float())
    sinks = torch.randn((4, 2), generator=torch.Generator().manual_seed(1))
    check_rows(b, run(b))
    check_rows(b, run(b, sliding_window=37), sliding_window=37)
    check_rows(b, run(b, sinks=sinks), sinks=sinks)


@pytest.mark.parametrize("rows, split", [(1, 1), (100, 0), (100, 2)])
def test_values_near_the_smallest_normal_number(option, rows, split):
    """Scales of 2^-120 over many keys of equal weight: the sum is undone by the scales' power of two and by the weights' sum, one
    after the other; their product alone would be below what float32 holds."""
    option("prefill_split", split)
    b = make_batch([(rows, 4000)], Hq=2, Hkv=1, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=5)
    b["codes"][:, :, 1] = torch.randint(60, 128, b["codes"][:, :, 1].shape, generator=torch.Generator().manual_seed(3)).to(torch.int8)
    b["scales"][:, :, 1] = 2.0**-120
    b["q"] = b["q"] * 0.01
    check_rows(b, run(b))


# ---------------------------------------------------------------------------------- numbers at the end of their types


@pytest.mark.parametrize("rows", [1, 90])
def test_windows_beyond_32_bits_hide_nothing(rows):
    b = make_batch([(rows, 200), (1, 33)], Hq=4, Hkv=2, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=24)
    want = run(b)
    for window in (2**31 - 1, 2**31, 2**32 + 5):
        assert torch.equal(run(b, sliding_window=window), want)
    hint = ej.RaggedPageAttentionConfig(num_kv_pages_per_block=None, num_queries_per_block=2**32 + 1)
    check_rows(b, run(b, cfg=hint))
    assert launches() == 1


@pytest.mark.parametrize("rows, page", [(1, 16), (90, 16), (3, 5)])
@pytest.mark.parametrize("cap", [1000.0, 5e3, -2e5, 1e9, 2.0**100])
def test_large_soft_caps(rows, page, cap):
    """cap * tanh(x / cap) of logits far below the cap: 1 - 2 / (e^2t + 1) would lose them, cap * 2^-22 each."""
    b = make_batch([(rows, 200), (1, 33)], Hq=4, Hkv=2, dim=64, page=page, block=1, code=torch.int8, half=torch.float16, seed=26)
    check_rows(b, run(b, logits_soft_cap=cap), logits_soft_cap=cap)
    b["q"] = b["q"] * 30
    check_rows(b, run(b, logits_soft_cap=cap, softmax_scale=0.02), logits_soft_cap=cap, softmax_scale=0.02)


@pytest.mark.parametrize("rows", [1, 90])
@pytest.mark.parametrize("kw", [dict(logits_soft_cap=2.0**-90, softmax_scale=1.0), dict(softmax_scale=2.0**-140)])
def test_caps_and_scales_at_the_ends_of_float32(rows, kw):
    b = make_batch([(rows, 200), (1, 33)], Hq=4, Hkv=2, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=25)
    check_rows(b, run(b, **kw), **kw)


# ------------------------------------------------------------------------------------ rows that no sequence serves


def poisoned(b, **kw):
    """The call's output where the memory that it gets was full of NaN."""
    run(b, **kw)
    torch.cuda.synchronize()
    for _ in range(3):  # the allocator gives a freed block of the size to the next call
        t = torch.full(b["q"].shape, float("nan"), dtype=b["q"].dtype, device="cuda")
        del t
        out = run(b, **kw)
        assert torch.isfinite(out).all()
    return out


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("start, served", [([0, 1, 900], {0}), ([2, 3, 5], {2, 3, 4}), ([-3, 2, 4], {2, 3}), ([0, 3, 3000], {0, 1, 2}), ([7, 7, 7], set()), ([0, 0, -4], set())])
def test_rows_under_bad_offsets_are_zero(page, start, served):
    b = make_batch([(1, 40), (6, 30)], Hq=4, Hkv=2, dim=64, page=page, block=1, code=torch.int8, half=torch.bfloat16, seed=12)
    out = poisoned(b | dict(start=torch.tensor(start, dtype=torch.int32)))
    read_status()
    for t in range(7):
        assert bool(out[t].any()) == (t in served), t


@pytest.mark.parametrize("page", [16, 5])
def test_prompt_rows_under_bad_offsets_are_zero(page):
    b = make_batch([(100, 140), (120, 130)], Hq=4, Hkv=2, dim=64, page=page, block=1, code=torch.int8, half=torch.bfloat16, seed=13)
    out = poisoned(b | dict(start=torch.tensor([0, 100, 221], dtype=torch.int32)))
    assert read_status() & _cabi.ST_QLEN
    assert bool(out[:100].any(-1).all()) and not bool(out[100:].any())


def test_rows_are_zero_where_overlapping_offsets_need_more_items_than_there_are():
    """Each of five sequences claims all 1000 rows: more 128-row items than 1000 tokens can make."""
    b = make_batch([(1000, 1000)], Hq=4, Hkv=1, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=14)
    b["tab"], b["ctx"] = b["tab"].repeat(9, 1), b["ctx"].repeat(9)
    b["start"], b["n"] = torch.tensor([0, 1000] * 5, dtype=torch.int32), 9
    out = poisoned(b)
    assert read_status() & _cabi.ST_INTERNAL
    assert not bool(out.any())


# ------------------------------------------------------------------------------------------------ write and read


@pytest.mark.parametrize("half", HALVES)
def test_read_gives_a_nan_back_as_a_nan(half):
    g = torch.Generator().manual_seed(6)
    kv, scales = make_cache(g, 2, 1, 16, 64, torch.float8_e4m3fn, 16)
    codes = kv.view(torch.uint8).clone()
    codes[0, 0, 0, 3, 7], codes[1, 0, 1, 2, 0] = 0x7F, 0xFF
    kv, scales = codes.view(torch.float8_e4m3fn).cuda(), scales.cuda()
    slots = torch.arange(32, dtype=torch.int32, device="cuda")
    for which, got in enumerate(ej.quantized_kv_read(kv, scales, slots, dtype=half)):
        want = (kv.float() * scales.repeat_interleave(16, 3)[..., None])[:, 0, which].reshape(32, 1, 64)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(got).sum()) == 1


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("exponent", [127, 126, 125])
def test_write_behind_rows_of_the_largest_scales(code, exponent):
    """Kept rows stand under a scale of 2^127, the largest power of two there is: its inverse is no normal number."""
    g = torch.Generator().manual_seed(exponent)
    kv, scales = make_cache(g, 2, 1, 16, 64, code, 16)
    kv.view(torch.uint8).zero_()
    scales[:] = 2.0**exponent
    x = torch.randn((3, 1, 64), generator=g, dtype=torch.float64).mul(2.0**124).clamp(-3e38, 3e38).to(torch.bfloat16)
    x[0, 0, 0], x[0, 0, 1] = 3e38, -3e38
    slots = torch.tensor([17, 18, 19], dtype=torch.int32)
    want_c, want_s = q8_oracle.write(x, x, kv, scales, slots)
    kv, scales = kv.cuda(), scales.cuda()
    ej.quantized_kv_write(x.cuda(), x.cuda(), kv, scales, slots.cuda())
    assert np.array_equal(scales.cpu().double().numpy(), want_s)
    assert np.array_equal(kv.cpu().float().double().numpy(), want_c) and want_c.any()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim, page, block", [(64, 16, 16), (128, 16, 4), (256, 24, 8), (64, 5, 1)])
def test_write_to_pages_in_any_order(code, dim, page, block):
    """Rows that go on in a lower or a distant page."""
    g = torch.Generator().manual_seed(dim + page)
    kv, scales = make_cache(g, 40, 2, page, dim, code, block)
    order, at, slots = torch.randperm(40, generator=g), 0, []
    for c, n in ((3, 2 * page), (page - 1, 3 * page + 2), (0, 1), (page // 2, 4 * page)):
        held = -(-(c + n) // page)
        pos = torch.arange(c, c + n)
        slots.append(order[at: at + held][pos // page] * page + pos % page)
        at += held
    slots = torch.cat(slots).to(torch.int32)
    x = (torch.randn((slots.numel(), 2, dim), generator=g) * torch.exp2(torch.randint(-9, 4, (slots.numel(), 2, 1), generator=g).float())).to(torch.float16)
    want_c, want_s = q8_oracle.write(x, -x, kv, scales, slots)
    kv, scales = kv.cuda(), scales.cuda()
    ej.quantized_kv_write(x.cuda(), (-x).cuda(), kv, scales, slots.cuda())
    assert np.array_equal(scales.cpu().double().numpy(), want_s) and np.array_equal(kv.cpu().float().double().numpy(), want_c)


# -------------------------------------------------------------------------------------------------- page tables


@pytest.mark.parametrize("rows", [2731, 4050, 4063, 4064, 4096, 4097, 16384])
def test_tables_of_rows_around_the_plain_shared_memory_limit(rows):
    """In a process of its own: once a larger table has raised the kernel's limit, the sizes below are served too."""
    code = f"""
        from tests.test_quantized_kv_gpu import check_tables, make_requests
        check_tables(make_requests([1, 0, 20, 3], [0, 17, 5, 16], page=16, pps=8, seed=1, rows={rows}), 16, 30)
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------------------ dispatch


@pytest.mark.parametrize("dim", [64, 128])
def test_the_query_hint_counts_in_a_padded_table_too(dim):
    """One chunk in a table of more rows than the batch has tokens: with the hint it is served by tensor tiles (three launches)."""
    b = make_batch([(200, 333), (1, 50), (3, 60)], Hq=4, Hkv=2, dim=dim, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=21, rows=256)
    check_rows(b, run(b))
    assert launches() == 1
    out = run(b, cfg=ej.RaggedPageAttentionConfig(num_kv_pages_per_block=None, num_queries_per_block=64))
    assert launches() == 3
    check_rows(b, out)
    # a hint that no sequence of the batch can reach spares the plan
    check_rows(b, run(b, cfg=ej.RaggedPageAttentionConfig(num_kv_pages_per_block=None, num_queries_per_block=205)))
    assert launches() == 1


@pytest.mark.parametrize("dim, Hq", [(64, 9), (64, 16), (256, 9), (256, 16)])
@pytest.mark.parametrize("code, half", [(torch.int8, torch.bfloat16), (torch.int8, torch.float16), (torch.float8_e4m3fn, torch.bfloat16), (torch.float8_e4m3fn, torch.float16)])
def test_more_than_eight_heads_per_kv_head(code, half, dim, Hq):
    b = make_batch([(1, 300), (2, 77), (1, 9), (1, 2500)], Hq=2 * Hq, Hkv=2, dim=dim, page=16, block=8, code=code, half=half, seed=Hq)
    check_rows(b, run(b))


# ------------------------------------------------------------------------------------------------------- capture


def test_the_first_call_of_a_process_is_captured():
    """The status word outlives the graph, and reports what its replays meet."""
    code = """
        import torch
        import ejkernel_b200 as ej
        from ejkernel_b200 import _cabi
        from ejkernel_b200.kernels._cuda.quantized_kv import read_status

        kv, scales = ej.allocate_quantized_kv(4, 1, 16, 64, dtype=torch.int8)
        x = torch.ones((3, 1, 64), dtype=torch.bfloat16, device="cuda")
        slots = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ej.quantized_kv_write(x, x, kv, scales, slots)
        graph.replay()
        assert read_status() == 0
        assert bool(kv[0, 0, :, 5:8].any(-1).all())
        slots.fill_(1 << 20)
        graph.replay()
        assert read_status() == _cabi.ST_PAGE_ID
        slots.copy_(torch.tensor([5, 6, 7]))
        x[1, 0, 3] = float("nan")
        for _ in range(2):
            graph.replay()
        assert read_status(clear=False) == _cabi.ST_NONFINITE and read_status() == _cabi.ST_NONFINITE and read_status() == 0
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("kind", ["int", "host"])
def test_a_number_of_sequences_that_the_host_holds_is_captured(kind):
    """A count that no call has used before is part of the graph, and stays what it was when the process forgets old counts."""
    from ejkernel_b200.kernels._cuda.ragged_page_attention import _interface

    b = make_batch([(1, 100), (2, 40), (1, 70)], Hq=4, Hkv=1, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=23, rows=5)
    gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}
    want = run(gpu)
    _interface._num_seqs_consts.clear()
    if kind == "host":
        gpu["n"] = torch.tensor([3])
    args = (gpu["q"], gpu["codes"], gpu["scales"], gpu["ctx"], gpu["tab"], gpu["start"], gpu["n"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ej.quantized_ragged_page_attention(*args)
    _interface._num_seqs_consts.clear()
    keep = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(64)]
    graph.replay()
    assert torch.equal(out, want) and keep
