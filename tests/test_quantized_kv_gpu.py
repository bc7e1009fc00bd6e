"""The kernels of the 8-bit cache against plain restatements in 64 bits.

Tolerances.  Codes, scales and tables are compared for equality: every quotient is by a power of two, so a code has one
right value.  Attention multiplies codes as 16-bit floats (exact) and sums in float32; what it rounds is

  * the queries: f16 as they are; bf16 queries are scaled by a power of two and taken to f16, exact but for elements
    2^-28 below their row's largest -- nothing at this scale;
  * a weight, to f16: 2^-11 relative, or 2^-31 of the largest weight where it falls below f16's normal range.  The split-KV
    kernel rounds p_j * v_scale_j once; the tensor tiles round p_j, and v_scale_j and its product with a code, which are
    both exact where the scales are powers of two.  A weight's error hits the term p_j |v_j|;
  * the logits' sum of D products and the exponential in float32: relative error of a weight below |y| * D * 2^-24 +
    2^-21 with |y| the logit (a few units here, D <= 256): |y| 2^-16 at most, 2^-13 with |y| <= 8;
  * the output, to its type: half a step, eps / 2 relative.

So |out - exact| <= w * sum p |v| + (eps / 2) * (1 + 2^-6) * |exact| + 2^-24 * max |v|.  The first term holds the weights, with
room for the float32 sums: w = 2^-11 + 2^-13 taken as 2^-10, and 3 * 2^-11 + 2^-13 taken as 2^-9 where scales are no powers of
two; the last one what underflows.
"""

import numpy as np
import pytest
import torch

import ejkernel_b200 as ej
from ejkernel_b200 import _cabi
from ejkernel_b200.kernels._cuda.quantized_kv import read_status
from oracle import q8_oracle

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]
HALVES = [torch.bfloat16, torch.float16]


def make_cache(g, pages, heads, page, dim, code, block, any_scale=False):
    scales = torch.exp2(torch.randint(-7, -3, (pages, heads, 2, page // block), generator=g).float())
    if any_scale:
        scales = scales * (1 + torch.rand(scales.shape, generator=g))
    x = torch.randn((pages, heads, 2, page // block, block * dim), generator=g) / scales[..., None]
    x = x.clamp(-q8_oracle.QMAX[code], q8_oracle.QMAX[code])
    codes = (x.round() if code == torch.int8 else x).to(code).view(pages, heads, 2, page, dim)
    return codes, scales


def make_batch(lens, *, Hq, Hkv, dim, page, block, code, half, seed=0, any_scale=False, extra_rows=0, spare=3, rows=None):
    """lens: (query rows, keys) of each sequence; `rows` of the tables behind the last sequence are idle."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-kv // page) for _, kv in lens]
    pps = max(held + [1]) + 1
    pages = sum(held) + spare
    codes, scales = make_cache(g, pages, Hkv, page, dim, code, block, any_scale)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    S = rows or len(lens)
    tab = torch.full((S, pps), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        tab[i, :h] = order[at: at + h]
        at += h
    start = [0]
    for n, _ in lens:
        start.append(start[-1] + n)
    start += [start[-1]] * (S - len(lens))
    q = torch.randn((start[-1] + extra_rows, Hq, dim), generator=g).to(half)
    ctx = torch.tensor([kv for _, kv in lens] + [0] * (S - len(lens)), dtype=torch.int32)
    return dict(q=q, codes=codes, scales=scales, ctx=ctx, tab=tab, start=torch.tensor(start, dtype=torch.int32), n=len(lens))


def run(b, **kw):
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}
    aux = kw.pop("sinks", None)
    return ej.quantized_ragged_page_attention(c["q"], c["codes"], c["scales"], c["ctx"], c["tab"], c["start"], c["n"],
                                              softmax_aux=None if aux is None else aux.cuda(), **kw)


def oracle(b, **kw):
    return q8_oracle.attention(b["q"], b["codes"], b["scales"], b["ctx"], b["tab"], b["start"], b["n"], with_bound=True,
                               softmax_scale=kw.get("softmax_scale"), window=kw.get("sliding_window"), cap=kw.get("logits_soft_cap"),
                               sinks=kw.get("sinks"))


def check(b, out, **kw):
    want, bound = oracle(b, **kw)
    got = out.double().cpu().numpy()
    v_max = np.abs(q8_oracle.values_of(b["codes"], b["scales"])[:, :, 1]).max()
    assert np.isfinite(got).all()
    exact_scales = bool((torch.frexp(b["scales"]).mantissa == 0.5).all())
    room = (2.0**-10 if exact_scales else 2.0**-9) * bound + torch.finfo(out.dtype).eps / 2 * (1 + 2.0**-6) * np.abs(want) + 2.0**-24 * v_max
    worst = (np.abs(got - want) / room).max()
    assert worst <= 1.0, worst


@pytest.fixture(autouse=True)
def clean_status():
    read_status()
    yield
    assert read_status() == 0


# ------------------------------------------------------------------------------------------------ attention


@pytest.mark.parametrize("half", HALVES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_types_and_head_dims(code, half, dim):
    b = make_batch([(1, 33), (5, 5), (1, 1), (3, 200), (40, 170)], Hq=8, Hkv=2, dim=dim, page=16, block=16, code=code, half=half, seed=dim)
    check(b, run(b))


@pytest.mark.parametrize("page, block", [(8, 8), (8, 1), (16, 4), (24, 8), (32, 32), (48, 16), (64, 2), (128, 128), (256, 64), (1, 1), (4, 2), (20, 4), (36, 1)])
def test_attention_pages_and_scale_blocks(page, block):
    b = make_batch([(1, 300), (2, 129), (1, 64), (9, 65), (1, page), (1, page + 1)], Hq=4, Hkv=2, dim=64, page=page, block=block, code=torch.int8,
                   half=torch.bfloat16, seed=page + block, any_scale=True)
    check(b, run(b))


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (3, 1), (6, 2), (7, 7), (9, 1), (16, 1), (40, 2), (24, 8)])
def test_attention_head_groups(Hq, Hkv):
    b = make_batch([(1, 140), (3, 77), (1, 9)], Hq=Hq, Hkv=Hkv, dim=128, page=16, block=8, code=torch.float8_e4m3fn, half=torch.float16, seed=Hq)
    check(b, run(b))


@pytest.mark.parametrize("kw", [dict(sliding_window=1), dict(sliding_window=50), dict(logits_soft_cap=2.0), dict(softmax_scale=-0.2), dict(softmax_scale=0.0),
                                dict(sliding_window=130, logits_soft_cap=20.0, softmax_scale=0.3)])
@pytest.mark.parametrize("code", CODES)
def test_attention_masks_and_scales(code, kw):
    b = make_batch([(1, 400), (60, 333), (7, 7), (1, 131)], Hq=8, Hkv=2, dim=64, page=16, block=16, code=code, half=torch.bfloat16, seed=4)
    check(b, run(b, **kw), **kw)


@pytest.mark.parametrize("rows", ["q", "kv", "one"])
def test_attention_sinks(rows):
    b = make_batch([(1, 100), (50, 90), (1, 2)], Hq=8, Hkv=2, dim=64, page=16, block=16, code=torch.int8, half=torch.float16, seed=5)
    sinks = torch.randn({"q": (8, 2), "kv": (2, 3), "one": (4,)}[rows], generator=torch.Generator().manual_seed(1)) * 2
    check(b, run(b, sinks=sinks), sinks=sinks)


def test_attention_long_contexts_are_split():
    b = make_batch([(1, 9001), (1, 20000), (2, 5000)], Hq=8, Hkv=1, dim=128, page=32, block=32, code=torch.int8, half=torch.bfloat16, seed=6, any_scale=True)
    check(b, run(b))


@pytest.mark.parametrize("code", CODES)
def test_attention_prompt_chunks(code):
    b = make_batch([(300, 300), (130, 900), (1, 500), (257, 700)], Hq=8, Hkv=2, dim=128, page=16, block=16, code=code, half=torch.bfloat16, seed=7)
    check(b, run(b))


@pytest.mark.parametrize("page, block", [(8, 8), (8, 1), (16, 2), (24, 8), (40, 4), (48, 16), (56, 8), (64, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("dim, window", [(64, None), (128, 70)])
def test_attention_prompt_pages_and_scale_blocks(page, block, dim, window):
    """Tiles that begin and end inside pages and scale blocks, with a window that begins inside one."""
    b = make_batch([(100, 333), (70, 70), (1, 200), (130, 517)], Hq=4, Hkv=2, dim=dim, page=page, block=block, code=torch.int8,
                   half=torch.bfloat16, seed=page + block, any_scale=True)
    kw = {} if window is None else dict(sliding_window=window)
    check(b, run(b, **kw), **kw)


@pytest.mark.parametrize("cap, scale", [(-3.0, None), (0.01, None), (5.0, 4.0), (50.0, -0.3)])
@pytest.mark.parametrize("block", [16, 2])
def test_attention_prompt_soft_caps(block, cap, scale):
    """Caps of either sign, one that every logit reaches and one that few reach."""
    b = make_batch([(90, 300), (1, 100), (200, 260)], Hq=4, Hkv=2, dim=64, page=16, block=block, code=torch.float8_e4m3fn, half=torch.float16, seed=8)
    kw = dict(logits_soft_cap=cap, softmax_scale=scale)
    check(b, run(b, **kw), **kw)


@pytest.mark.parametrize("rows", [1, 90])
def test_scales_need_no_more_than_their_own_alignment(rows):
    b = make_batch([(rows, 300), (1, 77)], Hq=4, Hkv=2, dim=128, page=16, block=4, code=torch.int8, half=torch.bfloat16, seed=9)
    want = run(b)
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}
    flat = torch.zeros(c["scales"].numel() + 1, device="cuda")
    scales = flat[1:].view(c["scales"].shape)
    scales.copy_(c["scales"])
    assert torch.equal(ej.quantized_ragged_page_attention(c["q"], c["codes"], scales, c["ctx"], c["tab"], c["start"], c["n"]), want)
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    for got, plain in zip(ej.quantized_kv_read(c["codes"], scales, slots), ej.quantized_kv_read(c["codes"], c["scales"], slots)):
        assert torch.equal(got, plain)
    x = torch.randn((40, 2, 128), generator=torch.Generator().manual_seed(10)).bfloat16().cuda()
    kv = c["codes"].clone()
    ej.quantized_kv_write(x, x, c["codes"], c["scales"], slots)
    ej.quantized_kv_write(x, x, kv, scales, slots)
    assert torch.equal(kv, c["codes"]) and torch.equal(scales, c["scales"])


@pytest.fixture
def option():
    old = {}

    def set_to(name, value):
        old.setdefault(name, _cabi.get_option(name))
        _cabi.set_option(name, value)

    yield set_to
    for name, value in old.items():
        _cabi.set_option(name, value)


@pytest.mark.parametrize("split", [0, 1, 2])
def test_attention_prompt_parts_are_combined(option, split):
    """2 = items are cut at every quota boundary, whatever the rule says: the parts of a row come from several CTAs."""
    option("prefill_split", split)
    sinks = torch.randn((4, 2), generator=torch.Generator().manual_seed(1))
    for kw in (dict(), dict(sliding_window=700, logits_soft_cap=10.0), dict(sinks=sinks)):
        b = make_batch([(200, 3000), (1, 700), (70, 70), (9, 2500)], Hq=4, Hkv=1, dim=128, page=16, block=8, code=torch.int8, half=torch.float16, seed=13, any_scale=True)
        check(b, run(b, **dict(kw)), **kw)


@pytest.mark.parametrize("rows", [1, 8, 64, 1000])
def test_attention_tiles_or_split_kv_by_the_hint(rows):
    """num_queries_per_block: from how many query tokens on a sequence is served by tensor tiles."""
    b = make_batch([(5, 300), (64, 100), (1, 40), (300, 301), (129, 640)], Hq=6, Hkv=2, dim=64, page=8, block=4, code=torch.float8_e4m3fn, half=torch.bfloat16, seed=14)
    out = run(b, cfg=ej.RaggedPageAttentionConfig(num_kv_pages_per_block=None, num_queries_per_block=rows))
    check(b, out)


@pytest.mark.parametrize("bit, lens", [(1, [(1, 600), (1, 50)]), (2, [(64, 600), (1, 50)])])
def test_a_wait_that_runs_out_is_reported(option, bit, lens):
    """The test hook keeps one stage from being announced: the waits for it give up, the call ends and says so."""
    b = make_batch(lens, Hq=4, Hkv=1, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=15)
    option("wait_ms", 5)
    option("test_withhold", bit)
    run(b)
    assert read_status() & _cabi.ST_TIMEOUT
    option("test_withhold", 0)
    option("wait_ms", 2000)
    check(b, run(b))


def test_attention_empty_sequences_and_rows_behind_the_last():
    b = make_batch([(0, 17), (1, 20), (0, 0), (4, 40)], Hq=4, Hkv=2, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=8, extra_rows=13, rows=9)
    out = run(b)
    check(b, out)
    assert int(torch.count_nonzero(out[5:])) == 0
    b["n"] = 0
    assert int(torch.count_nonzero(run(b))) == 0
    q = b["q"][:0]
    assert run(b | dict(q=q)).shape == q.shape


def test_attention_ignores_what_lies_behind_a_sequence_and_before_its_window():
    """Codes that are NaN and scales that are NaN or infinite in masked places leave the result as it is, bit for bit."""
    lens = [(1, 100), (1, 333), (5, 70), (140, 150)]
    b = make_batch(lens, Hq=4, Hkv=1, dim=64, page=16, block=4, code=torch.float8_e4m3fn, half=torch.bfloat16, seed=9)
    clean = run(b)
    check(b, clean)
    codes, scales = b["codes"].clone().view(torch.uint8), b["scales"].clone()
    used = set()
    for i, (_, kv) in enumerate(lens):
        for j in range(-(-kv // 16)):
            page = int(b["tab"][i, j])
            used.add(page)
            for off in range(16):
                if j * 16 + off >= kv:
                    codes[page, :, :, off] = 0x7F
            for blk in range(4):
                if j * 16 + blk * 4 >= kv:
                    scales[page, :, :, blk] = float("nan") if blk % 2 else float("inf")
    for page in range(codes.shape[0]):
        if page not in used:
            codes[page], scales[page] = 0xFF, float("nan")
    dirty = run(b | dict(codes=codes.view(torch.float8_e4m3fn), scales=scales))
    assert torch.equal(clean, dirty)
    # the keys that every row of a decode batch has left behind
    one = make_batch([(1, 500), (1, 90)], Hq=4, Hkv=1, dim=64, page=16, block=16, code=torch.float8_e4m3fn, half=torch.bfloat16, seed=10)
    clean = run(one, sliding_window=37)
    codes, scales = one["codes"].clone().view(torch.uint8), one["scales"].clone()
    for i, kv in enumerate((500, 90)):
        for key in range(kv - 37):
            codes[int(one["tab"][i, key // 16]), :, :, key % 16] = 0x7F
        for j in range((kv - 37) // 16):
            scales[int(one["tab"][i, j])] = float("nan")
    assert torch.equal(clean, run(one | dict(codes=codes.view(torch.float8_e4m3fn), scales=scales), sliding_window=37))


@pytest.mark.parametrize("code", CODES)
def test_attention_scales_far_apart(code):
    """Blocks of values 2^40 and more apart, queries that f16 does not hold, a block of zeros with the smallest scale."""
    b = make_batch([(1, 260), (3, 100), (40, 100)], Hq=4, Hkv=1, dim=64, page=16, block=16, code=code, half=torch.bfloat16, seed=11)
    far = torch.exp2(torch.randint(-30, 20, b["scales"][:, :, 1].shape, generator=torch.Generator().manual_seed(2)).float())
    b["scales"][:, :, 1] *= far
    b["scales"][:, :, 0] *= 2.0**-40
    b["q"] = (b["q"].double() * 2.0**40).to(torch.bfloat16)
    b["codes"].view(torch.uint8)[int(b["tab"][0, 3])] = 0
    b["scales"][int(b["tab"][0, 3])] = 2.0**-126
    check(b, run(b))


def test_attention_reports_bad_lengths_and_pages():
    b = make_batch([(1, 40), (2, 30)], Hq=4, Hkv=2, dim=64, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=12)
    good = run(b)
    bad = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in b.items()}
    bad["tab"][0, 1] = 1 << 20
    out = run(bad)
    assert read_status() == _cabi.ST_PAGE_ID and torch.equal(out[1:], good[1:])
    bad["tab"][0, 1] = -7
    run(bad)
    assert read_status() == _cabi.ST_PAGE_ID
    bad = b | dict(ctx=torch.tensor([1 << 29, 30], dtype=torch.int32))
    assert torch.equal(run(bad)[1:], good[1:])
    assert read_status() & _cabi.ST_KVLEN
    run(b | dict(ctx=torch.tensor([-1, 30], dtype=torch.int32)))
    assert read_status() & _cabi.ST_KVLEN
    run(b | dict(n=7))
    assert read_status() & _cabi.ST_NUM_SEQS
    run(b | dict(start=torch.tensor([0, 1, 900], dtype=torch.int32)))
    assert read_status() & _cabi.ST_QLEN


# ----------------------------------------------------------------------------------------- write and read


def same_cache(kv, scales, want_codes, want_scales, rows=None):
    got = kv.cpu().to(torch.float32).double().numpy()
    assert np.array_equal(scales.cpu().double().numpy(), want_scales)
    assert np.array_equal(got, want_codes)


@pytest.mark.parametrize("half", HALVES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim, page, block", [(64, 16, 16), (128, 16, 4), (256, 24, 8), (128, 64, 64), (64, 8, 1), (64, 5, 1), (128, 128, 128)])
def test_write(code, half, dim, page, block):
    g = torch.Generator().manual_seed(dim + page + block)
    kv, scales = make_cache(g, 40 if page < 64 else 16, 3, page, dim, code, block)
    slots, base = [], 0
    for c, n in ((0, 1), (3, 2), (page - 1, page + 2), (2 * page + 1, 3 * page), (1, 1)):  # cached, new
        pos = torch.arange(c, c + n)
        pages = torch.randperm(7 if page < 64 else 3, generator=g) if c + n > 2 * page else torch.arange(3)
        n_pages = -(-(c + n) // page)
        pages = torch.arange(n_pages)
        slots.append((base + pages[pos // page]) * page + pos % page)
        base += n_pages
    slots = torch.cat(slots).to(torch.int32)
    slots = torch.cat([slots[:1], torch.tensor([-1, -5], dtype=torch.int32), slots[1:], torch.tensor([-1], dtype=torch.int32)])
    T = slots.numel()
    x = torch.randn((T, 2, 3, dim), generator=g) * torch.exp2(torch.randint(-9, 4, (T, 2, 3, 1), generator=g).float())
    x = x.to(half)
    keys, values = x[:, 0], x[:, 1]  # views: rows are apart
    want = q8_oracle.write(keys, values, kv, scales, slots)
    kv, scales = kv.cuda(), scales.cuda()
    xc = x.cuda()
    got = ej.quantized_kv_write(xc[:, 0], xc[:, 1], kv, scales, slots.cuda())
    assert got[0] is kv and got[1] is scales
    same_cache(kv, scales, *want)
    # the same rows once more: the scales are large enough now, nothing moves
    ej.quantized_kv_write(xc[:, 0].contiguous(), xc[:, 1].contiguous(), kv, scales, slots.cuda())
    same_cache(kv, scales, *want)


@pytest.mark.parametrize("code", CODES)
def test_write_one_token_at_a_time_as_decode_does(code):
    """16 appends to one block, each larger than the last: the scale grows, what is there moves each time."""
    g = torch.Generator().manual_seed(3)
    kv, scales = make_cache(g, 2, 2, 16, 64, code, 16)
    want_kv, want_scales = kv, scales
    kv, scales = kv.cuda(), scales.cuda()
    for i in range(16):
        x = (torch.randn((1, 2, 64), generator=g) * 1.7**i).to(torch.bfloat16)
        slot = torch.tensor([16 + i], dtype=torch.int32)
        c, s = q8_oracle.write(x, -x, want_kv, want_scales, slot)
        want_kv, want_scales = torch.from_numpy(c).to(torch.float32).to(code), torch.from_numpy(s).float()
        ej.quantized_kv_write(x.cuda(), (-x).cuda(), kv, scales, slot.cuda())
        same_cache(kv, scales, c, s)


@pytest.mark.parametrize("code", CODES)
def test_write_zeros_infinities_nan_and_extremes(code):
    g = torch.Generator().manual_seed(4)
    kv, scales = make_cache(g, 4, 1, 16, 64, code, 4)
    x = torch.randn((12, 1, 64), generator=g)
    x[0:4] = 0.0                      # a block of zeros: the smallest scale
    x[4, 0, 3], x[5, 0, 1] = float("inf"), float("-inf")
    x[6, 0, 0] = float("nan")
    x[8:] = 1e-38                     # far below what a code times 2^-126 resolves
    x[9, 0, 5] = 3.0e38
    x = x.to(torch.bfloat16)
    slots = torch.arange(16, 28, dtype=torch.int32)
    want = q8_oracle.write(x, x, kv, scales, slots)
    kv, scales, xc = kv.cuda(), scales.cuda(), x.cuda()
    ej.quantized_kv_write(xc, xc, kv, scales, slots.cuda())
    assert read_status() == _cabi.ST_NONFINITE
    same_cache(kv, scales, *want)
    assert float(scales[1, 0, 0, 0]) == 2.0**-126
    # an infinity is written as the largest code, and read back as a finite value
    k, _ = ej.quantized_kv_read(kv, scales, slots.cuda(), dtype=torch.float16)
    assert torch.isfinite(k).all() and float(k[9, 0, 5]) == 65504.0


def test_write_old_scales_that_are_no_powers_of_two():
    g = torch.Generator().manual_seed(5)
    kv, scales = make_cache(g, 3, 2, 16, 128, torch.int8, 16, any_scale=True)
    x = torch.randn((5, 2, 128), generator=g).to(torch.float16)
    slots = torch.arange(3, 8, dtype=torch.int32)
    want_c, want_s = q8_oracle.write(x, x, kv, scales, slots)
    kv, scales, xc = kv.cuda(), scales.cuda(), x.cuda()
    ej.quantized_kv_write(xc, xc, kv, scales, slots.cuda())
    assert np.array_equal(scales.cpu().double().numpy(), want_s)
    # a quotient by such a scale is rounded once to 24 bits: a code can only differ where that lands on a tie
    got = kv.cpu().double().numpy()
    assert np.abs(got - want_c).max() <= 1 and (got != want_c).mean() < 1e-4


def test_write_and_read_slots_out_of_range():
    g = torch.Generator().manual_seed(6)
    kv, scales = make_cache(g, 2, 1, 16, 64, torch.int8, 16)
    before = kv.clone()
    kv, scales = kv.cuda(), scales.cuda()
    x = torch.ones((3, 1, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([32, -2147483648, 2147483647], dtype=torch.int32, device="cuda")
    ej.quantized_kv_write(x, x, kv, scales, slots)
    assert read_status() == _cabi.ST_PAGE_ID and torch.equal(kv.cpu(), before)
    k, v = ej.quantized_kv_read(kv, scales, slots)
    assert read_status() == _cabi.ST_PAGE_ID and not k.any() and not v.any()
    empty = x[:0]
    ej.quantized_kv_write(empty, empty, kv, scales, slots[:0])
    assert ej.quantized_kv_read(kv, scales, slots[:0])[0].shape == (0, 1, 64)


@pytest.mark.parametrize("half", HALVES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim, page, block", [(64, 16, 16), (128, 24, 2), (256, 7, 1)])
def test_read(code, half, dim, page, block):
    g = torch.Generator().manual_seed(dim)
    kv, scales = make_cache(g, 9, 3, page, dim, code, block, any_scale=True)
    slots = torch.randint(0, 9 * page, (77,), generator=g, dtype=torch.int32)
    slots[5] = -1
    slots[6] = slots[7]
    value = torch.from_numpy(q8_oracle.values_of(kv, scales)).permute(0, 3, 1, 2, 4).reshape(9 * page, 3, 2, dim)[slots.long()]
    value[5] = 0
    # float32 holds the product of a code and a scale to 24 bits, then it is rounded to the type: as one rounding, but
    # for what the first one moves onto a tie
    got = ej.quantized_kv_read(kv.cuda(), scales.cuda(), slots.cuda(), dtype=half)
    for i in range(2):
        err = (got[i].cpu().double() - value[:, :, i]).abs()
        assert bool((err <= value[:, :, i].abs() * (torch.finfo(half).eps / 2 + 2.0**-23)).all())


# -------------------------------------------------------------------------------------------------- page tables


def make_requests(q, ctx, *, page, pps, seed=0, rows=None, free=None, done=()):
    g = torch.Generator().manual_seed(seed)
    S = rows or len(q)
    held = [-(-c // page) for c in ctx]
    order = torch.randperm(sum(held) + 200, generator=g).to(torch.int32)
    tab = torch.full((S, pps), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        tab[i, :h] = order[at: at + h]
        at += h
    left = order[at:]
    stack = torch.full((order.numel(),), -9, dtype=torch.int32)
    stack[: left.numel()] = left
    pad = [0] * (S - len(q))
    fin = torch.zeros(S, dtype=torch.bool)
    fin[list(done)] = True
    return dict(query_lens=torch.tensor(list(q) + pad, dtype=torch.int32), context_lens=torch.tensor(list(ctx) + pad, dtype=torch.int32), block_tables=tab,
                free_pages=stack, num_free=torch.tensor([left.numel() if free is None else free], dtype=torch.int32), num_seqs=len(q), finished=fin)


def check_tables(r, page, T, status=0, finished=True):
    fin = r["finished"] if finished else None
    want = q8_oracle.page_tables(r["query_lens"], r["context_lens"], r["block_tables"], r["free_pages"], r["num_free"], r["num_seqs"], page, T, fin)
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in r.items()}
    lens, start, slots, left = ej.build_page_tables(c["query_lens"], c["context_lens"], c["block_tables"], c["free_pages"], c["num_free"], c["num_seqs"],
                                                    page_size=page, total_tokens=T, finished=c["finished"] if finished else None)
    assert read_status() == status
    assert lens.tolist() == want[0] and start.tolist() == want[1] and slots.tolist() == want[2] and left.tolist() == [want[3]]
    assert np.array_equal(c["block_tables"].cpu().numpy(), want[4]) and np.array_equal(c["free_pages"].cpu().numpy(), want[5])


@pytest.mark.parametrize("page", [1, 7, 16, 128])
def test_tables_mixed_batch(page):
    q, ctx = [1, 1, 40, 1, 0, 17, 1, 5], [0, page - 1, 3, page, 5, 2 * page, 0, 3 * page + 1]
    check_tables(make_requests(q, ctx, page=page, pps=60, seed=page, rows=11), page, sum(q) + 9, finished=False)
    q[3] = q[7] = 0
    check_tables(make_requests(q, ctx, page=page, pps=60, seed=page, rows=11, done=[3, 7]), page, sum(q) + 9)


def test_tables_more_rows_than_one_round_of_the_scan():
    g = np.random.default_rng(1)
    S = 2500
    ctx = g.integers(0, 90, S).tolist()
    done = sorted(g.choice(S, 300, replace=False).tolist())
    q = [0 if i in set(done) else int(n) for i, n in enumerate(g.integers(0, 3, S))]
    r = make_requests(q, ctx, page=8, pps=13, seed=2, rows=2600, done=done)
    r["free_pages"] = torch.cat([r["free_pages"], torch.full((4000,), -3, dtype=torch.int32)])
    check_tables(r, 8, sum(q) + 100)


def test_tables_returned_pages_are_used_at_once():
    """No page is free: what the finished requests return serves the others, the last returned first."""
    r = make_requests([0, 20, 0, 16], [40, 16, 33, 0], page=16, pps=8, seed=3, free=0, done=[0, 2])
    check_tables(r, 16, 36)


def test_tables_that_cannot_be_served():
    # the pool runs out at the third request; the fourth asks for no page
    check_tables(make_requests([16, 16, 40, 3, 16], [0, 0, 0, 2, 0], page=16, pps=8, free=3, seed=4), 16, 100, _cabi.ST_POOL)
    # a table is too short, its neighbours are served
    check_tables(make_requests([16, 40, 16], [0, 20, 0], page=16, pps=3, seed=5), 16, 80, _cabi.ST_KVLEN)
    # more tokens than the batch holds
    check_tables(make_requests([16, 40, 16, 0], [0, 20, 0, 0], page=16, pps=8, seed=6), 16, 50, _cabi.ST_QLEN)
    # negative counts, and a stack that is said to be larger than it is
    r = make_requests([4, 4], [0, 0], page=16, pps=8, seed=7)
    r["query_lens"][0] = -3
    check_tables(r, 16, 8, _cabi.ST_QLEN)
    r = make_requests([4, 4], [0, 0], page=16, pps=8, seed=7)
    r["num_free"][0] = 1 << 30
    r["free_pages"] = r["free_pages"].clamp(min=0)
    check_tables(r, 16, 8, _cabi.ST_POOL)
    # no room for the returned pages: the ones that fit are kept
    r = make_requests([0, 1], [50, 0], page=16, pps=8, seed=8, done=[0])
    r["free_pages"] = r["free_pages"][:202].contiguous()
    check_tables(r, 16, 8, _cabi.ST_POOL)
    # nobody is there, and a step without tokens
    r = make_requests([1], [0], page=16, pps=2, seed=9, rows=3)
    r["num_seqs"] = 0
    check_tables(r, 16, 5)
    check_tables(make_requests([0, 0], [5, 40], page=16, pps=8, seed=9, done=[1]), 16, 0)


# ------------------------------------------------------------------------------------------ together, as they are used


class Loop:
    """A serving loop's state: requests come, decode and go; the plain twin keeps every token's K and V in float64 rows of the
    cache, through the oracle's write."""

    def __init__(self, code, half, *, rows=6, pages=64, page=16, block=16, Hq=4, Hkv=2, dim=64, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.code, self.half, self.page, self.Hq, self.Hkv, self.dim, self.rows = code, half, page, Hq, Hkv, dim, rows
        self.kv, self.scales = ej.modules.operations.allocate_quantized_kv(pages, Hkv, page, dim, dtype=code, scale_block=block)
        self.tables = torch.full((rows, 32), -1, dtype=torch.int32, device="cuda")  # 512 tokens: the longest request gets 420
        self.free = torch.randperm(pages, generator=self.g).to(torch.int32).cuda()
        self.num_free = torch.tensor([pages], dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.n = torch.tensor([rows], dtype=torch.int32, device="cuda")
        self.cpu = dict(kv=self.kv.cpu(), scales=self.scales.cpu(), tables=self.tables.cpu(), free=self.free.cpu(), num_free=pages, lens=self.lens.cpu())

    def inputs(self, q, tokens):
        r = lambda h: torch.randn((tokens, h, self.dim), generator=self.g).to(self.half)  # noqa: E731
        return dict(q=torch.tensor(q, dtype=torch.int32), x=r(self.Hq), k=r(self.Hkv) * float(2.0 ** int(torch.randint(-4, 5, (1,), generator=self.g))), v=r(self.Hkv))

    def step(self, i, done=None):
        lens, start, slots, num_free = ej.build_page_tables(i["q"], self.lens, self.tables, self.free, self.num_free, self.n, page_size=self.page,
                                                            total_tokens=i["x"].shape[0], finished=done)
        ej.quantized_kv_write(i["k"], i["v"], self.kv, self.scales, slots)
        out = ej.quantized_ragged_page_attention(i["x"], self.kv, self.scales, lens, self.tables, start, self.n)
        self.lens.copy_(lens)
        self.num_free.copy_(num_free)
        return out, start

    def plain(self, i, done=None):
        c = self.cpu
        lens, start, slots, c["num_free"], tables, free = q8_oracle.page_tables(i["q"], c["lens"], c["tables"], c["free"], c["num_free"], self.rows, self.page, i["x"].shape[0], done)
        c["lens"], c["tables"], c["free"] = torch.tensor(lens, dtype=torch.int32), torch.from_numpy(tables), torch.from_numpy(free)
        codes, scales = q8_oracle.write(i["k"], i["v"], c["kv"], c["scales"], torch.tensor(slots, dtype=torch.int32))
        c["kv"], c["scales"] = torch.from_numpy(codes).float().to(self.code), torch.from_numpy(scales).float()
        return dict(q=i["x"], codes=c["kv"], scales=c["scales"], ctx=c["lens"], tab=c["tables"], start=torch.tensor(start, dtype=torch.int32), n=self.rows)


STEPS = [([40, 1, 0, 130, 7, 3], ()), ([1, 1, 20, 1, 1, 1], ()), ([1, 1, 1, 1, 0, 1], (4,)), ([1, 17, 1, 0, 9, 1], (3,)), ([1, 1, 1, 1, 1, 1], ())]


@pytest.mark.parametrize("code, half", [(torch.int8, torch.bfloat16), (torch.float8_e4m3fn, torch.float16)])
def test_a_serving_loop_of_the_operators(code, half):
    loop = Loop(code, half)
    for q, gone in STEPS:
        i = loop.inputs(q, sum(q) + 5)
        done = torch.zeros(loop.rows, dtype=torch.bool)
        done[list(gone)] = True
        c = {k: v.cuda() for k, v in i.items()}
        out, _ = loop.step(c, done.cuda())
        b = loop.plain(i, done)
        check(b, out)
        assert torch.equal(loop.lens.cpu(), loop.cpu["lens"]) and torch.equal(loop.tables.cpu(), loop.cpu["tables"])
        assert np.array_equal(loop.kv.cpu().float().numpy(), loop.cpu["kv"].float().numpy())


@pytest.mark.parametrize("tokens", [6, 200])
def test_a_step_is_captured_and_replayed(tokens):
    """One graph per batch shape, replayed on new inputs; two graphs of the same operators, in turn, and eager calls between."""
    loop = Loop(torch.int8, torch.bfloat16, pages=200, seed=3)
    first = loop.inputs([20, 1, 5, 2, 70, 3], 101)
    eager, _ = loop.step({k: v.cuda() for k, v in first.items()})
    check(loop.plain(first), eager)
    q = [1] * 6 if tokens == 6 else [100, 1, 1, 64, 30, 1]
    static = {k: v.cuda() for k, v in loop.inputs(q, tokens).items()}
    keep = [t.clone() for t in (loop.kv, loop.scales, loop.tables, loop.free, loop.num_free, loop.lens)]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = loop.step(static)
        graphs.append((graph, out))
    for t, k in zip((loop.kv, loop.scales, loop.tables, loop.free, loop.num_free, loop.lens), keep):
        assert torch.equal(t.view(torch.uint8) if t.dtype == torch.int8 else t, k.view(torch.uint8) if k.dtype == torch.int8 else k)  # capturing runs nothing
    for turn in range(4):
        i = loop.inputs(q, tokens)
        for k, v in i.items():
            static[k].copy_(v)
        graph, out = graphs[turn % 2]
        graph.replay()
        b = loop.plain(i)
        check(b, out)
        again = ej.quantized_ragged_page_attention(static["x"], loop.kv, loop.scales, loop.lens, loop.tables, b["start"].cuda(), loop.n)
        assert torch.equal(again, out)


def test_two_streams_at_once():
    """Each stream has its own scratch: calls that overlap on the device do not disturb one another."""
    batches = [make_batch([(1, 9000 + 100 * s), (1, 400), (40, 700)], Hq=8, Hkv=1, dim=128, page=16, block=16, code=CODES[s], half=torch.bfloat16, seed=20 + s) for s in range(2)]
    gpu = [{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()} for b in batches]
    alone = [run(b) for b in gpu]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for s, (stream, b) in enumerate(zip(streams, gpu)):
            with torch.cuda.stream(stream):
                outs[s].append(run(b))
    torch.cuda.synchronize()
    for s in range(2):
        check(batches[s], alone[s])
        assert all(torch.equal(o, alone[s]) for o in outs[s])


def test_results_do_not_depend_on_the_run():
    """No atomics on values: the parts of a row are combined in a fixed order."""
    b = make_batch([(1, 20000), (1, 777), (3, 6000), (200, 900)], Hq=8, Hkv=2, dim=64, page=16, block=16, code=torch.int8, half=torch.float16, seed=30)
    gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}
    outs = [run(gpu) for _ in range(6)]
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_workspace_counters_are_zero_after_every_call(option):
    from ejkernel_b200.kernels._cuda.quantized_kv import _interface

    b = make_batch([(1, 20000), (1, 50), (2, 3000)], Hq=8, Hkv=1, dim=128, page=16, block=16, code=torch.int8, half=torch.bfloat16, seed=31)
    good = run(b)
    counters = lambda: [int(torch.count_nonzero(w[: _cabi.Q8_TICKET_BYTES])) for w in _interface._scratch.values()]  # noqa: E731
    assert counters() and not any(counters())
    option("wait_ms", 5)
    option("test_withhold", 1)
    run(b)
    assert read_status() & _cabi.ST_TIMEOUT and not any(counters())
    option("test_withhold", 0)
    option("wait_ms", 2000)
    assert torch.equal(run(b), good)


@pytest.mark.parametrize("name, value", [("path", 1), ("overlap", 0), ("min_chunk", 64), ("min_chunk", 4096), ("prefill_rows", 0), ("prefill_rows", 1)])
def test_options(option, name, value):
    b = make_batch([(1, 2000), (5, 300), (70, 300), (1, 1)], Hq=8, Hkv=2, dim=128, page=16, block=4, code=torch.float8_e4m3fn, half=torch.bfloat16, seed=32)
    option(name, value)
    check(b, run(b))


def test_a_cache_beyond_32_bit_offsets():
    """Pages whose bytes lie past 2^32, codes and scales of several gigabytes."""
    pages, heads, page, dim = 36000, 8, 32, 256
    kv = torch.zeros((pages, heads, 2, page, dim), dtype=torch.int8, device="cuda")
    scales = torch.ones((pages, heads, 2, page), dtype=torch.float32, device="cuda")
    assert kv.numel() > 2**32
    g = torch.Generator().manual_seed(40)
    lens = [(1, 100), (3, 40), (64, 64)]
    b = make_batch(lens, Hq=16, Hkv=heads, dim=dim, page=page, block=1, code=torch.int8, half=torch.bfloat16, seed=41, spare=0)
    far = pages - 1 - torch.arange(b["codes"].shape[0])
    kv[far.cuda()], scales[far.cuda()] = b["codes"].cuda(), b["scales"].cuda()
    tab = torch.where(b["tab"] >= 0, far.to(torch.int32)[b["tab"].clamp(min=0).long()], -1)
    out = ej.quantized_ragged_page_attention(b["q"].cuda(), kv, scales, b["ctx"].cuda(), tab.cuda(), b["start"].cuda(), b["n"])
    check(b, out)
    x = torch.randn((5, heads, dim), generator=g).to(torch.float16)
    slots = torch.arange(far[0] * page + 3, far[0] * page + 8, dtype=torch.int32)
    ej.quantized_kv_write(x.cuda(), x.cuda(), kv, scales, slots.cuda())
    k, v = ej.quantized_kv_read(kv, scales, slots.cuda(), dtype=torch.float16)
    step = x.float().abs().amax(-1, keepdim=True) / 63  # a scale is above amax / 127 / 2 ... amax / 127
    assert bool(((k.cpu().float() - x.float()).abs() <= step * 0.51).all()) and torch.equal(k, v)


def test_misaligned_views_are_refused():
    kv, scales = ej.modules.operations.allocate_quantized_kv(2, 1, 16, 64, dtype=torch.int8)
    flat = torch.zeros(2 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    x = flat[4: 4 + 128].view(2, 1, 64)
    slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    with pytest.raises(_cabi.RpaLibraryError, match="aligned"):
        ej.quantized_kv_write(x, x, kv, scales, slots)
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(_cabi.RpaLibraryError, match="aligned"):
        ej.quantized_ragged_page_attention(x, kv, scales, i[:1], i[:1].view(1, 1), i[:2], 1)
    with pytest.raises(ValueError, match="is on"):
        ej.quantized_kv_write(x.contiguous(), x, kv.cpu(), scales, slots)
