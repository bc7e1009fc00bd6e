"""What is measured of the operators around a paged KV cache held in 8 bits.

Four operators that a serving step runs one after the other:

* ``tables``: block tables and slot maps from request lengths (``build_page_tables``);
* ``write``: the step's new key / value rows into the 8-bit cache, one scale for each block of tokens and head
  (``quantized_kv_write``), and the cache's values back (``quantized_kv_read`` over all of it, since the cache itself holds codes);
* ``read``: rows of the cache back in 16 bits (``quantized_kv_read``);
* ``attention``: mixed decode / chunked-prefill attention over that cache (``quantized_ragged_page_attention``).

The cache is ``kv_pages [pages, kv heads, 2 (K, V), page_size, head_dim]`` of codes (e4m3 or int8) and ``kv_scales [pages,
kv heads, 2, page_size / block]`` in float32: a value is its code times the scale of its block of ``block`` tokens.
"""

from __future__ import annotations

import math
import random

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
HALF = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one decode step's bookkeeping for a handful of requests: latency
        dict(name="tables, 4 decode requests", op="tables", seqs=4, rows=4, q_max=1, ctx_max=700, page=16, pps=64, pad=0, done=0, lengths=1),
        # a full batch: finished requests give pages back, new prompts come in beside decode rows, the token batch is padded
        dict(name="tables, 1000 requests", op="tables", seqs=1000, rows=1024, q_max=120, ctx_max=20000, page=16, pps=2048, pad=777, done=40, lengths=2),
        # one request's next token: the smallest append
        dict(name="write, one token", op="write", code="int8", half="bf16", seqs=1, q_max=1, heads=2, dim=64, page=16, block=16, lengths=3),
        # a decode batch: every token goes into a page that is partly filled
        dict(name="write, 256 decode tokens", op="write", code="e4m3", half="bf16", seqs=256, q_max=1, heads=8, dim=128, page=16, block=16, lengths=4),
        # chunks of prompts, one scale for 32 tokens of a 64-token page
        dict(name="write, prompts of 8 requests", op="write", code="int8", half="f16", seqs=8, q_max=2048, heads=8, dim=128, page=64, block=32, lengths=5),
        # a short prefix read back, scales for every token
        dict(name="read, 333 rows", op="read", code="int8", half="f16", rows=333, pages=64, heads=3, dim=64, page=8, block=1, lengths=6),
        # a long shared prefix read back for another worker
        dict(name="read, 65536 rows", op="read", code="e4m3", half="bf16", rows=65536, pages=4608, heads=8, dim=128, page=16, block=16, lengths=7),
        # one request, a short context: latency
        dict(name="attention, one short request", op="attention", code="int8", half="bf16", seqs=1, q_max=1, kv_min=17, kv_max=17, heads_q=4, heads=1, dim=64, page=16, block=16, window=0, cap=0.0, sinks=0, any_scale=False, lengths=8),
        # the decode batch that serving spends its time on
        dict(name="attention, 128 decode requests", op="attention", code="e4m3", half="bf16", seqs=128, q_max=1, kv_min=128, kv_max=8192, heads_q=32, heads=8, dim=128, page=16, block=16, window=0, cap=0.0, sinks=0, any_scale=False, lengths=9),
        # few requests of long context on one head shard: the long axis has to be split
        dict(name="attention, 4 long requests", op="attention", code="int8", half="f16", seqs=4, q_max=1, kv_min=60001, kv_max=131072, heads_q=8, heads=1, dim=128, page=32, block=32, window=0, cap=0.0, sinks=0, any_scale=True, lengths=10),
        # chunks of prompts and decode rows in one batch, with window, soft cap and sinks, odd page size
        dict(name="attention, mixed 24 requests", op="attention", code="int8", half="bf16", seqs=24, q_max=300, kv_min=1, kv_max=3001, heads_q=12, heads=4, dim=64, page=24, block=8, window=1000, cap=30.0, sinks=2, any_scale=False, lengths=11),
        # long prompts in chunks: the products bound it
        dict(name="attention, 4 prompt chunks", op="attention", code="e4m3", half="bf16", seqs=4, q_max=2048, kv_min=2048, kv_max=8192, heads_q=32, heads=8, dim=128, page=16, block=16, window=0, cap=0.0, sinks=0, any_scale=False, lengths=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "write", "read", "attention", "attention"])
    lengths = rng.randrange(100, 1 << 20)
    if op == "tables":
        seqs = _log(rng, 1, 1000)
        page = rng.choice([8, 16, 24, 32, 64, 128])
        q_max = rng.choice([1, 1, _log(rng, 2, 120)])
        return dict(op=op, seqs=seqs, rows=seqs + rng.choice([0, 0, rng.randrange(24)]), q_max=q_max, ctx_max=_log(rng, 1, 20000), page=page,
                    pps=20200 // page + 2, pad=rng.choice([0, _log(rng, 1, 777)]), done=rng.randrange(0, 1 + seqs // 20), lengths=lengths)
    code, half = rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "f16"])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 128])
    block = rng.choice([b for b in (1, 2, 4, 8, 16, 32, 64, 128) if page % b == 0])
    dim = rng.choice([64, 128, 128, 256])
    if op == "write":
        if rng.random() < 0.5:
            return dict(op=op, code=code, half=half, seqs=_log(rng, 1, 256), q_max=1, heads=rng.randrange(1, 9), dim=dim, page=page, block=block, lengths=lengths)
        return dict(op=op, code=code, half=half, seqs=_log(rng, 1, 8), q_max=_log(rng, 2, 1024), heads=rng.randrange(1, 9), dim=dim, page=page, block=block, lengths=lengths)
    if op == "read":
        rows = _log(rng, 1, 30000)
        return dict(op=op, code=code, half=half, rows=rows, pages=rows // page + 1 + rng.randrange(64), heads=rng.randrange(1, 9), dim=dim, page=page, block=block, lengths=lengths)
    heads = rng.choice([1, 2, 3, 4, 8])
    case = dict(op=op, code=code, half=half, seqs=1, q_max=1, kv_min=1, kv_max=1, heads_q=heads * rng.choice([1, 2, 3, 4, 8]), heads=heads, dim=dim,
                page=page, block=block, window=rng.choice([0, 0, _log(rng, 1, 4000)]), cap=rng.choice([0.0, 0.0, 30.0]), sinks=rng.choice([0, 0, 1, 4]),
                any_scale=rng.random() < 0.3, lengths=lengths)
    kind = rng.choice(["decode", "long", "mixed", "prompt"])
    if kind == "decode":
        case |= dict(seqs=_log(rng, 1, 128), kv_max=_log(rng, 1, 4096))
    elif kind == "long":
        case |= dict(seqs=rng.randrange(1, 4), kv_min=10000, kv_max=_log(rng, 20000, 100000), heads=1, heads_q=rng.choice([1, 4, 8, 16]))
    elif kind == "mixed":
        case |= dict(seqs=_log(rng, 2, 24), q_max=_log(rng, 2, 200), kv_max=_log(rng, 200, 2500))
    else:
        case |= dict(seqs=rng.randrange(1, 4), q_max=_log(rng, 64, 1024), kv_min=64, kv_max=_log(rng, 1024, 4096))
    return case


# ---------------------------------------------------------------- lengths: they follow from the case alone


def _table_lengths(case):
    r = random.Random(case["lengths"])
    n = case["seqs"]
    ctx = [r.randrange(0, case["ctx_max"] + 1) for _ in range(n)]
    # most requests decode one token, about one in eight brings a chunk of a prompt
    q = [r.randrange(2, case["q_max"] + 1) if case["q_max"] > 1 and r.random() < 0.125 else 1 for _ in range(n)]
    done = set(r.sample(range(n), case["done"]))
    q = [0 if i in done else v for i, v in enumerate(q)]
    return ctx, q, [i in done for i in range(n)]


def _write_lengths(case):
    r = random.Random(case["lengths"])
    if case["q_max"] == 1:
        q = [1] * case["seqs"]
    else:
        q = [r.randrange(case["q_max"] // 2, case["q_max"] + 1) for _ in range(case["seqs"])]
    ctx = [r.randrange(0, 3 * case["page"]) for _ in q]
    return ctx, q


def _attention_lengths(case):
    """(query rows, keys) of each request; in a mixed batch two of three only decode."""
    r = random.Random(case["lengths"])
    out = []
    for _ in range(case["seqs"]):
        if case["q_max"] == 1:
            q = 1
        elif case["q_max"] < 512 and r.random() < 0.67:
            q = 1
        else:
            q = r.randrange(max(1, case["q_max"] // 2), case["q_max"] + 1)
        kv = max(q, r.randrange(case["kv_min"], case["kv_max"] + 1))
        out.append((q, kv))
    return out


def _cdiv(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- what a user's program has in hand


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(gen, pages, case):
    """Codes of normally distributed values under scales that differ from block to block, as appends leave them."""
    code, page = case["code"], case["page"]
    e = torch.randint(-2, 2, (pages, case["heads"], 2, page // case["block"], 1), generator=gen, device="cuda")
    scales = torch.exp2(e.float() - (6.0 if code == "e4m3" else 4.0))
    if case.get("any_scale"):  # calibrated elsewhere: not powers of two
        scales = scales * (1.0 + torch.rand(scales.shape, generator=gen, device="cuda"))
    x = torch.randn((pages, case["heads"], 2, page // case["block"], case["block"] * case["dim"]), generator=gen, device="cuda")
    x.div_(scales).clamp_(-QMAX[code], QMAX[code])
    if code == "int8":
        x.round_()
    codes = x.to(CODE[code]).view(pages, case["heads"], 2, page, case["dim"])
    return codes, scales.squeeze(-1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    op = case["op"]
    if op == "tables":
        ctx, q, done = _table_lengths(case)
        rows, page = case["rows"], case["page"]
        held = [_cdiv(c, page) for c in ctx]
        need = sum(_cdiv(c + n, page) - h for c, n, h in zip(ctx, q, held))
        total = sum(held) + need + 64
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        tables = torch.full((rows, case["pps"]), -1, dtype=torch.int32, device="cuda")
        row = torch.repeat_interleave(torch.arange(len(ctx), device="cuda"), torch.tensor(held, device="cuda"))
        start = torch.tensor([0] + held, device="cuda").cumsum(0)
        tables[row, torch.arange(sum(held), device="cuda") - start[row]] = order[: sum(held)]
        free = torch.full((total,), -1, dtype=torch.int32, device="cuda")
        free[: total - sum(held)] = order[sum(held):]
        pad = [0] * (rows - len(ctx))
        state |= dict(query_lens=_int(q + pad), context_lens=_int(ctx + pad), tables=tables, free=free, num_free=_int([total - sum(held)]),
                      num_seqs=_int([len(ctx)]), finished=torch.tensor(done + [False] * len(pad), device="cuda"), tokens=sum(q) + case["pad"])
    elif op == "write":
        ctx, q = _write_lengths(case)
        page = case["page"]
        pages = sum(_cdiv(c + n, page) for c, n in zip(ctx, q))
        order = torch.randperm(pages, generator=gen, device="cuda")
        slots, at = [], 0
        for c, n in zip(ctx, q):
            pos = torch.arange(c, c + n, device="cuda")
            slots.append(order[at + pos // page] * page + pos % page)
            at += _cdiv(c + n, page)
        kv, scales = _cache(gen, pages, case)
        half = HALF[case["half"]]
        # a step's rows: some heads and some requests are larger than what the block held, so that some scales have to grow
        shape = (sum(q), case["heads"], case["dim"])
        size = torch.exp2(torch.randint(-3, 3, (shape[0], shape[1], 1), generator=gen, device="cuda").float())
        state |= dict(kv=kv, scales=scales, slots=torch.cat(slots).to(torch.int32),
                      keys=(torch.randn(shape, generator=gen, device="cuda") * size).to(half), values=(torch.randn(shape, generator=gen, device="cuda") * size).to(half),
                      all_slots=torch.arange(pages * page, dtype=torch.int32, device="cuda"), half=half)
    elif op == "read":
        kv, scales = _cache(gen, case["pages"], case)
        order = torch.randperm(case["pages"], generator=gen, device="cuda")
        pos = torch.arange(case["rows"], device="cuda")
        state |= dict(kv=kv, scales=scales, half=HALF[case["half"]], slots=(order[pos // case["page"]] * case["page"] + pos % case["page"]).to(torch.int32))
    else:
        lens = _attention_lengths(case)
        page = case["page"]
        held = [_cdiv(k, page) for _, k in lens]
        pages, pps = sum(held), max(held)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        tables = torch.zeros((len(lens), pps), dtype=torch.int32, device="cuda")
        at = 0
        for i, h in enumerate(held):
            tables[i, :h] = order[at: at + h]
            at += h
        kv, scales = _cache(gen, pages, case)
        q = [a for a, _ in lens]
        start = [0]
        for a in q:
            start.append(start[-1] + a)
        state |= dict(kv=kv, scales=scales, tables=tables, context_lens=_int([k for _, k in lens]), query_start_loc=_int(start), num_seqs=_int([len(lens)]),
                      queries=torch.randn((start[-1], case["heads_q"], case["dim"]), generator=gen, device="cuda").to(HALF[case["half"]]),
                      sinks=torch.randn((case["heads_q"], case["sinks"]), generator=gen, device="cuda") if case["sinks"] else None,
                      q_max=max(q), kv_max=max(k for _, k in lens), window=case["window"] or None, cap=case["cap"] or None)
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        import ejkernel_b200 as ej

        if op == "tables":
            lens, start, slots, num_free = ej.build_page_tables(
                state["query_lens"], state["context_lens"], state["tables"], state["free"], state["num_free"], state["num_seqs"],
                page_size=state["case"]["page"], total_tokens=state["tokens"], finished=state["finished"])
            return {"context_lens": lens, "query_start_loc": start, "slots": slots, "num_free": num_free, "tables": state["tables"], "free": state["free"]}
        if op == "write":
            ej.quantized_kv_write(state["keys"], state["values"], state["kv"], state["scales"], state["slots"])
            keys, values = ej.quantized_kv_read(state["kv"], state["scales"], state["all_slots"], dtype=state["half"])
            return {"keys": keys, "values": values, "scales": state["scales"]}
        if op == "read":
            return ej.quantized_kv_read(state["kv"], state["scales"], state["slots"], dtype=state["half"])
        return ej.quantized_ragged_page_attention(
            state["queries"], state["kv"], state["scales"], state["context_lens"], state["tables"], state["query_start_loc"], state["num_seqs"],
            sliding_window=state["window"], logits_soft_cap=state["cap"], softmax_aux=state["sinks"])
    if op == "tables":
        return _tables(state)
    if op == "write":
        _write(state)
        keys, values = _read(state["kv"], state["scales"], state["all_slots"], state["half"])
        return {"keys": keys, "values": values, "scales": state["scales"]}
    if op == "read":
        return _read(state["kv"], state["scales"], state["slots"], state["half"])
    return _attention(state)


# ---------------------------------------------------------------- the plain forms


def _tables(s):
    page, tables, free = s["case"]["page"], s["tables"], s["free"]
    rows, pps = tables.shape
    dev = tables.device
    live = torch.arange(rows, device=dev) < s["num_seqs"]
    gone = s["finished"] & live
    ctx = torch.where(live, s["context_lens"], 0).long()
    q = torch.where(live & ~gone, s["query_lens"], 0).long()
    held = (ctx + page - 1) // page
    col = torch.arange(pps, device=dev)
    # pages of finished requests go on top of the stack, in order
    back = (col[None, :] < held[:, None]) & gone[:, None]
    top = s["num_free"].long()
    at = top + back.reshape(-1).cumsum(0) - 1
    n = free.shape[0]
    grown = torch.cat([free, free.new_zeros(1)])
    grown[torch.where(back.reshape(-1), at, n)] = torch.where(back.reshape(-1), tables.reshape(-1), 0)
    free.copy_(grown[:n])
    top = top + back.sum()
    # every other request takes what its new tokens need, in order, from the top
    need = torch.where(gone, 0, (ctx + q + page - 1) // page - held)
    first = need.cumsum(0) - need
    fits = (first + need <= top) & ~gone
    take = (col[None, :] >= held[:, None]) & (col[None, :] < (held + need)[:, None]) & fits[:, None]
    src = (top - 1 - first[:, None] - (col[None, :] - held[:, None])).clamp(0, n - 1)
    tables.copy_(torch.where(take, free[src], tables))
    start = torch.cat([q.new_zeros(1), q.cumsum(0)])
    t = torch.arange(s["tokens"], device=dev)
    row = (torch.searchsorted(start, t, right=True) - 1).clamp(0, rows - 1)
    pos = ctx[row] + t - start[row]
    slot = tables[row, (pos // page).clamp(0, pps - 1)].long() * page + pos % page
    slot = torch.where((t < start[-1]) & fits[row], slot, -1)
    lens = torch.where(gone, 0, torch.where(fits, ctx + q, ctx))
    return {"context_lens": lens.to(torch.int32), "query_start_loc": start.to(torch.int32), "slots": slot.to(torch.int32),
            "num_free": (top - torch.where(fits, need, 0).sum()).to(torch.int32), "tables": tables, "free": free}


def _power(amax, code):
    """The smallest power of two, not below 2^-126, under which `amax` does not pass the largest code."""
    mant, e = torch.frexp(amax)
    j = e - 9 + (mant > 0.875) if code == "e4m3" else e - 7 + (mant > 0.9921875)
    j = torch.where(amax > 0, j, -126).clamp(min=-126)
    return ((j + 127) << 23).to(torch.int32).view(torch.float32)


def _to_code(x, code):
    x = x.clamp(-QMAX[code], QMAX[code])
    return (x.round() if code == "int8" else x).to(CODE[code])


def _write(s):
    case, kv, scales = s["case"], s["kv"], s["scales"]
    code, block = case["code"], case["block"]
    pages, heads, _, page, dim = kv.shape
    per = page // block
    slots = s["slots"].long()
    # codes and scales by (block, head, k or v): views of the cache
    blk = slots // block                                       # block of each row, over all pages
    x = torch.stack([s["keys"], s["values"]], 2).float()       # [rows, heads, 2, dim]
    touched, which = torch.unique(blk, return_inverse=True)
    n = touched.shape[0]
    amax = torch.zeros((n, heads, 2), device=x.device).index_reduce_(0, which, x.abs().amax(-1), "amax")
    first = torch.full((n,), block, device=x.device).index_reduce_(0, which, slots % block, "amin")
    new = _power(amax, code)
    pg, sub = touched // per, touched % per
    old = scales[pg, :, :, sub]                                # [blocks, heads, 2]
    keep = (first > 0)[:, None, None]
    scale = torch.where(keep, torch.maximum(old, new), new)
    # rows that the blocks held before, under the scale they have now
    byte = kv.view(torch.uint8).view(pages, heads, 2, per, block, dim)
    before = byte[pg, :, :, sub].view(CODE[code])              # [blocks, heads, 2, block, dim]
    ratio = torch.where(keep, old / scale, 1.0)[..., None, None]
    moved = _to_code(before.float() * ratio, code)
    offset = torch.arange(block, device=x.device)
    live = (offset < first[:, None])[:, None, None, :, None]
    byte[pg, :, :, sub] = torch.where(live, moved.view(torch.uint8), before.view(torch.uint8))
    scales[pg, :, :, sub] = scale
    rows = _to_code(x / scale[which][..., None], code).view(torch.uint8)
    byte[blk // per, :, :, blk % per, slots % block] = rows
    return kv, scales


def _read(kv, scales, slots, half):
    pages, heads, _, page, dim = kv.shape
    block = page // scales.shape[3]
    slots = slots.long()
    codes = kv.view(torch.uint8)[slots // page, :, :, slots % page].view(kv.dtype).float()          # [rows, heads, 2, dim]
    x = codes * scales[slots // page, :, :, slots % page // block][..., None]
    big = torch.finfo(half).max
    x = x.clamp(-big, big).to(half)
    return x[:, :, 0].contiguous(), x[:, :, 1].contiguous()


def _attention(s):
    case, kv, scales, q = s["case"], s["kv"], s["scales"], s["queries"].float()
    page, block, dim, heads = case["page"], case["block"], case["dim"], case["heads"]
    group = case["heads_q"] // heads
    dev = q.device
    lens, start = s["context_lens"].long(), s["query_start_loc"].long()
    q_len = start[1:] - start[:-1]
    key = torch.arange(s["kv_max"], device=dev)
    row = torch.arange(s["q_max"], device=dev)
    there = row[None, :] < q_len[:, None]                                       # [S, Q]
    at = (start[:-1, None] + row[None, :]).clamp(max=q.shape[0] - 1)
    qs = q[at].view(*at.shape, heads, group, dim)                               # [S, Q, H, G, D]
    pg = s["tables"].long()[:, key // page]                                     # [S, K]
    off = (key % page)[None, :].expand_as(pg)

    def values(which):
        codes = kv.view(torch.uint8)[pg, :, which, off].view(kv.dtype).float()  # [S, K, H, D]
        return codes * scales[pg, :, which, off // block][..., None]

    x = torch.einsum("sqhgd,skhd->shgqk", qs, values(0)) * dim**-0.5
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    pos = (lens - q_len)[:, None] + row[None, :]                                # [S, Q]
    see = (key <= pos[..., None]) & (key < lens[:, None, None])
    if s["window"]:
        see &= key > pos[..., None] - s["window"]
    x = x.masked_fill(~see[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, heads, group, 1, -1)
        top = torch.maximum(top, sink.amax(-1, keepdim=True))
    top = torch.where(top == float("-inf"), 0.0, top)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top).sum(-1, keepdim=True)
    out = torch.einsum("shgqk,skhd->sqhgd", x / total.clamp(min=1e-30), values(1))
    result = torch.zeros_like(s["queries"])
    result[at[there]] = out.reshape(*at.shape, heads * group, dim)[there].to(result.dtype)
    return result


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "tables":
        ctx, q, done = _table_lengths(case)
        page = case["page"]
        new = sum(_cdiv(c + n, page) - _cdiv(c, page) for c, n, d in zip(ctx, q, done) if not d)
        back = sum(_cdiv(c, page) for c, d in zip(ctx, done) if d)
        # lengths and flags in, lengths, starts and slots out, each new or returned page read and written, the page that a request goes on in
        return {"bytes": case["rows"] * (4 + 4 + 1 + 4 + 4) + 4 * (sum(q) + case["pad"]) + 8 * (new + back) + 4 * case["seqs"], "flops": 0}
    if op == "write":
        ctx, q = _write_lengths(case)
        page, block = case["page"], case["block"]
        pages = sum(_cdiv(c + n, page) for c, n in zip(ctx, q))
        row = 2 * case["heads"] * case["dim"]
        blocks = sum(_cdiv(c + n, block) - c // block for c, n in zip(ctx, q))
        there = pages * page
        # the rows in 16 bits in, in 8 bits out, their scales; then all of the cache in and its values out
        return {"bytes": sum(q) * (row * 3 + 4) + blocks * case["heads"] * 8 + there * (row * 3 + 4) + pages * (page // block) * case["heads"] * 8, "flops": 0}
    if op == "read":
        row = 2 * case["heads"] * case["dim"]
        return {"bytes": case["rows"] * (row * 3 + 4) + _cdiv(case["rows"], case["block"]) * case["heads"] * 8, "flops": 0}
    keys = pairs = rows = 0
    w = case["window"] or 1 << 40
    for q, kv in _attention_lengths(case):
        base = kv - q
        keys += kv - max(0, base - w + 1)
        pairs += sum(min(base + r + 1, w) for r in range(q))
        rows += q
    kv_bytes = keys * case["heads"] * 2 * (case["dim"] + 4 / case["block"])
    return {"bytes": int(kv_bytes + rows * case["heads_q"] * case["dim"] * 4), "flops": 4 * pairs * case["heads_q"] * case["dim"]}


# ---------------------------------------------------------------- the definitions in 64 bits


def _value64(codes, scales, page, block):
    """Values of whole pages [pages, heads, 2, page, dim] in 64 bits."""
    return codes.to(torch.float32).double() * scales.double().repeat_interleave(block, dim=3)[..., None]


def _round64(x, code):
    """The nearest code, ties to the even one; |x| does not pass the largest."""
    if code == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0**-6)))
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, e)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tables":
        return None  # whole numbers: they are compared as they are
    half = HALF[case["half"]]
    big = float(torch.finfo(half).max)
    page, block, heads, dim = case["page"], case["block"], case["heads"], case["dim"]
    if op in ("write", "read"):
        value = _value64(s["kv"], s["scales"], page, block)
        scale = s["scales"].double()
        if op == "write":
            ctx, q = _write_lengths(case)
            at, slots = 0, s["slots"].tolist()
            x = torch.stack([s["keys"], s["values"]], 2).double()
            top = QMAX[case["code"]]
            while at < len(slots):
                end, b = at, slots[at] // block
                while end < len(slots) and slots[end] // block == b:
                    end += 1
                pg, sub, o = b // (page // block), b % (page // block), slots[at] % block
                amax = x[at:end].abs().amax((0, 3))                                     # [heads, 2]
                fresh = torch.exp2(torch.ceil(torch.log2((amax / top).clamp(min=2.0**-126))))
                fresh = torch.where(amax <= top * fresh / 2, fresh / 2, fresh).clamp(min=2.0**-126)
                sc = fresh if o == 0 else torch.maximum(scale[pg, :, :, sub], fresh)
                rows = slice(sub * block, sub * block + o)
                value[pg, :, :, rows] = _round64(value[pg, :, :, rows] / sc[..., None, None], case["code"]) * sc[..., None, None]
                new = _round64((x[at:end] / sc[..., None]).clamp(-top, top), case["code"]) * sc[..., None]
                value[pg, :, :, sub * block + o: sub * block + o + end - at] = new.permute(1, 2, 0, 3)
                # rows behind the new ones keep their codes, whatever scale stands over them now
                tail = slice(sub * block + o + end - at, (sub + 1) * block)
                value[pg, :, :, tail] *= (sc / scale[pg, :, :, sub])[..., None, None]
                scale[pg, :, :, sub] = sc
                at = end
            slot = s["all_slots"].long()
        else:
            slot = s["slots"].long()
        x = value[slot // page, :, :, slot % page].clamp(-big, big)
        if op == "read":
            return [x[:, :, 0], x[:, :, 1]]
        return {"keys": x[:, :, 0], "values": x[:, :, 1], "scales": scale}
    out = torch.zeros(s["queries"].shape, dtype=torch.float64, device="cuda")
    group = case["heads_q"] // heads
    at = 0
    for i, (n, kv) in enumerate(_attention_lengths(case)):
        pg = s["tables"][i, : _cdiv(kv, page)].long()
        v = _value64(s["kv"][pg] if case["code"] == "int8" else s["kv"].view(torch.uint8)[pg].view(s["kv"].dtype), s["scales"][pg], page, block)
        k, v = (v[:, :, j].permute(1, 0, 2, 3).reshape(heads, -1, dim)[:, :kv] for j in (0, 1))
        for h in range(heads):
            q = s["queries"][at: at + n, h * group: (h + 1) * group].double().permute(1, 0, 2)          # [G, n, D]
            x = q @ k[h].T / math.sqrt(dim)
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            pos = torch.arange(kv - n, kv, device="cuda")[:, None]
            key = torch.arange(kv, device="cuda")[None, :]
            hidden = key > pos
            if case["window"]:
                hidden = hidden | (key <= pos - case["window"])
            x = x.masked_fill(hidden, float("-inf"))
            if s["sinks"] is not None:
                extra = s["sinks"][h * group: (h + 1) * group, None, :].double().expand(group, n, -1)
                p = torch.softmax(torch.cat([x, extra], -1), -1)[..., :kv]
            else:
                p = torch.softmax(x, -1)
            out[at: at + n, h * group: (h + 1) * group] = (p @ v[h]).permute(1, 0, 2)
        at += n
    return out
