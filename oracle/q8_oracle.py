"""Plain restatements, in 64 bits on the CPU, of the operators around the 8-bit paged KV cache (test infrastructure only).

The cache is ``codes [P, Hkv, 2, page, D]`` (e4m3 or int8) with ``scales [P, Hkv, 2, page / block]``.  Everything here walks
rows, blocks and sequences one after the other, from the operators' definitions.
"""

from __future__ import annotations

import math

import numpy as np
import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def values_of(codes: torch.Tensor, scales: torch.Tensor) -> np.ndarray:
    """The cache's values [P, Hkv, 2, page, D]."""
    block = codes.shape[3] // scales.shape[3]
    c = codes.cpu().to(torch.float32).numpy().astype(np.float64)
    return c * np.repeat(scales.cpu().numpy().astype(np.float64), block, axis=3)[..., None]


def round_to_code(x: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    """The nearest code value, ties to even; |x| <= QMAX."""
    if dtype == torch.int8:
        return np.rint(x)
    # e4m3: steps of 2^(e-3) in [2^e, 2^(e+1)), 2^-9 below 2^-6
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0**-7))), -6.0)
    step = 2.0 ** (e - 3)
    return np.rint(x / step) * step


def scale_for(amax: float, dtype: torch.dtype) -> float:
    s = 2.0**-126
    while amax > QMAX[dtype] * s:
        s *= 2.0
    return s


def write(keys, values, codes, scales, slots):
    """The cache after the write: (code values [P, Hkv, 2, page, D], scales), float64.  Inputs are not changed."""
    dtype = codes.dtype
    page, block = codes.shape[3], codes.shape[3] // scales.shape[3]
    per = page // block
    c = codes.cpu().to(torch.float32).numpy().astype(np.float64)
    s = scales.cpu().numpy().astype(np.float64).copy()
    x = [t.detach().cpu().to(torch.float64).numpy() for t in (keys, values)]
    slots = slots.cpu().numpy()
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= codes.shape[0] * page:
            t += 1
            continue
        b = slots[t] // block
        end = t
        while end < len(slots) and slots[end] >= 0 and slots[end] // block == b:
            end += 1
        first = slots[t] % block
        pg, sub = b // per, b % per
        for h in range(codes.shape[1]):
            for kv in range(2):
                rows = x[kv][t:end, h]
                finite = np.abs(rows[np.isfinite(rows)])
                sc = scale_for(float(finite.max()) if finite.size else 0.0, dtype)
                if first > 0:
                    old = s[pg, h, kv, sub]
                    if old >= sc:
                        sc = old
                    else:
                        kept = slice(sub * block, sub * block + first)
                        c[pg, h, kv, kept] = round_to_code(c[pg, h, kv, kept] * old / sc, dtype)
                s[pg, h, kv, sub] = sc
                for i in range(t, end):
                    with np.errstate(invalid="ignore"):
                        v = np.clip(x[kv][i, h] / sc, -QMAX[dtype], QMAX[dtype])
                    c[pg, h, kv, slots[i] % page] = round_to_code(np.where(np.isnan(v), 0.0, v), dtype)
        t = end
    return c, s


def attention(q, codes, scales, context_lens, block_tables, query_start_loc, num_seqs, *, softmax_scale=None, window=None,
              cap=None, sinks=None, with_bound=False):
    """float64 [T, Hq, D]; with ``with_bound`` also sum_j p_j |v_j|, what relative errors of the weights are taken of."""
    x = values_of(codes, scales)
    P, Hkv, _, page, D = x.shape
    q = q.detach().cpu().to(torch.float64).numpy()
    T, Hq, _ = q.shape
    G = Hq // Hkv
    scale = D**-0.5 if softmax_scale is None else softmax_scale
    lens, tab, start = context_lens.cpu().tolist(), block_tables.cpu().numpy(), query_start_loc.cpu().tolist()
    if sinks is not None:
        sinks = sinks.detach().cpu().to(torch.float64).numpy()
        sinks = np.repeat(sinks[None], Hq, 0) if sinks.ndim == 1 else np.repeat(sinks, Hq // sinks.shape[0], 0)
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for s in range(int(num_seqs)):
        n, kv = start[s + 1] - start[s], lens[s]
        if n <= 0:
            continue
        pages = tab[s, : -(-kv // page)]
        for h in range(Hkv):
            k = x[pages, h, 0].reshape(-1, D)[:kv]
            v = x[pages, h, 1].reshape(-1, D)[:kv]
            for r in range(n):
                pos = kv - n + r
                lo = max(0, pos - window + 1) if window else 0
                for g in range(G):
                    row, hq = start[s] + r, h * G + g
                    if pos < 0:
                        continue
                    y = (k[lo: pos + 1] @ q[row, hq]) * scale
                    if cap:
                        y = cap * np.tanh(y / cap)
                    m = y.max(initial=-math.inf)
                    if sinks is not None:
                        m = max(m, sinks[hq].max(initial=-math.inf))
                    if m == -math.inf:
                        continue
                    p = np.exp(y - m)
                    total = p.sum() + (np.exp(sinks[hq] - m).sum() if sinks is not None else 0.0)
                    out[row, hq] = p @ v[lo: pos + 1] / total
                    bound[row, hq] = p @ np.abs(v[lo: pos + 1]) / total
    return (out, bound) if with_bound else out


def page_tables(query_lens, context_lens, block_tables, free_pages, num_free, num_seqs, page_size, total_tokens, finished=None):
    """(lens, start, slots, num_free, tables, free) as the definition walks them, lists and arrays; inputs are not changed."""
    q, c = [max(v, 0) for v in query_lens.cpu().tolist()], context_lens.cpu().tolist()
    tab, free = block_tables.cpu().numpy().copy(), free_pages.cpu().numpy().copy()
    S, pps = tab.shape
    n = min(int(num_free), len(free))
    live = min(int(num_seqs), S)
    gone = [finished is not None and bool(finished[s]) for s in range(S)]
    for s in range(live):
        if gone[s]:
            for j in range(-(-c[s] // page_size)):
                if n < len(free):
                    free[n] = tab[s, j]
                    n += 1
    lens, start, slots, exhausted, raw = [0] * S, [0] * (S + 1), [-1] * total_tokens, False, 0
    for s in range(S):
        start[s] = min(raw, total_tokens)
        if s >= live or gone[s]:
            continue
        begin, raw = raw, raw + q[s]
        lens[s] = c[s]
        held = -(-c[s] // page_size)
        need = -(-(c[s] + q[s]) // page_size) - held
        if c[s] + q[s] > pps * page_size:
            continue
        if need > 0 and (exhausted or need > n):
            exhausted = True  # rows are served in order: no later row jumps the queue
            continue
        if raw > total_tokens:
            continue
        for j in range(need):
            n -= 1
            tab[s, held + j] = free[n]
        lens[s] = c[s] + q[s]
        for r in range(q[s]):
            pos = c[s] + r
            slots[begin + r] = int(tab[s, pos // page_size]) * page_size + pos % page_size
    start[S] = min(raw, total_tokens)
    return lens, start, slots, n, tab, free
