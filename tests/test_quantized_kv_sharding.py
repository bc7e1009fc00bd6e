"""KV-head sharding of the 8-bit attention with two gloo ranks on CPU: every rank holds its heads of the cache (axis 1 of
``kv_pages`` and ``kv_scales``) and of the queries; the local compute is the oracle, what is under test is the host logic."""

import os
import socket

import numpy as np
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from ejkernel_b200.modules.operations import quantized_kv
from ejkernel_b200.sharding import Mesh1D, P, kv_head_range
from oracle import q8_oracle


def _batch():
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-100, 101, (9, 4, 2, 8, 64), generator=g).to(torch.int8)
    scales = torch.exp2(torch.randint(-7, -4, (9, 4, 2, 2), generator=g).float())
    tab = torch.randperm(9, generator=g).to(torch.int32).view(3, 3)
    return dict(q=torch.randn((8, 8, 64), generator=g), codes=codes, scales=scales, ctx=torch.tensor([20, 24, 3], dtype=torch.int32), tab=tab,
                start=torch.tensor([0, 1, 6, 8], dtype=torch.int32), n=3)


def _local(queries, kv_pages, kv_scales, context_lens, block_tables, query_start_loc, num_seqs, **kw):
    return torch.from_numpy(q8_oracle.attention(queries, kv_pages, kv_scales, context_lens, block_tables, query_start_loc, num_seqs))


def _worker(rank, world, port, replicate, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    quantized_kv._attention = _local
    b = _batch()
    h0, h1 = kv_head_range(4, rank, world)
    specs = (P(None, "kv", None), P(None, "kv"), P(None, "kv"), P(), P(), P(), P())
    out = quantized_kv.quantized_ragged_page_attention(
        b["q"][:, h0 * 2: h1 * 2].contiguous(), b["codes"][:, h0:h1].contiguous(), b["scales"][:, h0:h1].contiguous(), b["ctx"], b["tab"], b["start"], b["n"],
        mesh=Mesh1D("kv"), in_specs=specs, out_specs=P() if replicate else P(None, "kv", None))
    ret[rank] = out.numpy()
    dist.destroy_process_group()


def _run(replicate):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ret = mp.get_context("spawn").Manager().dict()
    mp.spawn(_worker, args=(2, port, replicate, ret), nprocs=2)
    b = _batch()
    return ret, q8_oracle.attention(b["q"], b["codes"], b["scales"], b["ctx"], b["tab"], b["start"], b["n"])


def test_a_head_sharded_output_stays_local():
    ret, want = _run(False)
    assert np.array_equal(np.concatenate([ret[0], ret[1]], 1), want)


def test_a_replicated_output_is_gathered():
    ret, want = _run(True)
    assert np.array_equal(ret[0], want) and np.array_equal(ret[1], want)
