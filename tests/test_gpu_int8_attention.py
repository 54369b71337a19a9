"""GPU: the attention half of examples/int8_block.py before its MoE half, step by step against plain forms.

Products of int8 are exact sums and two float32 products, compared with the same float operations on the example's own
quants, and what the write leaves in cache and queries for equality (test_gpu_kv.py); attention as in
test_gpu_attention.py.
"""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest

import crosslane_amd as xl
from kv_ref import Cache, turned
from test_gpu_attention import check
from test_gpu_int8_block import DIM, EXPERTS, FF, K, lane, product  # noqa: F401
from test_gpu_kv import Batch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
import int8_block  # noqa: E402


def bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.bfloat16)


@pytest.mark.parametrize("n,steps", [(1, (40, 1, 1)), (3, (20, 2, 1))])
def test_block_with_attention(lane, n, steps):  # noqa: F811
    print(f"[gpu-step] int8 block with attention {n} {steps}", flush=True)
    s = torch.cuda.Stream()
    heads, kv, d, page = 8, 2, 64, 16
    seqs = int8_block.Sequences(n, 100, kv, d, page)
    ref = Cache(np.zeros(tuple(seqs.cache.shape), np.uint8), page, d)
    table, length = seqs.table.cpu().numpy(), 0
    for rows in steps:
        T = n * rows
        b = int8_block.Block(lane, T, 768, K, 4, 2, stream=s.cuda_stream, seed=T)
        att = int8_block.Attention(b, seqs, rows, heads, seed=5)
        y0 = torch.randn((T, DIM), device="cuda")
        b.res.copy_(torch.randn((T, DIM), device="cuda"))
        length += rows
        seqs.lens.fill_(length)
        torch.cuda.synchronize()
        att.step(y0)
        middle = b.res.clone()
        b.step(att.y)
        lane.sync(s.cuda_stream)

        qkv = product(att.x, att.x_scale, att.qkv_w, att.qkv_s).to(torch.bfloat16).view(T, heads + 2 * kv, d)
        assert torch.equal(att.qkv, qkv)
        x = qkv.float().cpu().numpy()
        place = np.tile(np.arange(length - rows, length), n)[None].astype(np.int32)
        y = turned(x[:, : heads + kv], att.freqs.cpu().numpy(), place, (d // 2,), False)
        q = bf16(y[:, :heads])
        assert torch.equal(att.q.cpu(), q)
        for t in range(T):
            p = int(place[0, t])
            for h in range(kv):
                ref.put(int(table[t // rows, p // page]), h, p % page, y[t, heads + h], x[t, heads + kv + h])
        assert np.array_equal(seqs.cache.cpu().numpy(), ref.raw)
        as_batch = object.__new__(Batch)
        as_batch.seqs, as_batch.starts, as_batch.P, as_batch.KV, as_batch.D, as_batch.rows, as_batch.table = \
            [(rows, length)] * n, np.arange(n + 1) * rows, page, kv, d, T, table
        check(as_batch, ref, q.float().numpy(), att.att.double().cpu().numpy(), heads, "bf16", d ** -0.5, 0, 0.0)
        a = att.att.view(T, -1).float().cpu()
        scale = a.abs().amax(1) / torch.full((T,), 127.0)
        quants = torch.round(a / scale[:, None]).cuda()
        assert torch.equal(att.y, product(quants, scale.cuda(), att.out_w, att.out_s))
        assert torch.isfinite(b.y).all() and torch.isfinite(middle).all()
