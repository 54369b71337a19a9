"""GPU: examples/int8_block.py, a block of an 8-bit model out of the lane's calls, step by
step against plain forms, and as a graph.

Tolerances, E = 2^-24: the norm's as in test_gpu_block_ops.py (33 E of a normed value);
products of int8 are exact sums and two float32 products, compared with the same float
operations on the example's own quants; SwiGLU 8 E and half a step of bf16.
"""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest

import crosslane_amd as xl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
import int8_block  # noqa: E402

E = 2.0 ** -24
DIM, FF, EXPERTS, K = 1024, 512, 16, 4


@pytest.fixture(scope="module")
def lane():
    with xl.Lane(DIM, FF, 1, EXPERTS, np.full((1, EXPERTS, 3), xl.IQ2_XXS, np.int32), max_picks=K, max_tokens=64) as ln:
        ln.generate(3)
        yield ln


def product(q, qs, w, ws):
    acc = (q.double() @ w.double().t()).float()
    return acc * qs[:, None] * ws


@pytest.mark.parametrize("T", [1, 3, 40])
def test_block(lane, T):
    print(f"[gpu-step] int8 block {T}", flush=True)
    s = torch.cuda.Stream()
    b = int8_block.Block(lane, T, 768, K, 4, 2, stream=s.cuda_stream, seed=T)
    y0 = torch.randn((T, DIM), device="cuda")
    b.res.copy_(torch.randn((T, DIM), device="cuda"))
    before = b.res.double().clone()
    torch.cuda.synchronize()
    b.step(y0)
    lane.sync(s.cuda_stream)

    a = y0.double()
    a = a / (a.square().mean(1, keepdim=True) + 1e-6).sqrt() * b.post_w.double() * b.block_gate.double()
    r = before + a
    assert ((b.res.double() - r).abs() <= 36 * E * a.abs() + 2 * E * (before.abs() + a.abs())).all()
    x = r / (r.square().mean(1, keepdim=True) + 1e-6).sqrt() * b.pre_w.double()
    off = 36 * E * (a.abs() + r.abs()).amax(1, keepdim=True) / (r.square().mean(1, keepdim=True)).sqrt() * b.pre_w.double().abs()
    assert ((b.x.double() - x).abs() <= 33 * E * x.abs() + 2 * off).all()
    assert ((b.q.double() * b.q_scale.double()[:, None] - x).abs() <= 0.5001 * b.q_scale.double()[:, None] + 2 * off).all()

    assert torch.equal(b.logits, product(b.q, b.q_scale, b.router_w, b.router_s))
    score = 1 / (1 + torch.exp(-b.logits.double()))
    key = (score + b.bias.double()).cpu().numpy()
    for t in range(T):
        value = [np.sort(key[t, 4 * j:4 * j + 4])[-2:].sum() for j in range(4)]
        kept = sorted(range(4), key=lambda j: (-value[j], j))[:2]
        best = sorted((e for e in range(EXPERTS) if e // 4 in kept), key=lambda e: (-key[t, e], e))[:K]
        assert b.ids[t].tolist() == best
        w = score[t, best] / (score[t, best].sum() + 1e-20) * 2.5
        assert ((b.w[t].double() - w).abs() <= 1.001 * E * w).all()

    g, u = product(b.q, b.q_scale, b.gate_w, b.gate_s).double(), product(b.q, b.q_scale, b.up_w, b.up_s).double()
    h = g / (1 + torch.exp(-g)) * u
    assert ((b.h.double() - h).abs() <= (8 * E + 1.001 * 2.0 ** -8) * h.abs() + 2.0 ** -126).all()
    hf = b.h.float().cpu()   # IEEE quotients (torch's by a number, on the GPU, are products by its inverse)
    hs = hf.abs().amax(1) / torch.full((T,), 127.0)
    hq = torch.round(hf / hs[:, None]).cuda()
    hs = hs.cuda()
    assert torch.equal(b.shared, product(hq, hs, b.down_w, b.down_s))

    # the routed experts, from the same picks by the host's call
    host = np.stack([lane.layer_forward(0, b.ids[t].tolist(), b.w[t].tolist(), b.x[t].cpu().numpy(),
                                        shared=b.shared[t].cpu().numpy()) for t in range(T)])
    got = b.y.cpu().numpy()
    assert np.abs(got - host).max() <= 5e-3 * np.abs(host).max()


@pytest.mark.parametrize("T", [1, 40])
def test_block_in_a_graph(lane, T):
    print(f"[gpu-step] int8 block graph {T}", flush=True)
    s = torch.cuda.Stream()
    b = int8_block.Block(lane, T, 768, K, 4, 2, stream=s.cuda_stream, seed=T)
    y0, start = torch.randn((T, DIM), device="cuda"), torch.randn((T, DIM), device="cuda")
    torch.cuda.synchronize()
    b.step(y0)
    lane.sync(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b.step(y0)
    for _ in range(3):
        y0.copy_(torch.randn((T, DIM), device="cuda"))
        b.res.copy_(start)
        torch.cuda.synchronize()
        b.step(y0)
        lane.sync(s.cuda_stream)
        want = [v.clone() for v in (b.res, b.ids, b.w, b.shared, b.y)]
        b.res.copy_(start)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, (b.res, b.ids, b.w, b.shared, b.y)))
