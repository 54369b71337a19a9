"""One MoE block of an 8-bit model around the lane's routed experts.

What a serving loop with an ordinary residual stream and int8 dense weights calls for
each block, on one stream, all of it on the GPU:

    norm      y of the block before -> gate, residual, norm; x in float for the routed
              experts and in int8 for the dense products, in one launch
    logits    the router's product with int8 weights
    route     sigmoid scores, a bias for balance, groups, top-k, renormalized weights
    shared    the shared expert: gate and up with SwiGLU, then down (int8 products)
    routed    the routed experts, joined with the shared one

    python examples/int8_block.py            # times a decode step and a prefill chunk

A decode step is captured into a HIP graph: its launches then cost the host one call.
"""
from __future__ import annotations

import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import crosslane_amd as xl  # noqa: E402


class Block:
    """Weights and buffers of one block for T tokens. `lane`'s layer `layer` holds its routed experts."""

    def __init__(self, lane, T: int, shared_ff: int, k: int, groups: int, top_groups: int, layer: int = 0, seed: int = 0,
                 stream=None):
        import torch
        self.torch, self.lane, self.layer, self.T, self.k = torch, lane, layer, T, k
        self.groups, self.top_groups, self.stream = groups, top_groups, stream
        D, E = lane.dim, lane.n_experts
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        # a model's weights come from its file; float ones are quantized once like this
        self.gate_w, self.gate_s = self.quantized(rand(shared_ff, D) / D ** 0.5)
        self.up_w, self.up_s = self.quantized(rand(shared_ff, D) / D ** 0.5)
        self.down_w, self.down_s = self.quantized(rand(D, shared_ff) / shared_ff ** 0.5)
        self.router_w, self.router_s = self.quantized(rand(E, D) / D ** 0.5)
        self.bias = 0.05 * rand(E)
        self.post_w, self.pre_w = 1 + 0.1 * rand(D), 1 + 0.1 * rand(D)
        self.block_gate = 0.5 + 0.1 * rand(D)
        f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        self.res, self.x, self.y = f(T, D), f(T, D), f(T, D)
        self.q, self.q_scale = torch.zeros((T, D), dtype=torch.int8, device="cuda"), f(T)
        self.logits, self.h, self.shared = f(T, E), torch.zeros((T, shared_ff), dtype=torch.bfloat16, device="cuda"), f(T, D)
        self.ids, self.w = torch.zeros((T, k), dtype=torch.int32, device="cuda"), f(T, k)
        need = max(xl.linear_i8_work_bytes(T, D, E), xl.linear_i8_work_bytes(T, D, shared_ff, gated=True),
                   xl.linear_i8_work_bytes(T, shared_ff, D))
        self.work = torch.empty(need, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def quantized(self, w):
        """A float matrix as int8 rows with a scale each."""
        q = self.torch.zeros((w.shape[0], (w.shape[1] + 15) // 16 * 16), dtype=self.torch.int8, device="cuda")[:, :w.shape[1]]
        scale = self.torch.zeros(w.shape[0], device="cuda")
        self.torch.cuda.synchronize()
        self.lane.quantize_rows_async(w, q, scale)
        self.lane.sync()   # w may go
        return q, scale

    def step(self, y_before) -> None:
        """y_before [T, dim]: the output of the block before. Updates `res`, leaves this block's output in `y`."""
        lane, s = self.lane, self.stream
        lane.block_norm_async(self.res, y=y_before, post_w=self.post_w, gate=self.block_gate, pre_w=self.pre_w,
                              res_out=self.res, x=self.x, q=self.q, q_scale=self.q_scale, stream=s)
        lane.linear_i8_async(self.q, self.router_w, self.router_s, self.logits, x_scale=self.q_scale, work=self.work, stream=s)
        lane.route_scored_async(self.logits, self.k, self.ids, self.w, score="sigmoid", bias=self.bias, groups=self.groups,
                                top_groups=self.top_groups, group_keys=2, scale=2.5, stream=s)
        lane.linear_i8_async(self.q, self.gate_w, self.gate_s, self.h, x_scale=self.q_scale, up=self.up_w, up_scale=self.up_s,
                             work=self.work, stream=s)
        lane.linear_i8_async(self.h, self.down_w, self.down_s, self.shared, work=self.work, stream=s)
        if self.T == 1:
            lane.layer_forward_async(self.layer, self.ids.view(-1), self.w.view(-1), self.x, self.y, shared=self.shared, stream=s)
        else:
            lane.grouped_forward_async(self.layer, self.ids, self.w, self.x, self.y, shared=self.shared, stream=s)


def main() -> None:
    import torch
    dim, ff, E, k = 4096, 2048, 64, 6
    stream = torch.cuda.Stream()
    with xl.Lane(dim, ff, 1, E, np.full((1, E, 3), xl.IQ2_XXS, np.int32), max_picks=k, max_tokens=512) as lane:
        lane.generate(1)
        for T in (1, 512):
            b = Block(lane, T, ff, k, 8, 4, stream=stream.cuda_stream)
            y = torch.randn((T, dim), device="cuda")
            torch.cuda.synchronize()
            b.step(y)
            lane.sync(stream.cuda_stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                b.step(y)
            for name, run, times in (("eager", lambda: b.step(y), 50), ("graph", graph.replay, 50)):
                with torch.cuda.stream(stream):
                    run()
                    torch.cuda.synchronize()
                    start = time.perf_counter()
                    for _ in range(times):
                        run()
                    torch.cuda.synchronize()
                us = (time.perf_counter() - start) / times * 1e6
                print(f"{T} tokens, {name}: {us:.1f} us a block", flush=True)
            lane.sync(stream.cuda_stream)


if __name__ == "__main__":
    main()
