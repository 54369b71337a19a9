"""GPU: the block norm with more rows than the workgroups that the chip holds, so that each
workgroup takes several of them in turn: the next row's loads ahead, the vectors over the
channels kept, writing in place while the next row is on its way.

Each case against 64 bits, and bit for bit against calls of so few rows that every row has
a workgroup of its own (which kernel runs depends on the width and the types alone).

Tolerances as in test_gpu_block_ops.py, E = 2^-24: 31 E for an inverse norm (54 E of the
sum of squares, halved by the root, and 4), one more for each product and sum behind it;
half a step of the output.
"""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

E = 2.0 ** -24
EPS = 1e-6
TYPES = {"f32": (torch.float32, 2.0 ** -24, 2.0 ** -149), "f16": (torch.float16, 2.0 ** -11, 2.0 ** -24),
         "bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -133)}   # half a step; spacing of the subnormals
FEW = 200   # rows of a call where each has a workgroup


@pytest.fixture(scope="module")
def lane():
    with xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32)) as ln:
        yield ln


CASES = [
    # rows for each CU (and 37 more), D, type, res_type, post, gate, alpha, pad
    (60, 64, "bf16", "f32", True, "channel", 1.0, 0),         # one wave a row: 24 workgroups to a CU
    (25, 500, "f32", "f32", True, "token", 0.5, 3),           # one wave
    (20, 1500, "f32", "bf16", True, "channel", 1.0, 0),       # three waves: 8 to a CU
    (12, 2304, "bf16", "bf16", True, "channel", 1.0, 0),      # two chunks a thread, kept: 5
    (12, 2304, "bf16", "bf16", False, "token", 2.25, 5),
    (9, 2700, "f32", "f32", True, "channel", -0.75, 1),       # one chunk a thread, six waves: 3
    (5, 4099, "f16", "f32", False, "token", 0.5, 5),          # nine waves: 2
    (5, 4099, "f32", "f16", True, "none", 1.0, 0),
    (7, 5120, "bf16", "bf16", True, "channel", 1.0, 0),
    (5, 8192, "bf16", "bf16", True, "channel", 1.0, 0),       # two chunks, kept
    (3, 8192, "f32", "f32", True, "token", 1.0, 0),           # sixteen waves of one chunk: 1
    (3, 16384, "bf16", "f16", True, "channel", 1.0, 8),       # two chunks, kept: 1
    (3, 16380, "f32", "f32", True, "channel", 1.0, 0),        # two chunks, none kept
    (3, 16384, "f16", "f32", True, "token", 1.0, 3),
    (3, 20000, "f32", "f32", True, "channel", 1.0, 0),        # four chunks
    (3, 20001, "bf16", "bf16", True, "token", 0.5, 0),
    (2, 32768, "bf16", "f32", True, "channel", 1.0, 0),
]


def made(case):
    per_cu, D, kind, rk, post, gate, alpha, pad = case
    T = per_cu * torch.cuda.get_device_properties(0).multi_processor_count + 37
    g = torch.Generator(device="cuda")
    g.manual_seed(D + per_cu)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    wide = lambda kind: n(T, D + pad).to(TYPES[kind][0])[:, :D]  # noqa: E731
    # rows of different sizes: one row's statistics in another's place show
    y, res = wide(kind), wide(rk)
    y *= torch.exp2((torch.arange(T, device="cuda") % 7 - 3).float()).to(y.dtype)[:, None]
    res *= torch.exp2((torch.arange(T, device="cuda") % 5 - 2).float()).to(res.dtype)[:, None]
    pw, nw = (1 + 0.1 * n(D)) if post else None, 1 + 0.1 * n(D)
    gt = {"none": lambda: None, "channel": lambda: n(D).to(y.dtype), "token": lambda: n(T, D).to(y.dtype)}[gate]()
    return T, D, y, res, pw, nw, gt


def outputs(T, D, y, res):
    return {"res_out": torch.full((T, D), 9.0, dtype=res.dtype, device="cuda"), "x": torch.full((T, D), 9.0, dtype=y.dtype, device="cuda"),
            "q": torch.full((T, (D + 15) // 16 * 16), 9, dtype=torch.int8, device="cuda")[:, :D], "q_scale": torch.full((T,), 9.0, device="cuda")}


def within(got, want, off, kind):
    _, half, spacing = TYPES[kind]
    tol = 1.001 * off + half * (want.abs() + off) + spacing
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rows_in_turn(lane, case):
    _, _, kind, rk, _, gate, alpha, _ = case
    print(f"[gpu-step] block_norm rows in turn {case}", flush=True)
    T, D, y, res, pw, nw, gt = made(case)
    got, few = outputs(T, D, y, res), outputs(T, D, y, res)
    torch.cuda.synchronize()
    lane.block_norm_async(res, y=y, post_w=pw, gate=gt, alpha=alpha, pre_w=nw, eps=EPS, **got)
    for i in range(0, T, FEW):
        s = slice(i, i + FEW)
        lane.block_norm_async(res[s], y=y[s], post_w=pw, gate=gt[s] if gate == "token" else gt, alpha=alpha, pre_w=nw, eps=EPS,
                              **{k: v[s] for k, v in few.items()})
    lane.sync()
    for k in got:
        assert torch.equal(got[k], few[k]), k
    for i in range(0, T, 1024):   # in 64 bits, some rows at a time
        s = slice(i, i + 1024)
        a, rel = y[s].double(), 0.0
        if pw is not None:
            a, rel = a / (a.square().mean(1, keepdim=True) + EPS).sqrt() * pw.double(), 33 * E
        if gt is not None:
            a, rel = a * (gt[s] if gate == "token" else gt).double(), rel + E
        scaled = alpha * res[s].double()
        r = scaled + a
        off = rel * a.abs() + E * r.abs() + E * (scaled.abs() + a.abs())
        within(got["res_out"][s], r, off, rk)
        rms = (r.square().mean(1, keepdim=True) + EPS).sqrt()
        x = r / rms * nw.double()
        moved = off.square().mean(1, keepdim=True).sqrt() / rms
        xoff = x.abs() * (33 * E + moved) + off / rms * nw.double().abs()
        within(got["x"][s], x, xoff, kind)
        d = got["q_scale"][s].double()[:, None]
        assert ((d[:, 0] * 127 - x.abs().amax(1)).abs() <= xoff.amax(1) + 2 * E * x.abs().amax(1)).all()
        assert ((got["q"][s].double() * d - x).abs() <= 0.5001 * d + xoff).all()


@pytest.mark.parametrize("case", [c for c in CASES if c[1] in (64, 2304, 5120, 8192, 16380, 16384, 20000)], ids=lambda c: "-".join(map(str, c)))
def test_rows_in_turn_in_place(lane, case):
    """res_out in res's and x in y's place: no row is written before it was read."""
    alpha = case[6]
    print(f"[gpu-step] block_norm rows in turn, in place {case}", flush=True)
    T, D, y, res, pw, nw, gt = made(case)
    want = outputs(T, D, y, res)
    q, qs = torch.zeros((T, (D + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :D], torch.zeros(T, device="cuda")
    torch.cuda.synchronize()
    args = dict(post_w=pw, gate=gt, alpha=alpha, pre_w=nw, eps=EPS)
    lane.block_norm_async(res, y=y, **args, **want)
    lane.block_norm_async(res, y=y, **args, res_out=res, x=y, q=q, q_scale=qs)
    lane.sync()
    assert torch.equal(res, want["res_out"]) and torch.equal(y, want["x"])
    assert torch.equal(q, want["q"]) and torch.equal(qs, want["q_scale"])


@pytest.mark.parametrize("D", [64, 2304, 5120, 20000])
def test_parts_of_the_norm_over_rows_in_turn(lane, D):
    """No y, no residual, no second norm: the turns that skip a reduction, bit for bit against few rows."""
    print(f"[gpu-step] block_norm parts, rows in turn {D}", flush=True)
    T, D, y, res, pw, nw, gt = made((60 if D == 64 else 12, D, "f32", "f32", True, "token", 1.0, 0))
    calls = [dict(res=res, pre_w=nw, out="x"), dict(res=None, y=y, post_w=pw, gate=gt, out="res_out"), dict(res=res, y=y, out="res_out"),
             dict(res=None, y=y, pre_w=nw, out="q"), dict(res=res, alpha=0.5, out="res_out")]
    for c in calls:
        c = dict(c)
        out = c.pop("out")
        names = ("q", "q_scale") if out == "q" else (out,)
        got, few = outputs(T, D, y, res), outputs(T, D, y, res)
        torch.cuda.synchronize()
        lane.block_norm_async(**c, **{n: got[n] for n in names})
        for i in range(0, T, FEW):
            s = slice(i, i + FEW)
            rows = {k: v[s] if k in ("res", "y", "gate") and v is not None else v for k, v in c.items()}
            lane.block_norm_async(**rows, **{n: few[n][s] for n in names})
        lane.sync()
        for n in got:
            assert torch.equal(got[n], few[n]), (c.keys(), n)
        assert not (got[names[0]][:, 0].float() == 9).all()


def test_values_whose_squares_pass_float32(lane):
    """Sums of squares are float32: past its range the norm is 0, with values of the other rows as they are."""
    print("[gpu-step] block_norm, squares past float32", flush=True)
    D = 100
    res = torch.ones((3, D), device="cuda")
    res[1] = 1e20
    x, one = torch.full((3, D), 9.0, device="cuda"), torch.ones(D, device="cuda")
    torch.cuda.synchronize()
    lane.block_norm_async(res, pre_w=one, eps=EPS, x=x)
    lane.sync()
    assert not x[1].any() and ((x[[0, 2]].double() - (1 + EPS) ** -0.5).abs() <= 33 * E).all()
