"""GPU: the int8 product at sizes that reach each of its kernels' tile shapes, with
several steps of K, ragged in every direction, rows padded with bytes that must not
count, against exact sums in 64 bits (formed on the GPU).

Tolerances: without SwiGLU none (the sum is exact and float32 products are IEEE's,
then one rounding). With it 8 half steps of float32 (expf within two steps, a sum, a
quotient, a product; as in test_gpu_block_ops.py) and half a step of the output.
"""
from __future__ import annotations

import sys

import numpy as np
import pytest

import crosslane_amd as xl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

E = 2.0 ** -24
TYPES = {"f32": (torch.float32, 2.0 ** -24), "f16": (torch.float16, 2.0 ** -11), "bf16": (torch.bfloat16, 2.0 ** -8)}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


@pytest.fixture(scope="module")
def lane():
    with xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32)) as ln:
        yield ln


def rows8(n, k, g, pad=16):
    """Random int8 rows of k bytes in a buffer whose other bytes are random too."""
    return torch.randint(-128, 128, (n, (k + 15) // 16 * 16 + pad), dtype=torch.int8, device="cuda", generator=g)[:, :k]


def sums(x, w):
    """x w^T in float64 (exact: below 2^53), 256 rows at a time, rounded to float32."""
    wt = w.double().t().contiguous()
    return torch.cat([torch.mm(x[i:i + 256].double(), wt).float() for i in range(0, x.shape[0], 256)])


SIZES = [
    # T, K, N, two matrices
    (1, 1337, 4099, False), (1, 1337, 2100, True), (17, 529, 2130, False), (17, 572, 2286, True), (3, 526, 5138, False),
    (24, 8189, 9213, False), (34, 7194, 4302, True), (3, 526, 9231, False), (3, 538, 6714, True), (71, 546, 8272, False),
    (3, 539, 8476, True), (195, 530, 8846, False), (65, 617, 8272, True), (388, 565, 8309, False), (131, 574, 8260, True),
    (641, 564, 6802, False), (397, 521, 6198, True), (5473, 526, 1309, False), (1034, 523, 7438, False),
    (409, 521, 8510, True), (1553, 542, 7120, False), (641, 529, 8770, True), (2051, 4099, 5123, False),
    (4097, 1025, 2051, True),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(map(str, s)))
def test_tiles(lane, size, kind):
    T, K, N, two = size
    print(f"[gpu-step] linear_i8 tiles {size} {kind}", flush=True)
    sys.stdout.flush()
    g = torch.Generator(device="cuda")
    g.manual_seed(T * 31 + N)
    x, mats = rows8(T, K, g), [rows8(N, K, g) for _ in range(2 if two else 1)]
    xs = torch.rand(T, device="cuda", generator=g) * 0.02 + 0.01
    ws = [torch.rand(N, device="cuda", generator=g) * 1e-3 + 1e-4 for _ in mats]
    dt, half = TYPES[kind]
    out = torch.full((T, N + 3), 9.0, dtype=dt, device="cuda")
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N, two), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    lane.linear_i8_async(x, mats[0], ws[0], out[:, :N], x_scale=xs, up=mats[1] if two else None,
                         up_scale=ws[1] if two else None, limit=7.0 if two else 0.0, work=work)
    lane.sync()
    assert (out[:, N:] == 9).all()
    y = [sums(x, w) * xs[:, None] * s for w, s in zip(mats, ws)]
    got = out[:, :N]
    if not two:
        assert torch.equal(got, y[0].to(dt))
        return
    gate, up = y[0].double().clamp(max=7.0), y[1].double().clamp(-7.0, 7.0)
    want = gate / (1 + torch.exp(-gate)) * up
    tol = 8 * E * want.abs() + half * want.abs() * 1.001 + TINY[kind] + 2.0 ** -126
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("T", [40, 300, 2051])
def test_tiles_again(lane, T):
    """A call's repetition, with other calls on their way behind it, gives the same bits."""
    print(f"[gpu-step] linear_i8 again {T}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    K, N = 2304, 5120
    x, w = rows8(T, K, g, 0), rows8(N, K, g, 0)
    xs, ws = torch.rand(T, device="cuda", generator=g), torch.rand(N, device="cuda", generator=g)
    outs = [torch.zeros((T, N), device="cuda") for _ in range(6)]
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for o in outs:
        lane.linear_i8_async(x, w, ws, o, x_scale=xs, work=work)
    lane.sync()
    assert torch.equal(outs[0], sums(x, w) * xs[:, None] * ws)
    assert all(torch.equal(outs[0], o) for o in outs[1:])
