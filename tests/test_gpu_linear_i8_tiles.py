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


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,N,two", [(1, 16384, 130, True), (1, 16385, 130, False), (1, 8200, 33, False), (1, 4097, 4100, True),
                                       (2, 16384, 70, False), (1, 7, 50, True)])
def test_rows_quantized_by_the_call(lane, T, K, N, two, kind):
    """One float row up to 16384 values is quantized inside the product: as the quantizer does it."""
    print(f"[gpu-step] linear_i8 float row {T} {K} {N} {two} {kind}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(K + N)
    x = torch.randn((T, K + 5), device="cuda", generator=g).to(TYPES[kind][0])[:, :K]
    mats = [rows8(N, K, g) for _ in range(2 if two else 1)]
    ws = [torch.rand(N, device="cuda", generator=g) * 1e-3 for _ in mats]
    q, qs = torch.zeros((T, (K + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :K], torch.zeros(T, device="cuda")
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N, two), dtype=torch.uint8, device="cuda")
    outs = [torch.zeros((T, N), device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    up = (mats[1], ws[1]) if two else (None, None)
    lane.quantize_rows_async(x, q, qs)
    lane.linear_i8_async(q, mats[0], ws[0], outs[0], x_scale=qs, up=up[0], up_scale=up[1], work=work)
    lane.linear_i8_async(x, mats[0], ws[0], outs[1], up=up[0], up_scale=up[1], work=work)
    lane.sync()
    assert torch.equal(outs[0], outs[1])
    xf = x.float().cpu().numpy()   # the quantizer in numpy's float32, whose division is IEEE's
    s = (np.abs(xf).max(1) / np.float32(127)).astype(np.float32)
    assert np.array_equal(qs.cpu().numpy(), s)
    assert np.array_equal(q.cpu().numpy(), np.clip(np.rint(xf / s[:, None]), -127, 127).astype(np.int8))
    if not two:
        assert torch.equal(outs[0], sums(q, mats[0]) * qs[:, None] * ws[0])


def test_quants_next_to_halves(lane):
    """Values whose quotient lies next to a half, where one reciprocal a row would round wrong."""
    print("[gpu-step] quantize_rows next to halves", flush=True)
    rng = np.random.default_rng(9)
    top = np.exp(rng.standard_normal(64) * 8).astype(np.float32)
    x = np.zeros((64, 2048), np.float32)
    half = (rng.integers(-126, 126, (64, 2047)) + 0.5).astype(np.float64)
    x[:, 1:] = (half * (top[:, None].astype(np.float64) / 127)).astype(np.float32)
    x[:, 1:] = np.nextafter(x[:, 1:], (rng.integers(0, 2, (64, 2047)) * 2 - 1) * np.float32(np.inf), dtype=np.float32)
    x[:, 0] = top
    s = (np.abs(x).max(1) / np.float32(127)).astype(np.float32)
    want = np.clip(np.rint(x / s[:, None]), -127, 127).astype(np.int8)
    q, qs = torch.zeros((64, 2048), dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda")
    d = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    lane.quantize_rows_async(d, q, qs)
    lane.sync()
    assert np.array_equal(qs.cpu().numpy(), s) and np.array_equal(q.cpu().numpy(), want)
