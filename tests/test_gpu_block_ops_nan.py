"""GPU: NaNs through the gate and up product with a limit. The definition's clamps keep a
NaN (as the product without a limit does), so a row or a channel that has one has NaNs in
its outputs, and no finite numbers; every other output is the definition's.

Tolerances: E = 2^-24, half a step of float32. Sums and their two products are exact or
IEEE's, then 8 E for SwiGLU (expf within two steps, a sum, a quotient, a product) and
half a step of the output, or half a subnormal's spacing. exp(-g) overflows float32 below
g = -88.7: the quotient is then 0 for at most 89 * 2^-128, times u.
"""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

E = 2.0 ** -24
TYPES = {"f32": (torch.float32, 2.0 ** -24, 2.0 ** -149), "f16": (torch.float16, 2.0 ** -11, 2.0 ** -24),
         "bf16": (torch.bfloat16, 2.0 ** -8, 2.0 ** -133)}   # half a step; spacing of the subnormals
NAN = float("nan")


def open_lane():
    return xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32))


def rows8(n, k, g):
    return torch.randint(-127, 128, (n, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda", generator=g)[:, :k]


def definition(q, qs, mats, lim):
    """In 64 bits from the float32 products; torch's clamp keeps a NaN."""
    g, u = [((q.double() @ w.double().t().contiguous()).float() * qs[:, None] * ws).double() for w, ws in mats]
    g, u = g.clamp(max=lim), u.clamp(-lim, lim)
    return g / (1 + torch.exp(-g)) * u


def close(got, want, kind, lim):
    _, half, spacing = TYPES[kind]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    tol = (8 * E + 1.001 * half) * want[ok].abs() + spacing / 2 + 89 * lim * 2.0 ** -128
    assert ((got.double()[ok] - want[ok]).abs() <= tol).all()


# T, K, N: the call of few tokens with one and with more token tiles, then calls of tiles
SIZES = [(1, 300, 70), (5, 129, 40), (30, 1000, 200), (70, 546, 4000), (300, 200, 300), (700, 529, 4400)]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(map(str, s)))
def test_nan_scales(size, kind):
    """int8 x: a NaN among the scales of the tokens, the gate's channels or the up channels. No flag: these are the caller's."""
    T, K, N = size
    print(f"[gpu-step] gated linear_i8, NaN scales {size} {kind}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(T + K)
    q, mats = rows8(T, K, g), [(rows8(N, K, g), torch.rand(N, device="cuda", generator=g) * 1e-2) for _ in range(2)]
    qs = torch.rand(T, device="cuda", generator=g) * 0.02 + 0.01
    if T > 1:
        qs[T // 2] = NAN
    mats[0][1][3] = NAN
    mats[1][1][N - 1] = NAN
    dt = TYPES[kind][0]
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N, True), dtype=torch.uint8, device="cuda")
    with open_lane() as lane:
        for lim in (7.0, 0.5):
            out = torch.zeros((T, N), dtype=dt, device="cuda")
            torch.cuda.synchronize()
            lane.linear_i8_async(q, mats[0][0], mats[0][1], out, x_scale=qs, up=mats[1][0], up_scale=mats[1][1], limit=lim, work=work)
            lane.sync()
            close(out, definition(q, qs, mats, lim), kind, lim)
            assert torch.isnan(out[:, [3, N - 1]]).all() and not torch.isnan(out[0, 4:N - 1]).any()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), NAN])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(map(str, s)))
def test_rows_that_are_no_numbers(size, kind, value):
    """Float x: the row's products are NaN, the call is reported, the other rows are theirs."""
    T, K, N = size
    print(f"[gpu-step] gated linear_i8, a row with {value} {size} {kind}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(T + N)
    dt = TYPES[kind][0]
    x = torch.randn((T, K), device="cuda", generator=g).to(dt)
    x[T // 2, K - 2] = value
    mats = [(rows8(N, K, g), torch.rand(N, device="cuda", generator=g) * 1e-2) for _ in range(2)]
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N, True), dtype=torch.uint8, device="cuda")
    out = torch.zeros((T, N), dtype=dt, device="cuda")
    torch.cuda.synchronize()
    with open_lane() as lane:
        lane.linear_i8_async(x, mats[0][0], mats[0][1], out, up=mats[1][0], up_scale=mats[1][1], limit=7.0, work=work)
        with pytest.raises(xl.XLError, match="non-finite"):
            lane.sync()
    torch.cuda.synchronize()
    assert torch.isnan(out[T // 2]).all()
    xf = x.float().cpu()   # IEEE quotients (torch's by a number, on the GPU, are products by its inverse)
    xf[T // 2] = 0
    s = xf.abs().amax(1) / torch.full((T,), 127.0)
    q = torch.where(s[:, None] > 0, torch.round(xf / s[:, None]), 0.0).cuda()
    s[T // 2] = NAN
    close(out, definition(q, s.cuda(), mats, 7.0), kind, 7.0)
