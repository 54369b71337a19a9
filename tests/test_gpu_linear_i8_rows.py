"""GPU: a token's outputs of the int8 product depend on that token alone: the same bits
whether it comes alone, in a slice that another kernel serves, or among tokens that
change. Sums are exact and the float operations behind them the same in every kernel, so
there is no tolerance."""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lane():
    with xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32)) as ln:
        yield ln


def rows8(n, k, g):
    """Random rows in a buffer whose other bytes are random too."""
    return torch.randint(-127, 128, (n, (k + 15) // 16 * 16 + 16), dtype=torch.int8, device="cuda", generator=g)[:, :k]


CASES = [
    # T, K, N, two matrices, x, out
    (40, 700, 300, False, "i8", "f32"), (300, 700, 300, True, "i8", "bf16"), (300, 515, 1030, False, "f32", "f32"),
    (129, 1337, 2100, True, "bf16", "f16"), (700, 529, 4400, True, "f16", "f32"), (1500, 257, 5123, False, "i8", "f16"),
    (1553, 542, 7120, False, "bf16", "bf16"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_a_token_alone_and_among_others(lane, case):
    T, K, N, two, kind, out_kind = case
    print(f"[gpu-step] linear_i8 tokens alone and together {case}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(T + K + N)
    mats = [(rows8(N, K, g), torch.rand(N, device="cuda", generator=g) * 1e-2) for _ in range(2 if two else 1)]
    up = dict(up=mats[1][0], up_scale=mats[1][1], limit=7.0) if two else {}
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N, two), dtype=torch.uint8, device="cuda")

    def tokens(n):
        if kind == "i8":
            return rows8(n, K, g), torch.rand(n, device="cuda", generator=g) * 0.02 + 0.01
        return torch.randn((n, K + 3), device="cuda", generator=g).to(TYPES[kind])[:, :K], None

    def call(x, xs):
        out = torch.full((x.shape[0], N), float("nan"), dtype=TYPES[out_kind], device="cuda")
        torch.cuda.synchronize()
        lane.linear_i8_async(x, mats[0][0], mats[0][1], out, x_scale=xs, work=work, **up)
        lane.sync()
        assert torch.isfinite(out).all()
        return out

    x, xs = tokens(T)
    part = lambda lo, hi: call(x[lo:hi], None if xs is None else xs[lo:hi])  # noqa: E731
    whole = call(x, xs)
    for t in (0, 1, T // 2, T - 2, T - 1):
        assert torch.equal(part(t, t + 1)[0], whole[t]), t
    for lo, hi in ((0, 2), (3, 20), (T - 33, T), (T // 3, T // 3 + T // 2), (1, T)):
        assert torch.equal(part(lo, hi), whole[lo:hi]), (lo, hi)
    # others' values: the kept tokens' bits stay, the changed ones' do not
    other, os_ = tokens(T)
    kept = torch.rand(T, device="cuda", generator=g) < 0.5
    x[~kept] = other[~kept]
    if xs is not None:
        xs[~kept] = os_[~kept]
    again = call(x, xs)
    assert torch.equal(again[kept], whole[kept]) and (again[~kept] != whole[~kept]).any(1).all()
