"""GPU: attention over caches whose results are known so exactly that a lost, doubled or misweighted tile of tokens shows, at
the borders of tiles, parts and windows. Caches, bounds and their derivation: kv_marks.py (checked in test_kv_marks.py)."""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl
import kv_marks
from kv_ref import attention
from test_gpu_attention import tokens, work_of
from test_gpu_kv import HALF, SMALLEST, TYPES, Batch, lane, step  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

CASES = [
    # sequences (rows, length), page, kv heads, q heads, D, kind, window
    ([(1, 200)], 64, 2, 8, 128, "f16", 0),
    ([(1, 9000), (1, 2)], 64, 1, 4, 64, "f16", 0),
    ([(1, 12000), (1, 1300)], 64, 1, 8, 128, "bf16", 0),
    ([(1, 40000)], 256, 1, 2, 64, "f16", 0),
    ([(1, 9000), (1, 5000)], 48, 1, 4, 128, "f16", 4097),
    ([(2, 9000)], 64, 1, 2, 256, "bf16", 0),
    ([(5, 5000), (3, 700), (12, 4097)], 16, 2, 4, 256, "f16", 3000),
    ([(4, 2049), (7, 31), (16, 4096)], 16, 1, 2, 128, "f16", 0),
    ([(70, 6000), (1, 2)], 64, 1, 1, 64, "f16", 0),
    ([(70, 5000)], 48, 1, 2, 128, "bf16", 0),
    ([(200, 4500)], 64, 1, 1, 256, "f16", 0),
    ([(300, 700), (65, 65), (129, 2000)], 16, 2, 4, 64, "f16", 0),
    ([(150, 1500), (200, 900)], 128, 1, 2, 128, "f16", 77),
    ([(260, 800)], 16, 1, 1, 256, "bf16", 130),
    ([(90, 1200)], 32, 1, 3, 64, "f16", 1),
]
ids = lambda c: "-".join(map(str, c)).replace(" ", "")  # noqa: E731


def run(lane, b, q, H, D, kind, **how):  # noqa: F811
    out = torch.full((b.rows, H, D), 7.0, dtype=TYPES[kind], device="cuda")
    work = work_of(b, H)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, work=work, **how)
    lane.sync()
    return out.double().cpu().numpy()


def fail(off, tol, what):
    bad = np.argwhere(~(off <= tol))
    return f"{what}: {len(bad)} of {off.size} outputs off, the worst {float(np.nanmax(off / tol)):.3g} of the bound; first {bad[:4].tolist()}, last {bad[-1:].tolist()}"


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_counts(lane, case):  # noqa: F811
    seqs, P, KV, H, D, kind, window = case
    step(f"attention, counts {case}")
    b = Batch(seqs, P, KV, D, seed=D)
    c = b.ref(0)
    kv_marks.fill(c, b.table, b.lens, kv_marks.counted(D))
    b.cache.copy_(torch.from_numpy(c.raw))
    got = run(lane, b, torch.zeros((b.rows, H, D), dtype=TYPES[kind], device="cuda"), H, D, kind, window=window)
    for i, (n, ln) in enumerate(seqs):
        upto = np.concatenate([np.zeros((1, D)), np.cumsum(tokens(b, c, i, 0)[1], 0)])
        hi = np.maximum(np.arange(ln - n, ln) + 1, 0)
        lo = np.maximum(hi - window, 0) if window else np.zeros_like(hi)
        want = ((upto[hi] - upto[lo]) / np.maximum(hi - lo, 1)[:, None])[:, None]
        off = np.abs(got[b.starts[i]:b.starts[i] + n] - want)
        tol = np.broadcast_to(kv_marks.bound_counted(want, HALF[kind], SMALLEST[kind]), off.shape)
        assert (off <= tol).all(), fail(off, tol, f"sequence {i}")


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_marks(lane, case):  # noqa: F811
    seqs, P, KV, H, D, kind, window = case
    step(f"attention, marks {case}")
    rng = np.random.default_rng(D)
    longest = max(ln for _, ln in seqs)
    near = [x for n, ln in seqs for p in (ln - 1, ln - n) for x in ((p, p - 1, p - window, p - window + 1) if window else (p, p - 1, p + 1))]
    marks = sorted({x for x in near + [0, 15, 16, 31, 32, 63, 64, 127, 128] if 0 <= x < longest})[:D]
    marks += [x for x in np.linspace(0, longest - 1, D - len(marks)).astype(int).tolist() if x not in marks]
    b = Batch(seqs, P, KV, D, seed=D)
    c = b.ref(0)
    kv_marks.fill(c, b.table, b.lens, kv_marks.marked(D, marks))
    b.cache.copy_(torch.from_numpy(c.raw))
    for turn in range(3):
        q = np.zeros((b.rows, H, D), np.float32)
        for i, (n, ln) in enumerate(seqs):
            q[b.starts[i]:b.starts[i] + n] = kv_marks.pairs(D, marks, range(ln - n, ln), window, H, rng)
        got = run(lane, b, torch.from_numpy(q).to(TYPES[kind]).cuda(), H, D, kind, scale=kv_marks.SCORE / D, window=window)
        for i, (n, ln) in enumerate(seqs):
            at = slice(b.starts[i], b.starts[i] + n)
            for h in range(KV):
                k, v = tokens(b, c, i, h)
                for head in range(h * H // KV, (h + 1) * H // KV):
                    want, A, V, _, cnt = attention(q[at, head].astype(np.float64), k, v, np.arange(ln - n, ln), kv_marks.SCORE / D, window, 0.0)
                    tol = kv_marks.bound_marked(want, A, V, cnt, HALF[kind], SMALLEST[kind])
                    off = np.abs(got[at, head] - want)
                    assert (off <= tol).all(), fail(off, tol, f"turn {turn}, sequence {i}, head {head}")
