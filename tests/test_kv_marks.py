"""The caches of kv_marks.py: that a lost or doubled run of tokens is outside their bounds, so that a kernel that loses one
fails test_gpu_attention_marks.py. On the CPU."""
from __future__ import annotations

import numpy as np
import pytest

import kv_marks
from kv_ref import Cache, attention, page_bytes

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def made(tokens_of, P, D, ln):
    n = -(-ln // P)
    c = Cache(np.zeros((n, 1, page_bytes(P, D)), np.uint8), P, D)
    kv_marks.fill(c, np.arange(n)[None], [ln], tokens_of)
    kv = [c.values(j, 0) for j in range(n)]
    return [np.concatenate([x[z] for x in kv])[:ln] for z in range(2)]


def test_the_cache_holds_what_it_should():
    k, v = made(kv_marks.counted(64), 48, 64, 100)
    want = np.zeros((100, 64))
    want[np.arange(100), np.arange(100) // 16] = 1 + np.arange(100) % 15
    assert np.array_equal(v, want) and np.isfinite(k).all()
    k, v = made(kv_marks.marked(128, [5, 40]), 16, 128, 60)
    want = np.zeros((60, 128))
    want[5], want[40] = kv_marks.hadamard(128)[:2]
    assert np.array_equal(k, want) and 0.5 < np.abs(v).mean() < 4
    assert np.array_equal(kv_marks.hadamard(64) @ kv_marks.hadamard(64).T, 64 * np.eye(64))


@pytest.mark.parametrize("D,ln,kind", [(64, 9000, "f16"), (128, 12000, "bf16"), (256, 9000, "bf16"), (64, 40000, "f16")])
def test_a_lost_or_doubled_run_shows_in_counts(D, ln, kind):
    _, v = made(kv_marks.counted(D), 64, D, ln)
    want = v.sum(0) / ln
    tol = kv_marks.bound_counted(want, HALF[kind], TINY[kind])
    for at in range(0, ln, 16):
        part, n = v[at:at + 16].sum(0), min(16, ln - at)
        for sign in (-1, 1):
            assert (np.abs((v.sum(0) + sign * part) / (ln + sign * n) - want) > tol).any(), at


@pytest.mark.parametrize("D,ln,kind", [(64, 40000, "bf16"), (128, 5000, "f16"), (256, 9000, "bf16")])
def test_a_lost_or_doubled_mark_shows(D, ln, kind):
    rng = np.random.default_rng(1)
    marks = [0, 31, 32, ln // 2, ln - 1]
    k, v = made(kv_marks.marked(D, marks), 64, D, ln)
    rows = kv_marks.hadamard(D)
    for a, b in ((0, 4), (1, 2), (3, 4)):
        q = (rows[a] + rows[b])[None].astype(np.float64)
        want, A, V, _, cnt = attention(q, k, v, np.array([ln - 1]), kv_marks.SCORE / D, 0, 0.0)
        assert np.allclose(want, (v[marks[a]] + v[marks[b]]) / 2, atol=1e-6)
        tol = kv_marks.bound_marked(want, A, V, cnt, HALF[kind], TINY[kind])
        for share in (0.0, 2 / 3):   # the first one lost, or doubled
            off = np.abs(share * v[marks[a]] + (1 - share) * v[marks[b]] - want)
            assert (off > tol).mean() > 0.8
    q = kv_marks.pairs(D, marks, [ln - 1, 40], 9, 3, rng)
    x = q @ k[marks].T.astype(np.float32) / D
    assert set(np.unique(x)) <= {0.0, 1.0, 2.0} and (x[0, :, 4] == 2).all()
