"""GPU: the scored router at expert counts that reach its widest kernels (8 and 32 experts
a lane) and ties within a lane and across lanes, against the definition in 64 bits one
token at a time (route64 of test_gpu_block_ops.py). Weights: one rounding to float32."""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl
from tests.test_gpu_block_ops import E, held, lane, route64, up  # noqa: F401  (lane: the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def run(lane, lg, bias, score, groups, top, keys, k, renorm, scale, kind="f32"):  # noqa: F811
    T, lg = lg.shape[0], lg.astype(np.float64)   # the definition's exponentials in 64 bits
    with np.errstate(over="ignore"):
        want_ids, want_w = route64(lg, bias, score, groups, top, keys, k, renorm, scale)
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), float("nan"), device="cuda")
    d, b = up(lg.astype(np.float32), 0, kind), None if bias is None else torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()
    lane.route_scored_async(d, k, ids, w, score=score, bias=b, groups=groups, top_groups=top, group_keys=keys, renorm=renorm, scale=scale)
    lane.sync()
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=1.001 * E, atol=2.0 ** -149)


# experts, groups (lanes a group, experts a lane): 512 in 1 (64, 8), 450 in 1 (64, 8), 1020 in 17 (2, 30),
# 1023 in 33 (1, 31), 1024 in 64 (1, 16), 1020 in 34 (1, 30), 700 in 1 (64, 11)
SHAPES = [(512, 1), (450, 1), (1020, 17), (1023, 33), (1024, 64), (1020, 34), (700, 1)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n,groups", SHAPES)
def test_values(lane, n, groups, score, kind):  # noqa: F811
    print(f"[gpu-step] route_scored {n} {groups} {score} {kind}", flush=True)
    rng = np.random.default_rng(n + groups)
    lg = held((2.0 * rng.standard_normal((13, n))).astype(np.float32), kind)   # bf16: many equal logits
    lg[rng.random((13, n)) < 0.1] = -np.inf
    lg[5, rng.random(n) < 0.97] = -np.inf
    bias = (0.2 * rng.standard_normal(n)).astype(np.float32) if score == "sigmoid" else None
    top = min(groups, 4)
    run(lane, lg, bias, score, groups, top, 2, 16, True, 2.5, kind)
    run(lane, lg, bias, score, groups, max(1, groups - 1), 1, 5, False, 1.0, kind)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n,groups", SHAPES)
def test_ties_and_masks(lane, n, groups, score):  # noqa: F811
    print(f"[gpu-step] route_scored ties {n} {groups} {score}", flush=True)
    rng = np.random.default_rng(n)
    lg = np.zeros((11, n), np.float32)
    lg[1] = -np.inf                                  # a row whose mask leaves nothing
    lg[2] = -np.inf
    lg[2, [n - 1, 70, 6, 5]] = [1.0, 1.0, -2.0, 1.0]  # fewer than k are left
    lg[3, ::3] = 1.0                                 # equal logits everywhere
    lg[4, 64::64] = 1.0                              # ... of one lane, where experts go round 64 lanes
    lg[5, 1::2] = 1.0                                # ... of every other lane or slot
    lg[6] = rng.integers(0, 3, n)                    # three values
    lg[7] = np.linspace(-300, 30, n)                 # scores down to underflow
    lg[8, 9] = np.finfo(np.float32).min              # lowest value: a score of 0, not a mask
    lg[9] = np.finfo(np.float32).min
    lg[10] = np.where(rng.random(n) < 0.5, -np.inf, rng.integers(0, 2, n))
    for top, keys, k in ((1, 1, 3), (min(groups, 3), 2, 16), (groups, 2, 9)):
        run(lane, lg, None, score, groups, top, keys, k, True, 1.0)
        run(lane, lg, np.full(n, 0.25, np.float32), score, groups, top, keys, k, False, 1.0)
