"""GPU: attention where scores leave float32, and calls repeated."""
from __future__ import annotations

import numpy as np
import pytest

import kv_marks
from test_gpu_attention import CASES, filled, work_of
from test_gpu_kv import TYPES, Batch, lane, rand_rows, step  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def differing(a, b, fill):
    """Where two results differ, for a message."""
    at = (a.view(torch.int16) != b.view(torch.int16)).nonzero()
    if not len(at):
        return ""
    x, y = a[tuple(at.T)].float(), b[tuple(at.T)].float()
    return (f"{len(at)} of {a.numel()} outputs differ, rows, heads and dims from {at.amin(0).tolist()} to {at.amax(0).tolist()}; "
            f"unwritten {int((x == fill).sum())} and {int((y == fill).sum())}, NaN {int(x.isnan().sum())} and {int(y.isnan().sum())}, "
            f"largest difference {float((x - y).abs().nan_to_num(0).max())}")


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_repeats(lane, case):  # noqa: F811
    """The same bits each time, whatever the output and the workspace held."""
    seqs, P, KV, H, D, kind, window, softcap, behind, before, pad = case
    step(f"attention repeated {case}")
    b = Batch(seqs, P, KV, D, behind, before, seed=D + H)
    filled(b, D, 0x7e)
    q, _ = rand_rows(b.rows, H, D, kind, 5, pad, 0.5)
    first = None
    for turn in range(8):
        out = torch.full((b.rows, H, D), 7.0, dtype=TYPES[kind], device="cuda")
        work = work_of(b, H, 0xFF if turn % 2 else 0)
        torch.cuda.synchronize()
        lane.attention_async(b.kv, q, out, window=window, softcap=softcap, work=work)
        lane.sync()
        first = out if first is None else first
        assert not differing(first, out, 7.0), (turn, differing(first, out, 7.0))


@pytest.mark.parametrize("rows,length,H,D", [(1, 40, 2, 64), (3, 2500, 4, 128), (2, 300, 1, 256), (90, 70, 2, 64), (200, 300, 1, 128), (70, 6000, 1, 64),
                                             (300, 500, 1, 256)])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_scores_past_float32(lane, rows, length, H, D, softcap):  # noqa: F811
    """Scores that float32 does not hold, of either sign: NaN, and zeros only for rows that see no token. With a cap they are
    cap and -cap."""
    step(f"attention, scores past float32 {rows} {length} {softcap}")
    b = Batch([(rows, length), (5, 3)], 16, 1, D)
    c = b.ref(0)
    ones, two = np.ones((16, D // 32)), np.full((16, D // 32), 2.0)
    kv_marks.fill(c, b.table, b.lens, lambda *_: ((np.zeros((16, D), int), np.ones((16, D), int)), ((ones, ones), (two, ones))))   # keys 1, values 3
    b.cache.copy_(torch.from_numpy(c.raw))
    q = torch.ones((b.rows, H, D), dtype=torch.float16, device="cuda")
    work = work_of(b, H)
    for scale in (3e38, -3e38):
        out = torch.full((b.rows, H, D), 7.0, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        lane.attention_async(b.kv, q, out, scale=scale, softcap=softcap, work=work)
        lane.sync()
        sees = np.array([p >= 0 for _, _, p in b.places()])
        got = out.float().cpu().numpy()
        assert not got[~sees].any() and (~sees).any()
        assert (np.isnan(got[sees]) if not softcap else got[sees] == 3).all()
