"""GPU: attention calls repeated."""
from __future__ import annotations

import pytest

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
