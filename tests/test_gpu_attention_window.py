"""GPU: attention with a window over a cache whose pages behind the window were given up, as a server with a sliding window
does: entries of the table that no row needs are no pages, and what the first page that is needed holds below the
window was never written. Tolerances as in test_gpu_attention.py."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_attention import check, filled, work_of
from test_gpu_kv import TYPES, Batch, open_lane, rand_rows, step

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

CASES = [
    # sequences (rows, length), page, kv heads, q heads, D, kind, window
    ([(1, 200)], 16, 2, 8, 128, "bf16", 40),          # the window begins with a tile of 32
    ([(1, 217)], 16, 2, 8, 128, "bf16", 40),          # ... and inside the second run of 16 of one
    ([(1, 201), (1, 90), (1, 3)], 48, 1, 3, 64, "f16", 33),
    ([(1, 9000)], 16, 1, 4, 128, "f16", 4088),        # in parts
    ([(4, 300), (2, 95)], 48, 2, 4, 256, "bf16", 50),
    ([(5, 333), (1, 100)], 16, 1, 16, 64, "bf16", 1),
    ([(200, 700)], 16, 1, 4, 128, "f16", 100),        # many rows
    ([(90, 500), (70, 177), (3, 9)], 48, 1, 2, 64, "bf16", 130),
    ([(150, 1500)], 16, 2, 4, 64, "f16", 40),
    ([(300, 900)], 48, 1, 1, 256, "f16", 77),
    ([(250, 400)], 16, 1, 1, 256, "bf16", 17),
    ([(70, 9000)], 16, 1, 1, 128, "bf16", 5000),      # in parts
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("below", [None, 0x7e7e, 0x7bff, 0x7c00, 0xfc00], ids=lambda b: hex(b) if b else "as-written")
def test_pages_given_up(case, below):
    """The entries of pages that no row needs are no pages (the device flag stays clear), and, but for None, every scale below
    the window in the first page that is needed is `below`: a NaN, the largest number, an infinity of either sign."""
    seqs, P, KV, H, D, kind, window = case
    step(f"attention, pages given up {case} {below}")
    b = Batch(seqs, P, KV, D, seed=D + H)
    c = filled(b, D)
    raw, table = c.raw.copy(), b.table.copy()
    gone = 0
    for i, (n, ln) in enumerate(seqs):
        lo = max(0, ln - n + 1 - window)
        table[i, : lo // P] = [-1, b.n_pages, 2 ** 31 - 1][i % 3]
        gone += lo // P
        if below is not None:
            for tok in range(lo // P * P, lo):
                for place, off in ((c.k_place, 2), (c.v_place, 8)):
                    for d in range(0, D, 32):
                        at = place(tok % P, d)[2]
                        for o in (0, off):
                            raw[b.table[i, tok // P], :, at + o:at + o + 2] = [below & 255, below >> 8]
    assert gone
    b.cache.copy_(torch.from_numpy(raw))
    b.d_table.copy_(torch.from_numpy(table))
    q, q32 = rand_rows(b.rows, H, D, kind, 5, 0, 0.5)
    out = torch.full((b.rows, H, D), 7.0, dtype=TYPES[kind], device="cuda")
    work = work_of(b, H)
    torch.cuda.synchronize()
    with open_lane() as ln:
        ln.attention_async(b.kv, q, out, window=window, work=work)
        ln.sync()   # (raises where a page was looked at that no row needs)
    check(b, c, q32, out.double().cpu().numpy(), H, kind, D ** -0.5, window, 0.0)


@pytest.mark.parametrize("rows", [1, 100])
def test_a_page_that_is_needed_is_still_missed(rows):
    """The page with the window's first token, and the one with the last row's: the device flag."""
    import crosslane_amd as xl
    for col in (lambda lo, ln: lo // 16, lambda lo, ln: (ln - 1) // 16):
        step(f"attention, a page missed {rows}")
        ln, window = 777, 48
        b = Batch([(rows, ln)], 16, 1, 64)
        filled(b, 1)
        b.d_table[0, col(max(0, ln - rows + 1 - window), ln)] = -1
        q, _ = rand_rows(rows, 2, 64, "f16", 5)
        out = torch.zeros((rows, 2, 64), dtype=torch.float16, device="cuda")
        work = work_of(b, 2)
        torch.cuda.synchronize()
        with open_lane() as lane:
            lane.attention_async(b.kv, q, out, window=window, work=work)
            with pytest.raises(xl.XLError, match="cache page"):
                lane.sync()
