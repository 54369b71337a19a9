"""GPU: rotary positions and the 4-bit cache, written and read back, against numpy.

The write is exact: its float32 steps and the float64 angles are numpy's, so every byte of
the cache, and every value of q_out, is compared for equality. (A cosine may differ in the last of its
53 bits from numpy's; it is rounded to 24, which hides that but for one in 2^28.) The read is one product
that is exact in float32 and one sum, rounded to float32 and then to the output: 2^-24 of the value and
half a step of the output, or half a subnormal's spacing.
"""
from __future__ import annotations

import sys

import numpy as np
import pytest

import crosslane_amd as xl
from kv_ref import Cache, page_bytes, turned

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}
FILL = 0xA5


def step(msg):
    print(f"[gpu-step] {msg}", flush=True)
    sys.stdout.flush()


def open_lane():
    return xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32))


@pytest.fixture(scope="module")
def lane():
    with open_lane() as ln:
        yield ln


class Batch:
    """Sequences of (rows, length), their pages anywhere in a cache full of FILL; `behind` rows more than they have."""

    def __init__(self, seqs, P, KV, D, behind=0, before=0, stride_pad=0, seed=0, fill=FILL, max_rows=None):
        rng = np.random.default_rng(seed)
        self.seqs, self.P, self.KV, self.D = seqs, P, KV, D
        cols = max(max(-(-ln // P) for _, ln in seqs), 1) + 1
        need = sum(-(-ln // P) for _, ln in seqs)
        self.n_pages = need + 2
        order = rng.permutation(self.n_pages)[:need]
        self.table = np.full((len(seqs), cols), -7, np.int32)
        at = 0
        for i, (_, ln) in enumerate(seqs):
            n = -(-ln // P)
            self.table[i, :n] = order[at:at + n]
            at += n
        self.starts = before + np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.lens = np.array([ln for _, ln in seqs], np.int32)
        self.rows = int(self.starts[-1]) + behind
        pb = page_bytes(P, D)
        whole = torch.full((self.n_pages, KV * pb + stride_pad), fill, dtype=torch.uint8, device="cuda")
        self.whole = whole
        self.cache = whole[:, :KV * pb].view(self.n_pages, KV, pb) if not stride_pad else \
            torch.as_strided(whole, (self.n_pages, KV, pb), (KV * pb + stride_pad, pb, 1))
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
        self.d_table, self.d_lens, self.d_starts = up(self.table), up(self.lens), up(self.starts)
        self.kv = xl.KVBatch(self.cache, self.d_table, self.d_lens, self.d_starts, self.rows, D,
                             max_rows=max_rows or max(1, max(n for n, _ in seqs)))

    def places(self):
        """(row, sequence, position) of every row of the sequences."""
        for i, (n, ln) in enumerate(self.seqs):
            for j in range(n):
                yield int(self.starts[i]) + j, i, ln - n + j

    def ref(self, fill=FILL):
        raw = np.full((self.n_pages, self.KV, page_bytes(self.P, self.D)), fill, np.uint8)
        return Cache(raw, self.P, self.D)


def rand_rows(T, heads, D, kind, seed, pad=0, spread=1.0):
    """[T, heads, D] inside wider rows of NaNs, and its float32 values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, heads, D), generator=g) * torch.exp(spread * torch.randn((1, heads, D), generator=g))
    buf = torch.full((T, heads * D + pad), float("nan"), dtype=TYPES[kind])
    buf[:, :heads * D] = x.to(TYPES[kind]).view(T, -1)
    d = buf.cuda()[:, :heads * D].unflatten(1, (heads, D))
    return d, buf[:, :heads * D].float().view(T, heads, D).numpy()


WRITES = [
    # sequences (rows, length), page, kv heads, q heads, D, kind, axes, n_freqs, sections, interleaved, behind, before, pad
    ([(1, 1)], 16, 1, 1, 64, "f32", 1, 32, None, False, 0, 0, 0),
    ([(1, 1000)], 64, 8, 32, 128, "bf16", 1, 64, None, False, 0, 0, 0),
    ([(5, 5), (0, 9), (1, 17), (33, 70)], 16, 2, 6, 64, "f16", 1, 32, None, True, 3, 2, 8),
    ([(40, 130), (3, 3)], 48, 3, 3, 128, "bf16", 3, 64, (24, 20, 20), False, 0, 0, 5),
    ([(17, 50)], 1024, 1, 16, 256, "f32", 2, 100, (100, 0), True, 1, 0, 3),
    ([(9, 100), (2, 2)], 32, 2, 4, 64, "f16", 3, 13, (1, 5, 7), False, 0, 0, 1),
    ([(7, 33)], 16, 5, 0, 128, "f32", 0, 0, None, False, 2, 0, 0),
    ([(4, 2), (3, 0), (2, 5)], 16, 1, 2, 64, "bf16", 1, 24, None, False, 0, 0, 0),      # rows before the first token
    ([(600, 601)], 16, 1, 2, 64, "bf16", 1, 32, None, True, 0, 0, 0),
]


@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_write_and_read(lane, case):
    seqs, P, KV, H, D, kind, axes, n, sections, inter, behind, before, pad = case
    step(f"kv write and read {case}")
    b = Batch(seqs, P, KV, D, behind, before, stride_pad=16 * (pad % 3), seed=D)
    T = b.rows
    k, k32 = rand_rows(T, KV, D, kind, 1, pad)
    v, v32 = rand_rows(T, KV, D, kind, 2, pad)
    ref, at = b.ref(), list(b.places())
    q = q_out = freqs = pos = None
    q32 = np.zeros((T, 0, D), np.float32)
    if n:
        f = (10000.0 ** (-np.arange(n) / n)).astype(np.float32)
        f[0] = 0.7390851   # no short binary fraction
        freqs = torch.from_numpy(f).cuda()
        if axes > 1:
            places = np.random.default_rng(3).integers(-50, 2 ** 22, (axes, T)).astype(np.int32)
            wide = torch.full((axes, T + pad), -1, dtype=torch.int32)
            wide[:, :T] = torch.from_numpy(places)
            pos = wide.cuda()[:, :T]
        else:
            places = np.zeros((1, T), np.int32)
            for t, _, p in at:
                places[0, t] = p
        if H:
            q, q32 = rand_rows(T, H, D, kind, 3, pad)
            q_out = torch.full((T, H * D + pad), 7.0, dtype=TYPES[kind], device="cuda")[:, :H * D].unflatten(1, (H, D))
        secs = sections or (n,)
        k32, q32 = turned(k32, f, places, secs, inter), turned(q32, f, places, secs, inter)
    torch.cuda.synchronize()
    lane.kv_write_async(b.kv, k, v, q=q, q_out=q_out, freqs=freqs, positions=pos, sections=sections, interleaved=inter)
    lane.sync()
    for t, i, p in at:
        if p >= 0:
            for h in range(KV):
                ref.put(b.table[i, p // P], h, p % P, k32[t, h], v32[t, h])
    assert np.array_equal(b.cache.cpu().numpy(), ref.raw)
    assert (b.whole[:, KV * page_bytes(P, D):] == FILL).all()
    if q is not None:
        want = np.full((T, H, D), 7.0, np.float32)
        for t, _, p in at:
            want[t] = q32[t] if p >= 0 else 0
        assert torch.equal(q_out.cpu(), torch.from_numpy(want).to(TYPES[kind]))

    for out in TYPES:
        got = [torch.full((T, KV * D + pad), 7.0, dtype=TYPES[out], device="cuda")[:, :KV * D].unflatten(1, (KV, D)) for _ in range(2)]
        torch.cuda.synchronize()
        lane.kv_read_async(b.kv, *got)
        lane.sync()
        want = np.full((2, T, KV, D), 7.0)
        for t, i, p in at:
            for h in range(KV):
                want[:, t, h] = [x[p % P] for x in ref.values(b.table[i, p // P], h)] if p >= 0 else 0
        for g, w in zip(got, want):
            off = np.abs(g.double().cpu().numpy() - w)
            assert (off <= (1.001 * HALF[out] + 2.0 ** -24) * np.abs(w) + SMALLEST[out]).all(), off.max()


def test_values_at_the_ends(lane):
    """Equal values, tiny ones (scales that are subnormal or 0 in float16), and ones past the range."""
    step("kv write: ends of the range")
    D, rows = 64, []
    for lo, hi in ((1.0, 1.0), (0.0, 0.0), (-3e-8, 4e-8), (1e-7, 2e-6), (1.0, 1.00001), (-1e30, 1e30), (40000.0, 50000.0), (-32768.0, 32768.0),
                   (-70000.0, 1.0), (-1e-40, 1e-40)):
        rows.append(np.linspace(lo, hi, D, dtype=np.float32))
    T = len(rows)
    b = Batch([(T, T)], 16, 1, D)
    x = np.stack(rows)[:, None, :]
    d = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    lane.kv_write_async(b.kv, d, -d)
    lane.sync()
    ref = b.ref()
    for t in range(T):
        ref.put(b.table[0, 0], 0, t, x[t, 0], -x[t, 0])
    assert np.array_equal(b.cache.cpu().numpy(), ref.raw)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_that_are_not_finite(D):
    """Held as NaNs, with the device flag; their neighbours as ever."""
    step(f"kv write: not finite {D}")
    T, KV = 6, 3
    b = Batch([(T, T)], 16, KV, D)
    k, k32 = rand_rows(T, KV, D, "f32", 1)
    v, v32 = rand_rows(T, KV, D, "f32", 2)
    for x, x32, t, h, d, bad in ((k, k32, 2, 1, D - 1, np.nan), (k, k32, 5, 0, 0, np.inf), (v, v32, 2, 1, 3, -np.inf), (v, v32, 0, 2, D // 2, np.nan)):
        x[t, h, d] = bad
        x32[t, h, d] = bad
    torch.cuda.synchronize()
    with open_lane() as ln:
        ln.kv_write_async(b.kv, k, v)
        with pytest.raises(xl.XLError, match="non-finite"):
            ln.sync()
    ref = b.ref()
    for t in range(T):
        for h in range(KV):
            ref.put(b.table[0, 0], h, t, k32[t, h], v32[t, h])
    assert np.array_equal(b.cache.cpu().numpy(), ref.raw)


def test_batches_out_of_range():
    """Pages that are none, lengths past the table, starts that descend or pass the rows: the device
    flag, nothing outside the cache and the outputs, and the other sequences as ever."""
    D, P, KV = 64, 16, 2
    for what in ("page", "length", "starts", "rows", "max_rows"):
        step(f"kv batch out of range: {what}")
        b = Batch([(4, 20), (5, 30), (3, 40)], P, KV, D, behind=2, stride_pad=16, max_rows=5)
        k, k32 = rand_rows(b.rows, KV, D, "f32", 1)
        v, v32 = rand_rows(b.rows, KV, D, "f32", 2)
        off = {1}
        if what == "page":
            b.d_table[1, 1] = b.n_pages
            off_pos = lambda p: p >= 16   # noqa: E731
        else:
            off_pos = lambda p: True   # noqa: E731
        if what == "length":
            b.d_lens[1] = b.table.shape[1] * P + 1
        if what == "starts":
            b.d_starts[:] = torch.tensor([0, 4, 3, 12], dtype=torch.int32)
            off = {0, 1, 2}
        if what == "rows":
            b.d_starts[3] = b.rows + 1
            off = {2}
        if what == "max_rows":
            b.kv = xl.KVBatch(b.cache, b.d_table, b.d_lens, b.d_starts, b.rows, D, max_rows=4)
        got = [torch.full((b.rows, KV, D), 7.0, device="cuda") for _ in range(2)]
        q = torch.zeros((b.rows, KV, D), dtype=torch.float16, device="cuda")
        out = torch.full_like(q, 7.0)
        torch.cuda.synchronize()
        for call in (lambda ln: ln.kv_write_async(b.kv, k, v), lambda ln: ln.kv_read_async(b.kv, *got),
                     lambda ln: ln.attention_async(b.kv, q, out, work=torch.empty(xl.attention_work_bytes(b.kv, KV) + 256, dtype=torch.uint8,
                                                                                  device="cuda"))):
            with open_lane() as ln:
                call(ln)
                with pytest.raises(xl.XLError, match="cache page, length or start"):
                    ln.sync()
        assert (b.whole[:, KV * page_bytes(P, D):] == FILL).all()
        ref = b.ref()
        for t, i, p in b.places():
            if i not in off or (what == "page" and not off_pos(p)):
                for h in range(KV):
                    ref.put(b.table[i, p // P], h, p % P, k32[t, h], v32[t, h])
        if what != "starts":   # (of descending starts some rows still belong to a sequence)
            assert np.array_equal(b.cache.cpu().numpy(), ref.raw), what
        assert (out[-2:] == 7).all() and (got[0][-2:] == 7).all()
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("rows", [3, 40])
def test_read_into_columns(lane, rows):
    """Keys and values as columns of the same rows."""
    step(f"kv read into columns {rows}")
    b = Batch([(rows, 50), (2, 2)], 16, 2, 64)
    k, k32 = rand_rows(b.rows, 2, 64, "f16", 1)
    v, v32 = rand_rows(b.rows, 2, 64, "f16", 2)
    both = torch.full((b.rows, 5, 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    lane.kv_write_async(b.kv, k, v)
    lane.kv_read_async(b.kv, both[:, 3:], both[:, :2])
    lane.sync()
    ref = b.ref()
    for t, i, p in b.places():
        for h in range(2):
            ref.put(b.table[i, p // 16], h, p % 16, k32[t, h], v32[t, h])
    got = both.cpu().numpy()
    assert (got[:, 2] == 7).all()
    for t, i, p in b.places():
        for h in range(2):
            x, y = (z[p % 16] for z in ref.values(b.table[i, p // 16], h))
            assert np.abs(got[t, 3 + h] - x).max() <= 2.0 ** -23 * np.abs(x).max() and np.abs(got[t, h] - y).max() <= 2.0 ** -23 * np.abs(y).max()


def test_sections_refused(lane):
    step("cache write, sections refused")
    b = Batch([(1, 5)], 16, 1, 64)
    k = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    freqs = torch.ones(32, device="cuda")
    torch.cuda.synchronize()
    for sections in ((2 ** 32 + 32,), (32.0,), (33,), (-32,), (32, 0)):
        with pytest.raises(xl.XLError, match="section"):
            lane.kv_write_async(b.kv, k, k, freqs=freqs, sections=sections)
    lane.kv_write_async(b.kv, k, k, freqs=freqs, sections=[32])
    lane.sync()
