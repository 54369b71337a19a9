"""GPU: attention over the 4-bit cache against its definition in 64 bits.

Tolerances. U = 2^-11 is half a step of float16, E = 2^-24 of float32. A kernel may round
keys and values to float16 (U of each), hold q in float16 with a power of two for each row (2^-25 of
the row's largest value, besides values that are exact), and sum D products in float32 (2 D E of
the sum of their magnitudes); a row's scores are so off by at most
    S = (1.01 U + 2 D E) * X + 2^-25 * sqrt(D) * X' with X the largest sum of |q k| of a token that it sees,
X' bounded by 4 X here (keys' and q's values are alike in size); then by 16 E of the score for its scaling,
the cap (whose slope is at most 1; tanh within 4 E of 1: 8 E * cap) and the exponential's argument, and the exponential is within
4 E. Weights so differ by the factor exp(2 S'), S' all of that; they may be rounded to float16 (U, and 2^-25 of the largest weight below
its normal range), the values too, and sums of n tokens in float32 add (n + 64) E:
    |out - want| <= A (2.05 S' + 2.02 U + 2 (n + 64) E) + 2^-25 V + half a step of the output
with A the sum of p |v|, V the sum of |v| over the tokens seen, in units of which the largest weight is at least 1 / n.
"""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl
from kv_ref import attention, page_bytes
from test_gpu_kv import FILL, HALF, SMALLEST, TYPES, Batch, lane, open_lane, rand_rows, step  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U, E = 2.0 ** -11, 2.0 ** -24


def filled(b, seed=0, tail=None):
    """The batch's pages full of codes and scales, as a float64 reference sees them; places that no token has
    hold `tail` in every byte (NaN scales for 0x7e)."""
    rng = np.random.default_rng(seed)
    c = b.ref()
    raw = c.raw
    P, D, KV = b.P, b.D, b.KV
    raw[:, :, :c.k_scales] = rng.integers(0, 256, raw[:, :, :c.k_scales].shape)
    raw[:, :, c.v_codes:c.v_scales] = rng.integers(0, 256, raw[:, :, c.v_codes:c.v_scales].shape)
    s = (0.3 * np.exp(0.3 * rng.standard_normal((2, b.n_pages, KV, P, D // 32)))).astype(np.float16)
    m = (-7.5 * s.astype(np.float64) + 0.3 * rng.standard_normal(s.shape)).astype(np.float16)
    both = np.stack([s, m], -1)
    raw[:, :, c.k_scales:c.v_codes] = np.ascontiguousarray(both[0]).view(np.uint8).reshape(b.n_pages, KV, -1)
    v = both[1].reshape(b.n_pages, KV, P // 4, 4, D // 32, 2).transpose(0, 1, 2, 4, 5, 3)
    raw[:, :, c.v_scales:] = np.ascontiguousarray(v).view(np.uint8).reshape(b.n_pages, KV, -1)
    if tail is not None:   # page parts behind the sequences, and pages of none
        used = np.zeros((b.n_pages, P), bool)
        for i, (_, ln) in enumerate(b.seqs):
            for j in range(ln):
                used[b.table[i, j // P], j % P] = True
        for page in range(b.n_pages):
            for tok in np.nonzero(~used[page])[0]:
                for place, off in ((c.k_place, 2), (c.v_place, 8)):
                    for d in range(0, D, 32):
                        at = place(int(tok), d)[2]
                        raw[page, :, [at, at + 1, at + off, at + off + 1]] = tail
    b.cache.copy_(torch.from_numpy(raw))
    return c


def tokens(b, c, i, head):
    """Keys and values of a sequence's tokens in float64."""
    n = -(-b.seqs[i][1] // b.P)
    kv = [c.values(b.table[i, j], head) for j in range(n)]
    return [np.concatenate([x[z] for x in kv])[:b.seqs[i][1]] if n else np.zeros((0, b.D)) for z in range(2)]


def check(b, c, q32, got, H, kind, scale, window, softcap, fill=7.0):
    r = H // b.KV
    seen_rows = np.zeros(b.rows, bool)
    for i, (n, ln) in enumerate(b.seqs):
        t0 = int(b.starts[i])
        pos = np.arange(ln - n, ln)
        seen_rows[t0:t0 + n] = True
        for h in range(b.KV):
            k, v = tokens(b, c, i, h)
            for head in range(h * r, h * r + r):
                want, A, V, X, cnt = attention(q32[t0:t0 + n, head].astype(np.float64), k, v, pos, scale, window, softcap)
                S = ((1.01 * U + 2 * b.D * E) * X + 2.0 ** -25 * np.sqrt(b.D) * 4 * X + 16 * E * X + 8 * E * softcap)[:, None]
                tol = A * (2.05 * S + 2.02 * U + 2 * (cnt[:, None] + 64) * E) + 2.0 ** -25 * V
                tol = tol + 1.001 * HALF[kind] * (np.abs(want) + tol) + SMALLEST[kind]
                off = np.abs(got[t0:t0 + n, head] - want)
                assert (off <= tol).all(), (i, head, float((off / tol).max()), np.argwhere(~(off <= tol))[:4])
                assert (got[t0:t0 + n, head][cnt == 0] == 0).all()
    assert (got[~seen_rows] == fill).all()


def work_of(b, H, lane_fill=0xFF):
    return torch.full((xl.attention_work_bytes(b.kv, H),), lane_fill, dtype=torch.uint8, device="cuda")


CASES = [
    # sequences (rows, length), page, kv heads, q heads, D, kind, window, softcap, behind, before, pad
    ([(1, 1)], 16, 1, 1, 64, "f16", 0, 0.0, 0, 0, 0),
    ([(1, 200)], 64, 8, 32, 128, "bf16", 0, 0.0, 0, 0, 0),
    ([(1, 31), (1, 32), (1, 33), (1, 16), (1, 17)], 16, 2, 2, 128, "bf16", 0, 0.0, 3, 1, 8),
    ([(1, 3000)], 48, 1, 16, 128, "f16", 0, 0.0, 0, 0, 0),
    ([(1, 2000), (1, 5)], 16, 1, 3, 256, "bf16", 0, 20.0, 0, 0, 4),
    ([(1, 700), (0, 40), (1, 1)], 256, 2, 10, 64, "f16", 100, 0.0, 0, 0, 0),
    ([(4, 100), (5, 5), (3, 61)], 32, 2, 8, 128, "bf16", 0, 0.0, 0, 0, 0),
    ([(5, 333), (2, 40)], 16, 4, 12, 256, "f16", 64, 50.0, 1, 0, 2),
    ([(12, 90)], 16, 1, 16, 64, "bf16", 7, 0.0, 0, 0, 0),
    ([(2, 70)], 64, 1, 64, 128, "f16", 0, 0.0, 0, 0, 0),
    ([(33, 33)], 16, 2, 2, 128, "f16", 0, 0.0, 0, 0, 0),
    ([(129, 400), (1, 20), (64, 64)], 48, 3, 6, 64, "bf16", 0, 0.0, 2, 0, 3),
    ([(200, 333)], 64, 1, 4, 128, "bf16", 50, 0.0, 0, 0, 0),
    ([(150, 1500)], 128, 2, 4, 128, "f16", 0, 30.0, 0, 0, 0),
    ([(70, 300), (90, 91)], 16, 1, 5, 256, "bf16", 0, 0.0, 0, 0, 1),
    ([(300, 300)], 1024, 1, 1, 256, "f16", 33, 0.0, 0, 0, 0),
    ([(9, 4), (40, 20), (3, 0), (2, 30)], 16, 2, 4, 64, "f16", 0, 0.0, 0, 0, 0),      # rows before the first token
    ([(9, 4), (3, 1)], 16, 1, 2, 128, "bf16", 1, 0.0, 0, 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("tail", [None, 0x7e, 0x7b, 0xfc], ids=["", "nan-tail", "large-tail", "minus-nan-tail"])
def test_attention(lane, case, tail):  # noqa: F811
    seqs, P, KV, H, D, kind, window, softcap, behind, before, pad = case
    step(f"attention {case} {tail}")
    b = Batch(seqs, P, KV, D, behind, before, stride_pad=16 * (pad % 3), seed=D + H)
    c = filled(b, D, tail)
    q, q32 = rand_rows(b.rows, H, D, kind, 5, pad, 0.5)
    out = torch.full((b.rows, H * D + pad), 7.0, dtype=TYPES[kind], device="cuda")[:, :H * D].unflatten(1, (H, D))
    work = work_of(b, H)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, window=window, softcap=softcap, work=work)
    lane.sync()
    check(b, c, q32, out.double().cpu().numpy(), H, kind, D ** -0.5, window, softcap)
    again = torch.full_like(out, 7.0)
    lane.attention_async(b.kv, q, again, window=window, softcap=softcap, work=work)
    lane.sync()
    assert torch.equal(out, again)


@pytest.mark.parametrize("rows,length,H", [(1, 300, 4), (3, 300, 8), (80, 300, 2)])
def test_peaked_and_large(lane, rows, length, H):  # noqa: F811
    """One token that takes all the weight, q of a size that float16 does not hold, and a scale given."""
    step(f"attention, peaked {rows}")
    b = Batch([(rows, length)], 16, 1, 128)
    c = filled(b, 3)
    q, q32 = rand_rows(rows, H, 128, "bf16", 5, 0, 0.5)
    big = 2.0 ** 60
    q *= big
    out = torch.full((rows, H, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    work = work_of(b, H)
    torch.cuda.synchronize()
    for scale in (1.0 / big, 0.05 / big, -1.0 / big, 0.0):
        lane.attention_async(b.kv, q, out, scale=scale, work=work)
        lane.sync()
        check(b, c, q32 * np.float32(big), out.double().cpu().numpy(), H, "bf16", scale, 0, 0.0)


@pytest.mark.parametrize("rows,H", [(1, 4), (6, 2), (70, 2), (40, 8)])
def test_not_finite(lane, rows, H):  # noqa: F811
    """A token held as NaN makes the rows that see it NaN and no others, q's own NaN or infinity its row and head."""
    step(f"attention, not finite {rows}")
    ln = 150
    for is_v in (False, True):
        b = Batch([(rows, ln), (1, 40)], 16, 2, 64)
        c = filled(b, 4)
        bad = (ln - rows // 2 - 1, 20)   # the tokens: the row in the middle's, and one that a window hides
        for tok in bad:
            for d in (0, 32):
                at = (c.v_place if is_v else c.k_place)(tok % 16, d)[2]
                for o in (0, 8 if is_v else 2):
                    c.raw[b.table[0, tok // 16], 1, at + o:at + o + 2] = [0, 0x7e]
        b.cache.copy_(torch.from_numpy(c.raw))
        q, q32 = rand_rows(b.rows, H, 64, "f16", 5)
        out = torch.full((b.rows, H, 64), 7.0, dtype=torch.float16, device="cuda")
        work = work_of(b, H)
        torch.cuda.synchronize()
        for window in (0, 50):
            lane.attention_async(b.kv, q, out, window=window, work=work)
            lane.sync()
            got = out.float().cpu().numpy()
            want = np.zeros((b.rows, H), bool)
            for t, i, p in b.places():
                if i == 0 and any(tok <= p and (not window or tok > p - window) for tok in bad):
                    want[t, H // 2:] = True
            assert np.array_equal(np.isnan(got).all(2), want) and np.array_equal(np.isnan(got).any(2), want)
            # what is finite is right: with the NaN token's values taken as 0, rows that do not see it are the definition's
            for h in range(H):
                k, v = tokens(b, c, 0, h // (H // 2))
                k, v = np.nan_to_num(k), np.nan_to_num(v)
                ref = attention(q32[:rows, h].astype(np.float64), k, v, np.arange(ln - rows, ln), 0.125, window, 0.0)[0]
                ok = ~want[:rows, h]
                assert np.allclose(got[:rows, h][ok], ref[ok], atol=0.02)
    b = Batch([(rows, ln)], 16, 2, 64)
    filled(b, 4)
    q, q32 = rand_rows(rows, H, 64, "f16", 5)
    q[rows - 1, 1, 7] = float("inf")
    q[0, 0, 63] = float("nan")
    out = torch.full((rows, H, 64), 7.0, dtype=torch.float16, device="cuda")
    work = work_of(b, H)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, work=work)
    lane.sync()
    got = torch.isnan(out).all(2).cpu().numpy()
    want = np.zeros((rows, H), bool)
    want[rows - 1, 1] = want[0, 0] = True
    assert np.array_equal(got, want) and np.array_equal(torch.isnan(out).any(2).cpu().numpy(), want)


def test_shared_pages(lane):  # noqa: F811
    """Sequences with a common prefix in the same pages."""
    step("attention, shared pages")
    b = Batch([(1, 40), (2, 50), (30, 60)], 16, 2, 64)
    b.table[1, :2] = b.table[2, :2] = b.table[0, :2]
    b.d_table.copy_(torch.from_numpy(b.table))
    c = filled(b, 9)
    q, q32 = rand_rows(b.rows, 4, 64, "f16", 5)
    out = torch.full((b.rows, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    work = work_of(b, 4)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, work=work)
    lane.sync()
    check(b, c, q32, out.double().cpu().numpy(), 4, "f16", 0.125, 0, 0.0)


@pytest.mark.parametrize("rows", [3, 90])
def test_wide_windows(lane, rows):  # noqa: F811
    """Windows as long as a number can be, with rows before the first token."""
    step(f"attention, wide windows {rows}")
    b = Batch([(rows, rows - 2), (rows, 200)], 16, 1, 64)
    c = filled(b, 2)
    q, q32 = rand_rows(b.rows, 2, 64, "f16", 5, 0, 0.5)
    work = work_of(b, 2)
    for window in (0, 2 ** 31 - 1, 2 ** 26, 200):
        out = torch.full((b.rows, 2, 64), 7.0, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        lane.attention_async(b.kv, q, out, window=window, work=work)
        lane.sync()
        check(b, c, q32, out.double().cpu().numpy(), 2, "f16", 0.125, window, 0.0)


@pytest.mark.parametrize("rows,length,D,H,kind", [(1, 9000, 64, 4, "f16"), (1, 12000, 128, 8, "bf16"), (2, 9000, 256, 2, "bf16"),
                                                  (1, 40000, 64, 2, "bf16"), (70, 6000, 64, 1, "f16"), (70, 5000, 128, 1, "bf16"),
                                                  (200, 4500, 256, 1, "f16")])
def test_many_splits(lane, rows, length, D, H, kind):  # noqa: F811
    """Tokens in more parts than one thread joins, next to a sequence that leaves most parts without tokens."""
    step(f"attention, many splits {rows} {length} {D}")
    b = Batch([(rows, length), (1, 2)], 64, 1, D)
    c = filled(b, 7)
    q, q32 = rand_rows(b.rows, H, D, kind, 5, 0, 0.5)
    out = torch.full((b.rows, H, D), 7.0, dtype=TYPES[kind], device="cuda")
    work = work_of(b, H)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, work=work)
    lane.sync()
    check(b, c, q32, out.double().cpu().numpy(), H, kind, D ** -0.5, 0, 0.0)


@pytest.mark.parametrize("KV,H,rows,D", [(1, 1024, 1, 64), (1, 63, 1, 128), (1, 65, 1, 128), (256, 256, 1, 64), (64, 1024, 2, 64),
                                         (1, 192, 1, 256), (1, 97, 2, 256), (3, 1023, 1, 64)])
def test_head_counts(lane, KV, H, rows, D):  # noqa: F811
    """Groups around where the rows of one token are many, and the most heads of each kind."""
    step(f"attention, heads {KV} {H} {rows} {D}")
    b = Batch([(rows, 70), (rows, 9)], 1008, KV, D)
    c = filled(b, 7, 0x7e)
    q, q32 = rand_rows(b.rows, H, D, "f16", 5, 0, 0.5)
    out = torch.full((b.rows, H, D), 7.0, dtype=torch.float16, device="cuda")
    work = work_of(b, H)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, work=work)
    lane.sync()
    check(b, c, q32, out.double().cpu().numpy(), H, "f16", D ** -0.5, 0, 0.0)


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("softcap", [1e-20, 1e-3, 16384.0])
def test_softcap_ends(lane, rows, softcap):  # noqa: F811
    """Caps at the ends of what a call takes, with scores far above the small ones and far below the large one."""
    step(f"attention, softcap {rows} {softcap}")
    b = Batch([(rows, 150)], 16, 1, 128)
    c = filled(b, 7)
    q, q32 = rand_rows(b.rows, 2, 128, "bf16", 5, 0, 0.5)
    out = torch.full((b.rows, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    work = work_of(b, 2)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, softcap=softcap, work=work)
    lane.sync()
    check(b, c, q32, out.double().cpu().numpy(), 2, "bf16", 128 ** -0.5, 0, float(np.float32(softcap)))


def test_window_refused(lane):  # noqa: F811
    step("attention, windows refused")
    b = Batch([(1, 5)], 16, 1, 64)
    q = torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    for window in (-1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(xl.XLError, match="window"):
            lane.attention_async(b.kv, q, torch.zeros_like(q), window=window)
