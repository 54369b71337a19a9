"""GPU: the calls around a block of an 8-bit model (scored router, block norm, row
quantizer, int8 product) against plain forms in 64 bits.

Tolerances, E = 2^-24 (half a step of float32): a sum of squares takes at most 32
sums in a thread, 6 in the wave and 16 over the waves, so 54 E, which is 27 E of
its root, and the mean, the epsilon, the root and the quotient add 4: 31 E for an
inverse norm. Products and sums after it add one E each. Rounding to a 16-bit
output adds half its step. The quantizer and the product without SwiGLU are exact:
whole numbers, and float operations that numpy does alike.
"""
from __future__ import annotations

import sys

import numpy as np
import pytest

import crosslane_amd as xl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

E = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}   # spacing of the subnormals


def step(msg):
    print(f"[gpu-step] {msg}", flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def lane():
    with xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32)) as ln:
        yield ln


def up(a, pad=0, kind="f32", fill=float("nan")):
    """A matrix on the GPU as `kind`, in a buffer with `pad` more columns full of `fill`."""
    a = torch.from_numpy(np.ascontiguousarray(a)).to(TYPES[kind])
    buf = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=a.dtype)
    buf[:, : a.shape[1]] = a
    return buf.cuda()[:, : a.shape[1]]


def up8(a, pad=0, fill=77):
    """An int8 matrix with 16-byte aligned rows; the bytes behind a row's end are `fill`."""
    n, k = a.shape
    buf = np.full((n, (k + 15) // 16 * 16 + pad), fill, np.int8)
    buf[:, :k] = a
    return torch.from_numpy(buf).cuda()[:, :k]


def held(a, kind):
    """`a` as `kind` holds it, in float64."""
    return torch.from_numpy(np.ascontiguousarray(a)).to(TYPES[kind]).double().numpy()


# ---- router ------------------------------------------------------------------
def route64(lg, bias, score, groups, top, keys, k, renorm, scale):
    """The definition, one token at a time, sorting (key, -index) pairs."""
    T, n = lg.shape
    ids, w = np.zeros((T, k), np.int32), np.zeros((T, k))
    size = n // groups
    for t in range(T):
        on = np.isfinite(lg[t])
        s = np.zeros(n)
        if score == "sigmoid":
            s[on] = 1 / (1 + np.exp(-lg[t][on]))
        elif on.any():
            e = np.exp(lg[t][on] - lg[t][on].max())
            s[on] = e / e.sum()
        key = np.where(on, s + (0 if bias is None else bias), -1e300)
        rows = list(range(n))
        if groups > 1:
            value = [sum(sorted(key[g * size:(g + 1) * size])[::-1][:keys]) for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top]
            rows = [e for e in rows if e // size in kept]
        best = sorted(rows, key=lambda e: (-key[e], e))[:k]
        ids[t] = best
        w[t] = s[best]
        if renorm:
            w[t] /= w[t].sum() + 1e-20
    return ids, w * scale


ROUTES = [
    # T, n, k, score, groups, top, keys, renorm, scale, biased, kind, masked share, pad
    (1, 256, 8, "sigmoid", 8, 4, 2, True, 2.5, True, "f32", 0.0, 0),
    (5, 384, 6, "softmax", 1, 1, 1, True, 1.0, False, "bf16", 0.0, 0),
    (3, 1, 1, "softmax", 1, 1, 1, False, 1.0, False, "f32", 0.0, 3),
    (2, 16, 16, "sigmoid", 1, 1, 1, True, 0.0, True, "f16", 0.3, 1),
    (7, 64, 4, "softmax", 64, 5, 1, False, 16.0, True, "f32", 0.2, 0),
    (6, 65, 3, "sigmoid", 5, 2, 2, True, 1.0, False, "f32", 0.2, 7),
    (257, 100, 10, "softmax", 4, 1, 1, True, 1.0, True, "f32", 0.5, 0),
    (9, 1024, 16, "softmax", 16, 3, 2, True, 2.5, True, "f16", 0.1, 0),
    (4, 1024, 2, "sigmoid", 512, 1, 2, False, 1.0, False, "bf16", 0.9, 0),
    (33, 511, 8, "sigmoid", 7, 6, 2, True, 1.0, True, "f32", 0.05, 2),
    (64, 160, 6, "softmax", 8, 3, 1, False, 16.0, False, "bf16", 0.0, 0),
    (2, 130, 5, "softmax", 65, 65, 2, True, 1.0, False, "f32", 0.99, 0),
]


@pytest.mark.parametrize("case", ROUTES, ids=lambda c: "-".join(map(str, c)))
def test_route_scored(lane, case):
    T, n, k, score, groups, top, keys, renorm, scale, biased, kind, masked, pad = case
    step(f"route_scored {case}")
    rng = np.random.default_rng(T * 7 + n)
    lg = held((2.0 * rng.standard_normal((T, n))).astype(np.float32), kind)
    lg[rng.random((T, n)) < masked] = -np.inf
    bias = (0.2 * rng.standard_normal(n)).astype(np.float32) if biased else None
    want_ids, want_w = route64(lg, bias, score, groups, top, keys, k, renorm, scale)
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), float("nan"), device="cuda")
    d = up(lg.astype(np.float32), pad, kind, 0.5)
    b = None if bias is None else torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()
    lane.route_scored_async(d, k, ids, w, score=score, bias=b, groups=groups, top_groups=top, group_keys=keys, renorm=renorm,
                            scale=scale)
    lane.sync()
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # one rounding to float32; the doubles behind it are off by parts of 1e-15
    np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=1.001 * E, atol=1e-45)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_scored_ties_masks_and_far_logits(lane, score, groups):
    step(f"route_scored ties {score} {groups}")
    n, k = 32, 6
    lg = np.zeros((7, n), np.float32)
    lg[1] = -np.inf                               # a row whose mask leaves nothing
    lg[2] = -np.inf
    lg[2, [30, 3]] = [1.0, -2.0]                  # fewer than k are left
    lg[3, ::3] = 1.0                              # ties between equal logits
    lg[4] = np.linspace(-300, 30, n)              # scores down to underflow
    lg[5, 9] = np.finfo(np.float32).min           # lowest value: a score of 0, not a mask
    lg[6] = np.finfo(np.float32).min
    want_ids, want_w = route64(lg.astype(np.float64), None, score, groups, min(groups, 2), 2, k, True, 1.0)
    ids = torch.zeros((7, k), dtype=torch.int32, device="cuda")
    w = torch.zeros((7, k), device="cuda")
    d = up(lg)
    torch.cuda.synchronize()
    lane.route_scored_async(d, k, ids, w, score=score, groups=groups, top_groups=min(groups, 2), group_keys=2)
    lane.sync()
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=1.001 * E, atol=2.0 ** -149)
    assert np.array_equal(ids.cpu().numpy()[1], np.arange(k)) and not w.cpu().numpy()[1].any()


# ---- block norm ----------------------------------------------------------------
def norm64(y, res, gate, post, pre, alpha, eps):
    """r, x and bounds of what float32 may be off by at each."""
    rel_a = 0.0
    a = mag = None
    if y is not None:
        a = y.copy()
        if post is not None:
            a = a / np.sqrt((a * a).mean(1, keepdims=True) + eps) * post
            rel_a += 33 * E
        if gate is not None:
            a = a * gate
            rel_a += E
    r = np.zeros_like(y if res is None else res)
    mag = np.zeros_like(r)
    if res is not None:
        r, mag = alpha * res, np.abs(alpha * res)
    off = np.zeros_like(r)
    if a is not None:
        r, mag = r + a, mag + np.abs(a)
        off = rel_a * np.abs(a)
    off = off + E * np.abs(r) + E * mag * (res is not None)
    if pre is None:
        return r, off, None, None
    rms = np.sqrt((r * r).mean(1, keepdims=True) + eps)
    x = r / rms * pre
    # the norm of r moves by no more than r's own error does
    moved = np.sqrt((off * off).mean(1, keepdims=True)) / rms
    return r, off, x, np.abs(x) * (33 * E + moved) + off / rms * np.abs(pre)


def near(got, want, off, kind):
    tol = 1.001 * off + HALF[kind] * (np.abs(want) + off) + SMALLEST[kind]
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


NORMS = [
    # T, D, type, res_type, post, gate, alpha, pre, pad
    (1, 1, "f32", "f32", True, "channel", 1.0, True, 0),
    (3, 7, "f16", "f32", False, "token", 0.5, True, 1),
    (2, 8, "bf16", "bf16", True, "none", 1.0, True, 0),
    (5, 63, "bf16", "f32", True, "token", -0.75, True, 3),
    (4, 512, "f32", "bf16", True, "channel", 1.0, True, 0),
    (4, 513, "f16", "f16", False, "channel", 2.25, True, 5),
    (3, 2304, "bf16", "bf16", True, "channel", 1.0, False, 0),
    (9, 4099, "f16", "f32", False, "token", 0.5, True, 5),
    (2, 5120, "f32", "f32", True, "channel", 1.0, True, 0),
    (2, 8192, "bf16", "f32", True, "channel", 1.0, True, 8),
    (2, 8200, "bf16", "f16", True, "token", 1.0, True, 0),
    (2, 16384, "f32", "f32", True, "channel", 1.0, True, 0),
    (2, 16391, "f16", "bf16", True, "channel", 1.0, True, 0),
    (1, 32768, "f32", "f32", True, "token", 1.0, True, 0),
    (700, 1000, "bf16", "bf16", True, "channel", 1.0, True, 0),
]


def norm_case(case, rng):
    T, D, kind, rk, post, gate, alpha, pre, pad = case
    n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    y, res = n(T, D), 3 * n(T, D)
    g = {"none": None, "channel": n(D), "token": n(T, D)}[gate]
    return y, res, g, (1 + 0.1 * n(D)) if post else None, (1 + 0.1 * n(D)) if pre else None


@pytest.mark.parametrize("case", NORMS, ids=lambda c: "-".join(map(str, c)))
def test_block_norm(lane, case):
    T, D, kind, rk, post, gate, alpha, pre, pad = case
    step(f"block_norm {case}")
    y, res, g, pw, nw = norm_case(case, np.random.default_rng(D + T))
    r, roff, x, xoff = norm64(held(y, kind), held(res, rk), None if g is None else held(g, kind),
                              None if pw is None else pw.astype(np.float64), None if nw is None else nw.astype(np.float64),
                              alpha, 1e-6)
    dy, dres = up(y, pad, kind), up(res, pad, rk)
    dg = None if g is None else torch.from_numpy(g).to(TYPES[kind]).cuda()
    vec = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    dpw, dnw = vec(pw), vec(nw)
    ro = torch.full((T, D + pad), 9.0, dtype=TYPES[rk], device="cuda")
    xo = torch.full((T, D + pad), 9.0, dtype=TYPES[kind], device="cuda")
    q = torch.full((T, (D + 15) // 16 * 16 + 16), 9, dtype=torch.int8, device="cuda")
    qs = torch.zeros(T, device="cuda")
    torch.cuda.synchronize()
    lane.block_norm_async(dres, y=dy, post_w=dpw, gate=dg, alpha=alpha, pre_w=dnw, eps=1e-6, res_out=ro[:, :D],
                          x=xo[:, :D] if pre else None, q=q[:, :D] if pre else None, q_scale=qs if pre else None)
    lane.sync()
    near(ro[:, :D].double().cpu().numpy(), r, roff, rk)
    assert (ro[:, D:] == 9).all() and (xo[:, D:] == 9).all()   # nothing behind the rows
    if not pre:
        return
    near(xo[:, :D].double().cpu().numpy(), x, xoff, kind)
    s = qs.double().cpu().numpy()
    big = np.abs(x).max(1)
    assert (np.abs(s * 127 - big) <= xoff.max(1) + 2 * E * big).all()
    got = q.cpu().numpy()
    assert not got[:, D:(D + 15) // 16 * 16].any() and (got[:, (D + 15) // 16 * 16:] == 9).all()
    # a quant is off by half a step at most, and x by its own error
    assert (np.abs(got[:, :D] * s[:, None] - x) <= 0.5001 * s[:, None] + xoff).all()


def test_block_norm_parts_and_in_place(lane):
    step("block_norm parts")
    T, D = 5, 777
    y, res, g, pw, nw = norm_case((T, D, "f32", "f32", True, "token", 1.0, True, 0), np.random.default_rng(3))
    dy, dres, dg, dpw, dnw = (torch.from_numpy(v).cuda() for v in (y, res, g, pw, nw))
    d64 = [v.astype(np.float64) for v in (y, res, g, pw, nw)]
    ro, xo = torch.zeros((T, D), device="cuda"), torch.zeros((T, D), device="cuda")
    torch.cuda.synchronize()
    lane.block_norm_async(dres, pre_w=dnw, x=xo)                       # the norm before a block alone
    lane.block_norm_async(None, y=dy, post_w=dpw, gate=dg, res_out=ro)  # a block's own norm and gate, no residual
    lane.sync()
    _, _, x, xoff = norm64(None, d64[1], None, None, d64[4], 1.0, 1e-6)
    near(xo.double().cpu().numpy(), x, xoff, "f32")
    r, roff, _, _ = norm64(d64[0], None, d64[2], d64[3], None, 1.0, 1e-6)
    near(ro.double().cpu().numpy(), r, roff, "f32")
    r, roff, x, xoff = norm64(*d64, 0.5, 1e-6)
    lane.block_norm_async(dres, y=dy, post_w=dpw, gate=dg, alpha=0.5, pre_w=dnw, res_out=dres, x=dy)   # both in place
    lane.sync()
    near(dres.double().cpu().numpy(), r, roff, "f32")
    near(dy.double().cpu().numpy(), x, xoff, "f32")


def test_block_norm_zero_rows(lane):
    step("block_norm zeros")
    z = torch.zeros((3, 100), device="cuda")
    one = torch.ones(100, device="cuda")
    x, q, s = torch.ones((3, 100), device="cuda"), torch.ones((3, 112), dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
    torch.cuda.synchronize()
    lane.block_norm_async(z, y=z.clone(), post_w=one, pre_w=one, x=x, q=q[:, :100], q_scale=s)
    lane.sync()
    assert not x.any() and not q.any() and not s.any()


# ---- row quantizer ---------------------------------------------------------------
def quant32(x):
    """The quantizer in numpy's float32, whose division and rounding are IEEE's."""
    x = x.astype(np.float32)
    s = (np.abs(x).max(1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.clip(np.rint(x / s[:, None]), -127, 127)
    return np.where(s[:, None] > 0, q, 0).astype(np.int8), s


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("T,K,pad", [(1, 1, 0), (3, 15, 1), (2, 16, 0), (5, 511, 3), (4, 2301, 0), (2, 8192, 8), (3, 8193, 0),
                                     (2, 32768, 0), (2, 32771, 5), (1, 65536, 0), (600, 512, 0)])
def test_quantize_rows(lane, T, K, pad, kind):
    step(f"quantize_rows {T} {K} {pad} {kind}")
    rng = np.random.default_rng(K)
    x = rng.standard_normal((T, K)).astype(np.float32) * np.exp(2 * rng.standard_normal((T, 1))).astype(np.float32)
    x[-1] = 0 if T > 2 else x[-1]
    want_q, want_s = quant32(held(x, kind))
    q = torch.full((T, (K + 15) // 16 * 16 + 16), 9, dtype=torch.int8, device="cuda")
    s = torch.full((T,), -1.0, device="cuda")
    d = up(x, pad, kind)
    torch.cuda.synchronize()
    lane.quantize_rows_async(d, q[:, :K], s)
    lane.sync()
    got = q.cpu().numpy()
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(got[:, :K], want_q)
    assert not got[:, K:(K + 15) // 16 * 16].any() and (got[:, (K + 15) // 16 * 16:] == 9).all()


def test_quantize_rows_ties_and_tiny(lane):
    step("quantize_rows ties")
    x = np.zeros((4, 32), np.float32)
    x[0, :9] = [127, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5]   # halves go to the even quant
    x[1, :3] = [1e-42, -5e-43, 2e-44]                                   # a subnormal scale
    x[2, 0] = 1e-45                                                      # a scale that underflows to 0
    x[3, :2] = [3.4e38, -1.7e38]
    want_q, want_s = quant32(x)
    q, s = torch.ones((4, 32), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    d = up(x)
    torch.cuda.synchronize()
    lane.quantize_rows_async(d, q, s)
    lane.sync()
    assert np.array_equal(s.cpu().numpy(), want_s) and np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("what", ["rows", "norm", "route", "linear"])
def test_values_that_are_no_numbers_are_reported(what, value):
    if what == "route" and value == float("-inf"):
        value = float("nan")   # -inf masks an expert
    step(f"{what} {value}")
    with xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32)) as ln:
        x = torch.ones((3, 64), device="cuda")
        x[1, 40] = value
        q, s = torch.ones((3, 64), dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
        one = torch.ones(64, device="cuda")
        ids, w = torch.zeros((3, 4), dtype=torch.int32, device="cuda"), torch.zeros((3, 4), device="cuda")
        out = torch.zeros((3, 8), device="cuda")
        w8, ws = torch.ones((8, 64), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
        work = torch.empty(xl.linear_i8_work_bytes(3, 64, 8), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        if what == "rows":
            ln.quantize_rows_async(x, q, s)
        elif what == "norm":
            ln.block_norm_async(x, pre_w=one, q=q, q_scale=s)
        elif what == "route":
            ln.route_scored_async(x, 4, ids, w)
        else:
            ln.linear_i8_async(x, w8, ws, out, work=work)
        with pytest.raises(xl.XLError, match="non-finite"):
            ln.sync()
        torch.cuda.synchronize()
        if what in ("rows", "norm"):
            assert torch.isnan(s).tolist() == [False, True, False] and not q[1].any() and q[0].any()
        if what == "linear":   # the row's products are no finite wrong numbers
            assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()
        if what == "route":
            assert ((ids >= 0) & (ids < 64)).all()


# ---- int8 product -------------------------------------------------------------------
def product32(q, qs, w, ws):
    """Exact sums, then the call's float32 operations."""
    acc = q.astype(np.int64) @ w.astype(np.int64).T if q.shape[0] * q.shape[1] * w.shape[0] < 1 << 24 else \
        (torch.from_numpy(q).double() @ torch.from_numpy(w).double().t()).numpy().astype(np.int64)
    return acc.astype(np.float32) * qs[:, None] * ws[None, :]


def swiglu64(g, u, lim):
    g, u = g.astype(np.float64), u.astype(np.float64)
    if lim > 0:
        g, u = np.minimum(g, lim), np.clip(u, -lim, lim)
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


def linear_case(lane, T, K, N, gated, lim, x_kind, out_kind, xpad=0, wpad=0, opad=0, extreme=False, seed=0, stream=None):
    rng = np.random.default_rng([T, K, N, seed])
    mats = []
    for _ in range(2 if gated else 1):
        w = np.full((N, K), -128, np.int8) if extreme else rng.integers(-127, 128, (N, K)).astype(np.int8)
        mats.append((w, (rng.random(N) * 0.02 / np.sqrt(K) + 1e-4).astype(np.float32)))
    if x_kind == "i8":
        q = np.full((T, K), -128, np.int8) if extreme else rng.integers(-128, 128, (T, K)).astype(np.int8)
        qs = (rng.random(T) * 0.02 + 0.01).astype(np.float32)
        x, xs = up8(q, xpad), torch.from_numpy(qs).cuda()
    else:
        f = rng.standard_normal((T, K)).astype(np.float32)
        q, qs = quant32(held(f, x_kind))
        x, xs = up(f, xpad, x_kind), None
    dm = [(up8(w, wpad), torch.from_numpy(ws).cuda()) for w, ws in mats]
    out = torch.full((T, N + opad), 9.0, dtype=TYPES[out_kind], device="cuda")
    work = torch.full((xl.linear_i8_work_bytes(T, K, N, gated),), 0x5A, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    (w, ws), (u, us) = dm[0], dm[1] if gated else (None, None)
    lane.linear_i8_async(x, w, ws, out[:, :N], x_scale=xs, up=u, up_scale=us, limit=lim, work=work, stream=stream)
    lane.sync(stream)
    g = product32(q, qs, *mats[0])
    got = out[:, :N].double().cpu().numpy()
    assert (out[:, N:] == 9).all()
    if not gated:   # the same float operations: equal, but for the one rounding of `out`
        assert np.array_equal(got, held(g, out_kind))
        return
    want = swiglu64(g, product32(q, qs, *mats[1]), lim)
    # expf within two steps of float32, then a sum, a quotient and a product
    near(got, want, 8 * E * np.abs(want) + 2.0 ** -126, out_kind)


LINEARS = [
    # T, K, N, gated, limit, x, out
    (1, 1, 1, False, 0.0, "f32", "f32"), (1, 5120, 400, False, 0.0, "f32", "f32"), (1, 4096, 333, True, 0.0, "bf16", "bf16"),
    (2, 15, 17, True, 7.0, "i8", "f32"), (3, 16, 16, False, 0.0, "i8", "f16"), (4, 17, 15, False, 0.0, "f16", "f32"),
    (5, 300, 65, True, 0.0, "f32", "bf16"), (8, 2304, 129, False, 0.0, "i8", "bf16"), (9, 65, 257, False, 0.0, "bf16", "f32"),
    (15, 129, 63, True, 10.0, "i8", "f16"), (16, 1024, 256, False, 0.0, "f32", "f32"), (17, 1023, 127, False, 0.0, "f16", "f16"),
    (24, 5120, 96, True, 10.0, "bf16", "bf16"), (32, 64, 1111, False, 0.0, "i8", "f32"), (33, 2301, 90, True, 0.0, "i8", "f32"),
    (48, 127, 255, False, 0.0, "bf16", "bf16"), (63, 255, 64, True, 1.0, "f32", "f32"), (64, 4097, 130, False, 0.0, "i8", "f32"),
    (65, 128, 520, False, 0.0, "f32", "f16"), (96, 640, 320, True, 0.0, "i8", "bf16"), (127, 63, 129, False, 0.0, "i8", "f32"),
    (128, 2304, 512, False, 0.0, "bf16", "bf16"), (130, 31, 33, True, 7.0, "f32", "f32"), (192, 1536, 257, True, 0.0, "i8", "f32"),
    (256, 256, 256, False, 0.0, "i8", "f32"), (257, 1111, 300, False, 0.0, "f32", "f32"), (300, 512, 700, True, 0.0, "bf16", "f16"),
    (333, 2301, 1111, False, 0.0, "f16", "f16"), (512, 384, 513, False, 0.0, "i8", "bf16"), (513, 97, 640, True, 0.0, "i8", "f32"),
    (1024, 200, 1500, False, 0.0, "bf16", "f32"), (1100, 1000, 260, True, 10.0, "f32", "bf16"), (2050, 130, 515, False, 0.0, "i8", "f32"),
    (40, 8192, 40, False, 0.0, "i8", "f32"), (700, 4096, 24, False, 0.0, "i8", "f32"), (2, 64, 5000, True, 0.0, "i8", "f32"),
]


@pytest.mark.parametrize("case", LINEARS, ids=lambda c: "-".join(map(str, c)))
def test_linear_i8(lane, case):
    step(f"linear_i8 {case}")
    linear_case(lane, *case)


@pytest.mark.parametrize("case", [(1, 100, 37, False, 0.0, "i8", "f32"), (20, 100, 70, True, 0.0, "i8", "f16"),
                                  (130, 333, 140, False, 0.0, "f32", "bf16"), (300, 515, 300, True, 0.0, "i8", "f32")],
                         ids=lambda c: "-".join(map(str, c)))
def test_linear_i8_strides(lane, case):
    step(f"linear_i8 strides {case}")
    linear_case(lane, *case, xpad=16 if case[5] == "i8" else 5, wpad=48, opad=3)


@pytest.mark.parametrize("T", [1, 17, 100, 260])
def test_linear_i8_largest_sums(lane, T):
    step(f"linear_i8 extreme {T}")   # 65536 products of 2^14
    linear_case(lane, T, 65536, 20, False, 0.0, "i8", "f32", extreme=True)


def test_linear_i8_far_rows(lane):
    """Rows whose offsets pass 32 bits."""
    step("linear_i8 far rows")
    T, K, N, stride = 2100, 64, 80, 1 << 20
    rng = np.random.default_rng(5)
    x = torch.zeros(T * stride, dtype=torch.int8, device="cuda").view(T, stride)[:, :K]
    w = torch.zeros(2 * 2100 * stride, dtype=torch.int8, device="cuda").view(4200, stride)[-N:, :K]
    q, wq = rng.integers(-127, 128, (T, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    x.copy_(torch.from_numpy(q)), w.copy_(torch.from_numpy(wq))
    xs, ws = torch.full((T,), 0.01, device="cuda"), torch.full((N,), 0.02, device="cuda")
    out = torch.zeros((T, N), device="cuda")
    work = torch.empty(xl.linear_i8_work_bytes(T, K, N), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for lo, hi in ((0, T), (T - 3, T), (T - 40, T)):
        out.zero_()
        torch.cuda.synchronize()
        lane.linear_i8_async(x[lo:hi], w, ws, out[lo:hi], x_scale=xs[lo:hi], work=work)
        lane.sync()
        want = product32(q[lo:hi], np.full(hi - lo, 0.01, np.float32), wq, np.full(N, 0.02, np.float32))
        assert np.array_equal(out[lo:hi].cpu().numpy(), want)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_linear_i8_rows_do_not_depend_on_each_other(lane, T):
    """A call's repetition gives the same bits."""
    step(f"linear_i8 again {T}")
    rng = np.random.default_rng(T)
    x = torch.from_numpy(rng.standard_normal((T, 700)).astype(np.float32)).cuda()
    w, ws = up8(rng.integers(-127, 128, (300, 700)).astype(np.int8)), torch.ones(300, device="cuda")
    work = torch.empty(xl.linear_i8_work_bytes(T, 700, 300), dtype=torch.uint8, device="cuda")
    a, b = torch.zeros((T, 300), device="cuda"), torch.ones((T, 300), device="cuda")
    torch.cuda.synchronize()
    lane.linear_i8_async(x, w, ws, a, work=work)
    lane.linear_i8_async(x, w, ws, b, work=work)
    lane.sync()
    assert torch.equal(a, b)


# ---- streams and graphs ----------------------------------------------------------------
def test_streams(lane):
    """Calls on other streams than the context's, in turn."""
    step("block ops on streams")
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for i, s in enumerate((sa, sb, sa)):
        linear_case(lane, 3 + 20 * i, 500, 100, bool(i & 1), 0.0, "f32", "f32", stream=s.cuda_stream, seed=i)


@pytest.mark.parametrize("T", [1, 30, 400])
def test_block_in_a_graph(lane, T):
    """All four calls captured together; every replay on new inputs equals the eager calls."""
    step(f"graph {T}")
    D, N, E_, k = 640, 300, 64, 6
    s = torch.cuda.Stream()
    rng = np.random.default_rng(T)
    f = lambda *sh: torch.from_numpy(rng.standard_normal(sh).astype(np.float32)).cuda()  # noqa: E731
    y, res, logits, one = f(T, D), f(T, D), f(T, E_), torch.ones(D, device="cuda")
    w8 = [up8(rng.integers(-127, 128, (N, D)).astype(np.int8)) for _ in range(2)]
    ws = torch.full((N,), 1e-3, device="cuda")
    work = torch.empty(xl.linear_i8_work_bytes(T, D, N, True), dtype=torch.uint8, device="cuda")

    def buffers():
        return {"ro": torch.zeros((T, D), device="cuda"), "q": torch.zeros((T, D), dtype=torch.int8, device="cuda"),
                "qs": torch.zeros(T, device="cuda"), "h": torch.zeros((T, N), device="cuda"),
                "h2": torch.zeros((T, N), device="cuda"), "q2": torch.zeros((T, D), dtype=torch.int8, device="cuda"),
                "qs2": torch.zeros(T, device="cuda"), "ids": torch.zeros((T, k), dtype=torch.int32, device="cuda"),
                "w": torch.zeros((T, k), device="cuda")}

    def block(b):
        p = s.cuda_stream
        lane.block_norm_async(res, y=y, post_w=one, pre_w=one, res_out=b["ro"], q=b["q"], q_scale=b["qs"], stream=p)
        lane.route_scored_async(logits, k, b["ids"], b["w"], stream=p)
        lane.linear_i8_async(b["q"], w8[0], ws, b["h"], x_scale=b["qs"], up=w8[1], up_scale=ws, work=work, stream=p)
        lane.linear_i8_async(y, w8[0], ws, b["h2"], work=work, stream=p)
        lane.quantize_rows_async(y, b["q2"], b["qs2"], stream=p)

    eager, graphed = buffers(), buffers()
    torch.cuda.synchronize()
    block(eager)
    lane.sync(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        block(graphed)
    for _ in range(4):
        y.copy_(f(T, D)), res.copy_(f(T, D)), logits.copy_(f(T, E_))
        torch.cuda.synchronize()
        block(eager)
        lane.sync(s.cuda_stream)
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(eager[name], graphed[name]), name
