"""The 4-bit cache in numpy, value by value from the layout that crosslane.h gives, and the
definitions of the calls over it: what test_gpu_kv*.py compares with."""
from __future__ import annotations

import numpy as np

F = np.float32
NAN16 = 0x7e00


def page_bytes(P, D):
    return P * D * 5 // 4


class Cache:
    """One kv head's slabs of a cache's bytes [n_pages, kv_heads, page_bytes]."""

    def __init__(self, raw, P, D):
        self.raw, self.P, self.D, self.G = raw, P, D, D // 32
        self.k_scales, self.v_codes, self.v_scales = P * D // 2, P * (D // 2 + D // 8), P * (D + D // 8)

    def k_place(self, tok, d):
        """Byte and shift of a key's code, byte of its group's scales."""
        g, c, e = d // 32, d % 32 // 8, d % 8
        nibble = e // 2 + 4 * (e % 2)
        return 4 * (tok * self.D // 8 + c * self.G + g) + nibble // 2, 4 * (nibble % 2), self.k_scales + 4 * (tok * self.G + g)

    def v_place(self, tok, d):
        quad, b, e = tok // 4, tok % 4 // 2, tok % 2
        half = (((quad * (self.D // 8) + d // 8) * 2 + b) * 2 + d % 8 // 4) * 2 + e
        return (self.v_codes + 2 * half + d % 4 // 2, 4 * (d % 2),
                self.v_scales + 2 * ((quad * self.G + d // 32) * 8 + tok % 4))

    def half(self, page, head, at):
        return self.raw[page, head, at:at + 2].copy().view(np.float16)[0]

    def put(self, page, head, tok, k, v):
        """Rows k and v (float32, D) of one token: groups quantized as the call defines it."""
        for row, is_v in ((k, False), (v, True)):
            s, m, code = quantized(row)
            for d in range(self.D):
                at, shift, sc = (self.v_place if is_v else self.k_place)(tok, d)
                b = int(self.raw[page, head, at])
                self.raw[page, head, at] = (b & ~(15 << shift) & 255) | (int(code[d]) << shift)
                g = d // 32
                self.raw[page, head, sc:sc + 2] = np.frombuffer(s[g:g + 1].tobytes(), np.uint8)
                off = 8 if is_v else 2
                self.raw[page, head, sc + off:sc + off + 2] = np.frombuffer(m[g:g + 1].tobytes(), np.uint8)

    def places(self):
        """Byte, shift and scale offsets of keys and values for all tokens of a page: arrays [P, D]."""
        tok, d = np.arange(self.P)[:, None], np.arange(self.D)[None, :]
        return self.k_place(tok, d), self.v_place(tok, d)

    def values(self, page, head):
        """Keys and values [P, D] in float64, and their scales [P, D]."""
        slab = self.raw[page, head]
        out = []
        for (at, shift, sc), off in zip(self.places(), (2, 8)):
            half = lambda o: (slab[o].astype(np.uint16) | slab[o + 1].astype(np.uint16) << 8).view(np.float16).astype(np.float64)  # noqa: E731
            out.append((slab[at] >> shift & 15) * half(sc) + half(sc + off))
        return out


def quantized(row):
    """Scales, smallest values (float16) and codes of a float32 row, in the call's float32 steps."""
    D = row.size
    if not np.isfinite(row).all():
        bad = np.full(D // 32, NAN16, np.uint16).view(np.float16)
        return bad, bad, np.zeros(D, np.int64)
    x = np.clip(row.astype(F), F(-32768), F(32768)).reshape(-1, 32)
    m = x.min(1).astype(np.float16)
    s = np.maximum((x.max(1) - m.astype(F)) * F(1 / 15), F(0)).astype(np.float16)
    with np.errstate(divide="ignore"):
        inv = np.where(s > 0, F(1) / s.astype(F), F(0)).astype(F)
    code = np.clip(np.rint((x - m.astype(F)[:, None]) * inv[:, None]), 0, 15)
    return s, m, code.astype(np.int64).reshape(-1)


def turned(x, freqs, places, sections, interleaved):
    """Rows x [T, heads, D] (float32) turned: places [axes][T]."""
    n = freqs.size
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = places[axis].T.astype(np.float64) * freqs.astype(np.float64)
    c, s = np.cos(angle).astype(F)[:, None, :], np.sin(angle).astype(F)[:, None, :]
    y = x.copy()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = p, q
    else:
        y[..., :n], y[..., n:2 * n] = p, q
    return y


def attention(q, k, v, pos, scale, window, softcap):
    """Rows q [n, D] at positions pos of one head in float64 over k, v [L, D]. Also what bounds a kernel's
    error (see test_gpu_attention.py): the sums of p |v|, the sum of |v| seen, the largest sum of |q k|, the tokens seen."""
    x = (q @ k.T) * scale
    if softcap:
        x = softcap * np.tanh(x / softcap)
    j = np.arange(k.shape[0])[None, :]
    seen = j <= pos[:, None]
    if window:
        seen &= j > pos[:, None] - window
    x = np.where(seen, x, -np.inf)
    top = x.max(1, keepdims=True, initial=-np.inf)
    p = np.exp(x - np.where(np.isinf(top), 0, top))
    p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
    sums = np.where(seen, (np.abs(q) @ np.abs(k).T) * abs(scale), 0).max(1, initial=0)
    return p @ v, p @ np.abs(v), seen @ np.abs(v), sums, seen.sum(1)
