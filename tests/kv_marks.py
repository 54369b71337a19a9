"""Caches of the 4-bit format whose attention is known exactly, so that one lost, doubled or misweighted tile of tokens
shows: what test_gpu_attention_marks.py runs and test_kv_marks.py checks on the CPU.

counted  Queries are 0, so every weight is 1 before the division, and value rows hold one whole number of 1 to 15: token j's
         in dim j // 16 of D. Sums are whole numbers below 2^24, exact in float32, and weights and values are exact in
         float16. What is left are the quotient (1 / n and a product: 3 * 2^-24 of it) and the output's half step.

marked   Keys are 0 but for marked tokens, which have rows of a Hadamard matrix; a query is the sum of two of those rows, so
         that two tokens share the weight, whichever parts of the tokens they lie in. Products are exact (whole numbers).
         Scores of the two are 32 (of one drawn twice 64), of all others 0. With E = 2^-24 and U = 2^-11: a score times log2(e) is
         off by 4 E * 92.4, the exponential by 4 E, so weights by the factor exp(2 * 374 E); weights are rounded to float16 (U, and 2^-25
         of the largest one below its normal range), values are too (U); sums of n tokens add (n + 64) E twice:
             |out - want| <= A (800 E + 2.02 U + 2 (n + 64) E) + 2^-25 V + half a step of the output
         with A the sum of p |v| and V that of |v| over the tokens seen.
"""
from __future__ import annotations

import numpy as np

E, U = 2.0 ** -24, 2.0 ** -11
SCORE = 32.0


def slab(c, places, codes, scales):
    """One kv head's bytes of a page: codes of keys and values [P, D] and their (s, m) [P, G]."""
    out = np.zeros(c.raw.shape[2], np.uint8)
    for (at, shift, sc), code, (s, m), off in zip(places, codes, scales, (2, 8)):
        np.add.at(out, at, (code << shift).astype(np.uint8))
        for x, o in ((s, 0), (m, off)):
            b = np.ascontiguousarray(x.astype(np.float16)).view(np.uint8).reshape(*x.shape, 2)
            out[sc[:, ::32] + o], out[sc[:, ::32] + o + 1] = b[..., 0], b[..., 1]
    return out


def fill(c, table, lens, tokens_of):
    """The pages of each sequence, from tokens_of(sequence, head, positions) -> codes and scales for `slab`."""
    P, places = c.P, c.places()
    for i, ln in enumerate(lens):
        for j in range(-(-int(ln) // P)):
            for h in range(c.raw.shape[1]):
                c.raw[table[i, j], h] = slab(c, places, *tokens_of(i, h, np.arange(j * P, (j + 1) * P)))


def counted(D):
    def tokens_of(_seq, _head, at):
        n, one = at.size, np.ones((at.size, D // 32))
        v = np.zeros((n, D), np.int64)
        v[np.arange(n), at // 16 % D] = 1 + at % 15
        k = np.random.default_rng(int(at[0])).integers(0, 16, (n, D))
        return (k, v), ((one, -7 * one), (one, 0 * one))
    return tokens_of


def hadamard(D):
    h = np.ones((1, 1), np.int64)
    while h.shape[0] < D:
        h = np.block([[h, h], [h, -h]])
    return h


def marked(D, marks):
    """marks: positions, one for each row of the Hadamard matrix at most."""
    rows = hadamard(D)

    def tokens_of(seq, head, at):
        rng = np.random.default_rng(1000 * seq + 100 * head + int(at[0]))
        n, G = at.size, D // 32
        k, s, m = np.zeros((n, D), np.int64), np.zeros((n, G)), np.zeros((n, G))
        for i, t in enumerate(marks):
            for j in np.nonzero(at == t)[0]:
                k[j], s[j], m[j] = (rows[i] + 1) // 2, 2.0, -1.0
        v = rng.integers(0, 16, (n, D))
        sv = 0.3 * np.exp(0.3 * rng.standard_normal((n, G)))
        return (k, v), ((s, m), (sv, -7.5 * sv + 0.3 * rng.standard_normal((n, G))))
    return tokens_of


def pairs(D, marks, positions, window, heads, rng):
    """For each row (at `positions`) and head two marked tokens that it sees, and its q: the sum of their rows. (None where
    it sees none: q is 0.) Also two that the window or the row's own position hides, added where there are any."""
    rows = hadamard(D)
    q = np.zeros((len(positions), heads, D), np.float32)
    for t, p in enumerate(positions):
        seen = [i for i, x in enumerate(marks) if x <= p and (not window or x > p - window)]
        hidden = [i for i, x in enumerate(marks) if i not in seen]
        near = sorted(hidden, key=lambda i: min(abs(marks[i] - p), abs(marks[i] - p + window) if window else 1 << 30))[:2]
        for h in range(heads):
            if seen:
                a, b = rng.choice(seen), rng.choice(seen)
                q[t, h] = rows[a] + rows[b] + sum(rows[i] for i in near)
    return q


def bound_counted(want, half, smallest):
    return (4 * E + 1.001 * half) * np.abs(want) + smallest


def bound_marked(want, A, V, count, half, smallest):
    tol = A * (800 * E + 2.02 * U + 2 * (count[:, None] + 64) * E) + 2.0 ** -25 * V
    return tol + 1.001 * half * (np.abs(want) + tol) + smallest
