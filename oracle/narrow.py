"""The operators in few bits (include/sm_base2.h: sm_plate8_*, sm_narrow_*) from their definitions, in Python's whole
numbers and numpy int64, a row at a time: the digits of a row, the product with an 8-bit plate, the cache of 4 or 8-bit
digits and the attention over it.  Nothing here follows the device's layouts, tiles or splits."""
from __future__ import annotations

import numpy as np

CHUNK = 256


def rsh(x, s: int):
    """x 2^-s rounded half up, x an int or an int64 array (Python's shifts: s may be any number)"""
    if isinstance(x, np.ndarray):
        return np.array([rsh(int(v), s) for v in x.ravel()], dtype=np.int64).reshape(x.shape)
    return (x + (1 << (s - 1))) >> s if s > 0 else x << -s


def wrap(x: int) -> int:
    """x modulo 2^64 as int64"""
    return (x + (1 << 63)) % (1 << 64) - (1 << 63)


def digits(x, bits: int):
    """a row's digits of `bits` bits and its level sh"""
    x = [int(v) for v in x]
    sh = max(max(abs(v) for v in x).bit_length() - (bits - 1), 0)
    top = 1 << (bits - 1)
    return np.array([min(max(rsh(v, sh), -top), top - 1) for v in x], dtype=np.int64), sh


def values(d, sh: int):
    return np.array([wrap(int(v) << sh) for v in d], dtype=np.int64)


def product(X, w, e, b):
    """rows of X through a plate of 8-bit digits"""
    out = np.zeros((len(X), w.shape[1]), dtype=np.int64)
    for r, x in enumerate(X):
        x8, sh = digits(x, 8)
        pile = x8 @ w.astype(np.int64)
        out[r] = [wrap(rsh(int(p), -(int(k) + sh)) + int(c)) for p, k, c in zip(pile, e, b)]
    return out


class Cache:
    """digits and levels of every (stream, head, position); zeros where nothing is written"""

    def __init__(self, streams, heads, dim, ctx, bits):
        self.bits, self.ctx, self.dim = bits, ctx, dim
        self.k, self.v = (np.zeros((streams, heads, ctx, dim), np.int64) for _ in range(2))
        self.kl, self.vl = (np.zeros((streams, heads, ctx), np.int64) for _ in range(2))

    def places(self, rows, start, count, span=None):
        """(stream, row, position) of the call's rows that are there"""
        for s in range(len(start)):
            for t in range(rows if count is None else min(max(int(count[s]), 0), rows)):
                if 0 <= int(start[s]) + t < (self.ctx if span is None else span):
                    yield s, t, int(start[s]) + t

    def write(self, k, v, start, count=None):
        """k, v: [streams][rows][heads][dim]"""
        for s, t, p in self.places(k.shape[1], start, count):
            for h in range(k.shape[2]):
                self.k[s, h, p], self.kl[s, h, p] = digits(k[s, t, h], self.bits)
                self.v[s, h, p], self.vl[s, h, p] = digits(v[s, t, h], self.bits)

    def read(self, rows, start, count, k, v):
        """into k and v"""
        for s, t, p in self.places(rows, start, count):
            for h in range(k.shape[2]):
                k[s, t, h] = values(self.k[s, h, p], int(self.kl[s, h, p]))
                v[s, t, h] = values(self.v[s, h, p], int(self.vl[s, h, p]))

    def attend(self, tab, q, start, count, span, scale, out):
        """into out; q, out: [streams][rows][query heads][dim]"""
        group = q.shape[2] // self.k.shape[1]
        for s, t, p in self.places(q.shape[1], start, count, span):
            for h in range(q.shape[2]):
                g = h // group
                out[s, t, h] = attend_row(tab, q[s, t, h], scale, *(a[s, g, :p + 1] for a in (self.k, self.kl, self.v, self.vl)))


def attend_row(tab, q, scale: int, k, kl, v, vl):
    """one row's attention over the positions of k, v (digits) and kl, vl (levels)"""
    arr = [int(a) for a in tab["arrival"]]
    arrival = lambda d: arr[d] if d < len(arr) else 0          # noqa: E731
    s16 = max(max(abs(int(x)) for x in q).bit_length() - 15, 0)
    y = [rsh(int(x), s16) * int(tab["exp2"][scale & 0xFFFF]) for x in q]
    q8, s8 = digits(y, 8)
    eq = s16 - 16 + (scale >> 16) - 16 + s8
    sc = [min(max(rsh(int(dot), -(eq + int(lev) - 16 + 10)), -(1 << 30)), 1 << 30) for dot, lev in zip(k @ q8, kl)]
    parts = []
    for j in range(0, len(sc), CHUNK):
        m, E = max(sc[j:j + CHUNK]), int(vl[j:j + CHUNK].max())
        u = [rsh(arrival(m - x), 2) for x in sc[j:j + CHUNK]]
        w = np.array([rsh(a, E - int(lev)) for a, lev in zip(u, vl[j:j + CHUNK])], dtype=np.int64)
        parts.append((m, E, sum(u), [rsh(int(n), 8) for n in w @ v[j:j + CHUNK]]))
    M, L = max(p[0] for p in parts), max(p[1] for p in parts)
    A = sum(rsh(a * arrival(M - m), 24) for m, _, a, _ in parts)
    N = [sum(rsh(n[d] * arrival(M - m), 24 + L - E) for m, E, _, n in parts) for d in range(k.shape[1])]
    lead = A.bit_length() - 1
    f = (L + 8) * 65536 - (lead * 65536 + int(tab["log2"][(A >> (lead - 16)) & 0xFFFF]))
    return np.array([wrap(rsh(n * int(tab["exp2"][f & 0xFFFF]), 16 - (f >> 16))) for n in N], dtype=np.int64)
