"""Plain numpy forms, in 64 bits, of the operators for serving many sequences, with the tolerances of their results."""
import numpy as np

EPS16 = 2.0 ** -11                     # half a step of fp16, relative
TINY16 = 2.0 ** -25                    # half a step of fp16 below its normal range


def rotary(x, pos, freqs, mag=1.0, half=False, inverse=False):
    """(result, tolerance): one fp16 rounding, and three 32-bit operations on terms of |x| + |y| with an angle good to
    2^-24 of half a turn (3.2 * 2^-24) and cos, sin to 2^-23: below 2^-20 of the terms."""
    x = x.astype(np.float64)
    n = len(freqs)
    a = np.asarray(pos, np.float64)[:, None] * np.asarray(freqs)[None] * (-1 if inverse else 1)
    c, s = (np.cos(a) * mag)[:, None], (np.sin(a) * mag)[:, None]
    out, size = x.copy(), np.zeros_like(x)
    i = np.arange(n)
    d0, d1 = (i, i + n) if half else (2 * i, 2 * i + 1)
    u, v = x[..., d0], x[..., d1]
    out[..., d0], out[..., d1] = u * c - v * s, u * s + v * c
    size[..., d0] = size[..., d1] = (np.abs(u) + np.abs(v)) * abs(mag)
    return out, np.abs(out) * EPS16 * (size > 0) + TINY16 * (size > 0) + size * 2.0 ** -20


def attend(q, k, v, scale):
    """One query head over k, v [tokens, d]: (out, lse, tolerance of out, tolerance of lse). Scores are 32-bit sums of d
    products, scaled and exponentiated there (2^-22 relative each), weights may be rounded to fp16 (2^-11)."""
    d = q.shape[-1]
    if len(k) == 0:
        return np.zeros(d), -np.inf, np.zeros(d), 0.0
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    s = k @ q * scale
    ds = (d + 4) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(q)).max() + (np.abs(s).max() + 1) * 2.0 ** -21
    m = s.max()
    p = np.exp(s - m)
    l = p.sum()
    out = p @ v / l
    size = p @ np.abs(v) / l
    lse = m + np.log(l)
    return out, lse, np.abs(out) * EPS16 + TINY16 + size * (EPS16 + 2 * ds + len(k) * 2.0 ** -24), ds + abs(lse) * 2.0 ** -23 + 2.0 ** -20


class Pages:
    """The bookkeeping of a paged cache, one row after the other."""

    def __init__(self, n_pages, page_size, n_rows, max_pages):
        self.p, self.width = page_size, max_pages
        self.table, self.lengths, self.refs = np.full((n_rows, max_pages), -1, np.int32), np.zeros(n_rows, np.int32), np.zeros(n_pages, np.int32)

    def fork(self, parents):
        n = len(self.lengths)
        table, lengths = self.table.copy(), self.lengths.copy()
        for r, p in enumerate(parents):
            if p == -1:
                table[r], lengths[r] = -1, 0
            elif 0 <= p < n:
                table[r], lengths[r] = self.table[p], self.lengths[p]
        for t, step in ((table, 1), (self.table, -1)):
            np.add.at(self.refs, t[(t >= 0) & (t < len(self.refs))], step)
        self.table, self.lengths = table, lengths

    def reserve(self, new):
        """(status, list of (source, destination, filled slots)); nothing changes unless the status is 0."""
        table, lengths, refs = self.table.copy(), self.lengths.copy(), self.refs.copy()
        copies = []
        free = list(np.flatnonzero(refs == 0))
        for r, add in enumerate(new):
            n = int(lengths[r])
            if n + add > self.width * self.p:
                return 5, []
            if add and n % self.p and refs[table[r, n // self.p]] > 1:
                if not free:
                    return 5, []
                src, dst = int(table[r, n // self.p]), int(free.pop(0))
                refs[src] -= 1
                refs[dst] = 1
                table[r, n // self.p] = dst
                copies.append((src, dst, n % self.p))
            for j in range(-(-n // self.p), -(-(n + add) // self.p)):
                if not free:
                    return 5, []
                table[r, j] = free.pop(0)
                refs[table[r, j]] = 1
            lengths[r] = n + add
        self.table, self.lengths, self.refs = table, lengths, refs
        return 0, copies

    def compact(self):
        """(where each page went, live pages, list of (source, destination))"""
        to = np.where(self.refs > 0, np.arange(len(self.refs)), -1).astype(np.int32)
        moves, lo, hi = [], 0, len(self.refs) - 1
        while True:
            while lo < hi and self.refs[lo] > 0:
                lo += 1
            while lo < hi and self.refs[hi] == 0:
                hi -= 1
            if lo >= hi:
                break
            moves.append((hi, lo))
            to[hi], self.refs[lo], self.refs[hi] = lo, self.refs[hi], 0
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], self.table).astype(np.int32)
        return to, int((self.refs > 0).sum()), moves


def beam_values(logits, scores, finished=None, pad=0):
    """[rows, vocab] values of all candidates in 64 bits."""
    x = np.clip(np.nan_to_num(logits.astype(np.float64), nan=-np.inf, posinf=65504.0, neginf=-np.inf), None, 65504.0)
    s = np.where(np.isnan(scores), -np.inf, np.asarray(scores, np.float32)).astype(np.float64)
    m = x.max(axis=1, keepdims=True)
    ok = np.isfinite(m)
    base = np.where(ok, m, 0.0)
    lse = base + np.log(np.maximum(np.exp(x - base).sum(axis=1, keepdims=True), 1e-300))
    with np.errstate(invalid="ignore"):
        v = np.where(ok, s[:, None] + (x - lse), -np.inf)
    if finished is not None:
        f = np.asarray(finished) != 0
        v[f] = -np.inf
        v[f, pad] = s[f]
    return v


def beam_select(logits, scores, beams, k, finished=None, pad=0):
    """(values, parent rows, tokens, smallest gap between neighbours that are not equal)"""
    v = beam_values(logits, scores, finished, pad)
    rows, vocab = v.shape
    flat = v.reshape(rows // beams, beams * vocab)
    order = np.argsort(-flat, axis=1, kind="stable")[:, :min(k + 1, beams * vocab)]
    best = np.take_along_axis(flat, order, 1)
    with np.errstate(invalid="ignore"):
        d = -np.diff(best, axis=1)
    d = d[np.isfinite(d) & (d > 0)]
    first = np.arange(rows // beams)[:, None] * beams
    o = order[:, :k]
    return best[:, :k], (first + o // vocab).astype(np.int32), (o % vocab).astype(np.int32), d.min() if d.size else np.inf
