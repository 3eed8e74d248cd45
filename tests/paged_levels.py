"""Batches on the paged cache whose scores are exact, for tests of how softmax weights are held.

Keys and queries are zeros but for their first element, so a score is one product of two fp16 numbers, which fp32 holds:
what is left of an output's error is its weights', their sums' and its own rounding."""
import numpy as np

from paged_reference import HD, World

OCTAVE = np.log2(np.e) / np.sqrt(128.0)  # of a weight, for a step of 1 in q k
FP16, TWO_FP16 = 2.0 ** -11, 2.0 ** -22  # half a step of a weight in one and in two fp16 numbers
FLOOR = 2.0 ** -31  # of the row's largest weight: what a weight may be off by however small it is


class Levels(World):
    """A World whose key at position i has the level level[i] (in place of q k: q's first element times it) and the value
    value[i] ([positions, 128]), the same in every kv head; `copies` sequences have the same pages and tokens."""

    def __init__(self, level, value, new=1, page=64, nq=12, nkv=2, copies=1):
        n = len(level)
        super().__init__(np.random.default_rng(n), [(n - new, new)], page, nq, nkv, spare=0, pad_rows=0)
        self.k[0][:] = 0
        self.k[0][:, :, 0] = level
        self.v[0][:] = value
        self.store(0)
        self.lens, self.k, self.v = self.lens * copies, self.k * copies, self.v * copies
        self.table = np.ascontiguousarray(np.repeat(self.table, copies, 0))
        self.context = np.repeat(self.context, copies)
        self.starts = np.arange(copies + 1, dtype=np.int32) * new
        self.rows = copies * new
        self.new, self.copies = new, copies

    def levels(self, q0):
        """Queries with first elements q0 [q heads]."""
        q = np.zeros((self.rows, self.nq, HD), np.float16)
        q[:, :, 0] = q0
        return q

    def attention_within(self, q, weight, round_weights=None):
        """(out, tolerance, log sums, theirs) of one copy's rows; `round_weights`: what to do to weights (as multiples of
        2^-7 of the row's largest) before they meet V, to see what that would give."""
        n = self.k[0].shape[1]
        shape = self.new, self.nq
        out, tol, lse, lse_tol = (np.zeros(shape + s) for s in ((HD,), (HD,), (), ()))
        for t in range(self.new):
            at = np.arange(n - self.new + t + 1)
            for h in range(self.nq):
                x = q[t, h, 0].astype(np.float64) * self.k[0][h // self.group, at, 0].astype(np.float64) * OCTAVE
                v = self.v[0][h // self.group, at].astype(np.float64)
                m = x.max()
                e = np.exp2(x - m)
                total = e.sum()
                out[t, h] = (e if round_weights is None else round_weights(128.0 * e) / 128.0) @ v / total
                rel, lse_tol[t, h] = errors(x, at.size)
                size = (e @ np.abs(v)) / total + np.abs(out[t, h])
                tol[t, h] = FP16 * np.abs(out[t, h]) + 2.0 ** -25 + (weight + rel) * size \
                    + FLOOR * (np.abs(v).sum(0) + at.size * np.abs(out[t, h])) / total
                lse[t, h] = (m + np.log2(total)) * np.log(2.0)
                lse_tol[t, h] += 2.0 ** -22 * abs(lse[t, h])
        return out, tol, lse, lse_tol


def errors(x, n):
    """Of a weight, relative, and of a log sum.  The exponent, at most `most` octaves, is rounded once (2^-24 of it), its
    scale is a number of 24 bits and so is the reference value (2^-24 of the score each): times ln 2.  The exponential has
    2^-22, and 2^-22 where the reference changes.  A sum of n terms takes them 16 at a time, or in 16 lanes and waves, at most
    n / 8 + 64 additions behind each other, of 2^-24 each; numerators and denominators have one each."""
    most = np.abs(x).max() + 64.0
    one = 3 * most * 2.0 ** -24 * np.log(2.0) + 2.0 ** -21
    return one + 2 * (n / 8 + 64) * 2.0 ** -24, one + (n / 8 + 64) * 2.0 ** -24


def check(got, lse, want, copies):
    """Every copy's rows."""
    out, tol, log, log_tol = want
    got = got.astype(np.float64).reshape(copies, *out.shape)
    off = np.abs(got - out) - tol
    assert np.all(off <= 0), (np.argwhere(off > 0)[:3], got[off > 0][:3], np.broadcast_to(out, got.shape)[off > 0][:3],
                              np.broadcast_to(tol, got.shape)[off > 0][:3])
    assert np.all(np.abs(lse.reshape(copies, *log.shape) - log) <= log_tol)


def far_below(n, depth, every=32, seed=0):
    """Levels and values: a key in `every` (the first of them) far above the others, with values of 0."""
    level = np.full(n, np.float16(-depth / (16 * OCTAVE)), np.float16)
    level[::every] = 0
    value = np.random.default_rng(seed).uniform(10000, 30000, (n, HD)).astype(np.float16)
    value[::every] = 0
    return level, value


def odd_weights(count):
    """First elements of q for which a key of level -1 has a weight that is far from any fp16 number (a quarter of a step and
    more), beside one of level 0."""
    q = np.arange(64, 3000) / 64.0
    w = 128.0 * np.exp2(-q * OCTAVE)
    off = np.abs(w.astype(np.float16).astype(np.float64) - w) / w
    found = q[off > 2.0 ** -12]
    return found[np.linspace(0, found.size - 1, count).astype(int)].astype(np.float16)


def cancelling(n, q0):
    """Levels 0 and -1 in turns, and values with which a head's outputs are nearly 0 in dims of its own: there an error that
    all weights of level -1 have in common is not hidden by the output's rounding."""
    level = np.where(np.arange(n) % 2, -1, 0).astype(np.float16)
    value = np.ones((n, HD))
    for d in range(HD):
        w = np.exp2(-float(q0[d % len(q0)]) * OCTAVE)
        value[level == 0, d] = -1000.0 * np.float16(w)
        value[level != 0, d] = 1000.0
    return level, value.astype(np.float16)
