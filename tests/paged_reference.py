"""The paged key/value cache and attention on it in 64 bits (numpy), from their definitions, for the GPU tests.

A World is a batch of sequences with a pool of pages.  Rows of pages that no sequence uses hold NaN, so that
whoever reads one shows it."""
import numpy as np

from helpers import dev

HD = 128


class World:
    """lens: (tokens before, new tokens) of each sequence, a negative first number for one that takes no part;
    `known`: rows that are in the cache already (default: all, the new tokens' too)."""

    def __init__(self, rng, lens, page=16, nq=12, nkv=2, joint=False, pad_rows=0, spare=2, holes=(), single=None,
                 k_level=0.5, known=None, first_row=0, stride_pages=1):
        self.rng, self.lens, self.page, self.nq, self.nkv, self.group = rng, lens, page, nq, nkv, nq // nkv
        blocks = [max(0, (a + n - 1) // page + 1) if a >= 0 else 1 for a, n in lens]
        self.max_pages = max(blocks) + spare
        order = rng.permutation(sum(blocks) + 3)
        self.num_pages = order.size
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        at = 0
        for s, b in enumerate(blocks):
            self.table[s, :b] = order[at:at + b]
            at += b
        self.k, self.v = [], []  # [kv heads, positions, 128] of each sequence, as stored
        shape = (self.num_pages, nkv, page, HD)
        self.k_pages, self.v_pages = (np.full(shape, np.nan, np.float16) for _ in range(2))
        for s, (a, n) in enumerate(lens):
            m = max(0, a + (n if known is None else known))
            k = (rng.standard_normal((nkv, m, HD)) + k_level * rng.standard_normal((nkv, 1, HD))).astype(np.float16)
            v = rng.standard_normal((nkv, m, HD)).astype(np.float16)
            self.k.append(k)
            self.v.append(v)
            self.store(s)
        for s, b in holes:  # a page that the table does not name
            self.table[s, b] = rng.choice([-1, -2**31, self.num_pages, 2**31 - 1])
        self.single = all(n == 1 for _, n in lens) and first_row == 0 if single is None else single
        starts = [first_row]
        for _, n in lens:
            starts.append(starts[-1] + n)
        self.starts = np.array(starts, np.int32)
        self.rows = starts[-1] + pad_rows
        if self.single:
            assert self.rows == len(lens)
        self.context = np.array([a for a, _ in lens], np.int32)
        self.joint, self.stride_pages = joint, stride_pages

    def store(self, s):
        """The rows of a sequence into its pages."""
        for x, pages in ((self.k[s], self.k_pages), (self.v[s], self.v_pages)):
            for b in range((x.shape[1] + self.page - 1) // self.page):
                part = x[:, b * self.page:(b + 1) * self.page]
                if 0 <= self.table[s, b] < self.num_pages:
                    pages[self.table[s, b], :, :part.shape[1]] = part

    def device(self, qe):
        """(cache, batch) on the GPU."""
        import torch
        if self.joint:
            pool = dev(np.stack([self.k_pages, self.v_pages], 1))
            k, v = pool[:, 0], pool[:, 1]
        elif self.stride_pages > 1:  # pages far apart
            size = self.nkv * self.page * HD
            pools = [torch.empty(self.num_pages * self.stride_pages * size, dtype=torch.float16, device="cuda")
                     for _ in range(2)]
            k, v = (p.as_strided(self.k_pages.shape, (self.stride_pages * size, self.page * HD, HD, 1)) for p in pools)
            k.copy_(dev(self.k_pages))
            v.copy_(dev(self.v_pages))
        else:
            k, v = dev(self.k_pages), dev(self.v_pages)
        self.tensors = k, v
        batch = qe.paged_batch(dev(self.table), dev(self.context), None if self.single else dev(self.starts), self.rows)
        return qe.paged_cache(k, v), batch

    def tokens(self):
        """(row, sequence, position) of every new token."""
        for s, (a, n) in enumerate(self.lens):
            if a >= 0:
                for t in range(n):
                    yield int(self.starts[s]) + t, s, a + t

    def has_page(self, s, pos):
        b = np.asarray(pos) // self.page
        inside = b < self.max_pages
        page = self.table[s, np.minimum(b, self.max_pages - 1)]
        return inside & (page >= 0) & (page < self.num_pages)

    def queries(self, scale=1.0):
        return (scale * self.rng.standard_normal((self.rows, self.nq, HD))).astype(np.float16)

    def attention(self, q, window=0, selected=None):
        """(out, its tolerance, log sums, theirs, rows that take part) for all rows."""
        out = np.zeros((self.rows, self.nq, HD))
        tol, lse, lse_tol = np.zeros_like(out), np.zeros((self.rows, self.nq)), np.zeros((self.rows, self.nq))
        live = np.zeros(self.rows, bool)
        for row, s, pos in self.tokens():
            live[row] = True
            for h in range(self.nkv):
                k, v = self.k[s][h], self.v[s][h]
                at = np.arange(min(pos + 1, k.shape[0]))
                if selected is None:
                    at = at[self.has_page(s, at) & (at > pos - window if window else True)]
                else:
                    blocks = [b for b in selected[row, h].tolist() if 0 <= b and b * self.page <= pos and b < self.max_pages]
                    at = np.concatenate([np.arange(b * self.page, min(pos + 1, (b + 1) * self.page)) for b in blocks]
                                        + [np.zeros(0, int)]).astype(int)
                    at = at[self.has_page(s, at)]
                heads = slice(h * self.group, (h + 1) * self.group)
                out[row, heads], tol[row, heads], lse[row, heads], lse_tol[row, heads] = \
                    softmax_rows(q[row, heads].astype(np.float64), k[at].astype(np.float64), v[at].astype(np.float64))
        return out, tol, lse, lse_tol, live


def softmax_rows(q, k, v):
    """softmax(q k^T / sqrt(128)) v of rows q, and the logarithm of the sum; no key: zeros and -inf.

    Tolerances.  A score is a sum of 128 products in fp32: at most 127 roundings of 2^-24 of sum |q k|, d <
    2^-17 sum |q k| / sqrt(128).  The exponent is scaled and shifted in one rounding (2^-24 of a number below 2^7 in
    bits: 2^-17 relative in the weight), the exponential has 2^-22: weights are off by d + 2^-16 relative, and as much
    again through the sum.  The weights are rounded to fp16 for the product (2^-11, or 2^-25 of the row's largest
    where subnormal); the sums of n terms have n roundings of 2^-24; the output is rounded once (2^-11, 2^-25 where
    subnormal).  The logarithm: d + 2^-16 + n 2^-24, and 2^-22 of itself."""
    rows, n = q.shape[0], k.shape[0]
    if n == 0:
        return np.zeros((rows, HD)), 0.0, np.full(rows, -np.inf), 0.0
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        s = (q @ k.T) / np.sqrt(128.0)
        m = s.max(-1, keepdims=True)
        e = np.exp(s - m)
        total = e.sum(-1, keepdims=True)
        p = e / total
        out = p @ v
        d = 2.0 ** -17 * (np.abs(q) @ np.abs(k).T).max(-1, keepdims=True) / np.sqrt(128.0)
        rel = 2 * (d + 2.0 ** -16) + (n + 64) * 2.0 ** -24
        tol = 2.0 ** -11 * np.abs(out) + (2.0 ** -11 + rel) * (p @ np.abs(v)) + 2.0 ** -25 * np.abs(v).sum(0) / total + 2.0 ** -25
        lse = (m + np.log(total))[:, 0]
        return out, tol, lse, d[:, 0] + 2.0 ** -16 + (n + 64) * 2.0 ** -24 + 2.0 ** -22 * np.abs(lse)


def check(got, lse, want, untouched):
    """Outputs against World.attention's; rows that take no part still hold `untouched`."""
    out, tol, log, log_tol, live = want
    got = got.reshape(out.shape).astype(np.float64)
    assert np.all(got[~live] == untouched)
    bad = ~(np.abs(got[live] - out[live]) <= tol[live])
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got[live] - out[live])[bad][:4], np.broadcast_to(tol[live], bad.shape)[bad][:4])
    if lse is not None:
        assert np.all(lse[~live] == untouched)
        none = np.isneginf(log[live])
        assert np.array_equal(np.isneginf(lse[live]), none)
        bad = ~(np.abs(np.where(none, 0, lse[live]) - np.where(none, 0, log[live])) <= log_tol[live])
        assert not bad.any(), (np.argwhere(bad)[:4], lse[live][bad][:4], log[live][bad][:4])


def bounds(k, live):
    """(high and low bytes, step) of the first `live` rows of keys [kv heads, rows, 128]."""
    x = k[:, :live].astype(np.float64)
    with np.errstate(invalid="ignore"):
        high, low = x.max(1), x.min(1)
        m = np.maximum(np.abs(high), np.abs(low)).max(-1)
    if not np.isfinite(x).all():
        fine = np.isfinite(x).all((1, 2))
        high, low, m = (np.where(fine.reshape(-1, *[1] * (y.ndim - 1)), y, 0) for y in (high, low, m))
    d = np.where(m > 0, m, 1)[:, None]
    out = np.concatenate([np.ceil(127 * high / d), np.floor(127 * low / d)], -1).astype(np.int8)
    if not np.isfinite(k[:, :live].astype(np.float64)).all():
        m = np.where(fine, m, np.inf)
    return out, m


def scores(q, high_low, step):
    """Scores of blocks for the q heads [group, 128] of a kv head: bounds [blocks, 256], steps [blocks]."""
    q = q.astype(np.float64)
    best = np.full(step.size, -np.inf, np.float32)
    b = high_low.astype(np.float64)
    for x in q:
        m = np.abs(x).max()
        if not np.isfinite(x).all() or m == 0:
            n, m = np.zeros(HD), 0.0
        else:
            n = np.rint(127 * x / m)
        dot = np.maximum(n * b[:, :HD], n * b[:, HD:]).sum(-1)
        best = np.maximum(best, dot.astype(np.float32) * np.float32(m))
    with np.errstate(invalid="ignore"):
        return np.where(np.isinf(step), np.inf, best * step.astype(np.float32))


def select(score, there, own, num, sinks, recent):
    """Ascending blocks and -1: score and there for blocks 0 .. own (or as many as there can be)."""
    block = np.arange(score.size)
    sure = (block < sinks) | (block > own - recent)
    order = np.lexsort((block, -score.astype(np.float64), ~sure))
    order = [b for b in order if there[b]][:num]
    return np.array(sorted(order) + [-1] * (num - len(order)))
