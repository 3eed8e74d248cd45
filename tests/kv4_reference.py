"""The 4-bit key/value cache and the log probabilities in 64 bits (numpy), from
their definitions, for the GPU tests: rows are uint8 [..., 80]."""
import numpy as np

ROW = 80
_SHIFTS = np.array([0, 16, 4, 20, 8, 24, 12, 28], np.uint32)


def parts(rows):
    """(nibbles [..., 128], scale [..., 4], low [..., 4]) of cache rows."""
    rows = np.ascontiguousarray(rows)
    words = np.ascontiguousarray(rows[..., :64]).view("<u4")
    n = ((words[..., None] >> _SHIFTS) & 15).reshape(*rows.shape[:-1], 128)
    par = np.ascontiguousarray(rows[..., 64:]).view("<f2").astype(np.float64)
    return n.astype(np.float64), par[..., 0::2], par[..., 1::2]


def values(rows):
    """What rows stand for: fp16(n * scale + low), as float64."""
    n, scale, low = parts(rows)
    g = n.reshape(*n.shape[:-1], 4, 32)
    with np.errstate(invalid="ignore"):
        return (g * scale[..., None] + low[..., None]).astype(np.float16).astype(np.float64).reshape(n.shape)


def pack(n, scale, low):
    """Rows from nibbles [..., 128] and fp16 (scale, low) [..., 4]."""
    words = (n.reshape(*n.shape[:-1], 16, 8).astype(np.uint32) << _SHIFTS).sum(-1, dtype=np.uint32)
    par = np.stack([scale.astype(np.float16), low.astype(np.float16)], -1).reshape(*n.shape[:-1], 8)
    return np.concatenate([np.ascontiguousarray(words).view(np.uint8), np.ascontiguousarray(par).view(np.uint8)], -1)


def random_rows(rng, *shape, spread=1.0, offset=1.0):
    """Rows whose values look like a cache's: groups with a level and a spread of their own."""
    n = rng.integers(0, 16, (*shape, 128))
    scale = (rng.random((*shape, 4)) * 0.3 + 0.05) * spread
    low = rng.standard_normal((*shape, 4)) * offset - 7.5 * scale
    return pack(n, scale, low)


def rotate(x, pos, rot, theta):
    """NeoX rotation of [T, heads, 128] at positions pos, pos + 1, ..."""
    half = rot // 2
    a = (pos + np.arange(x.shape[0], dtype=np.float64))[:, None] * theta ** (-2.0 * np.arange(half) / rot)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x0, x1 = x[..., :half], x[..., half:rot]
    return np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s, x[..., rot:]], -1)


def attention(q, k, v, last):
    """q [rows, 128], k, v [n, 128], last [rows]: row i takes cache rows 0..last[i].
    Returns (out, weights p [rows, n], log sum, the tolerance of a kernel's fp16 out, of its p, relative).

    Tolerances: a score is a sum of 128 products in fp32, at most 16 roundings in a row, so it is off by
    d = 2^-20 sum |q k| / sqrt(128), and so is the logarithm of the softmax sum; p is then off by 2 d, relative, and
    2^-19 for the exponentials and sums.  For the product with V, p is rounded to fp16 (2^-11, or 2^-25 absolute
    against the row's maximum where it is subnormal), the output once more (2^-11)."""
    with np.errstate(invalid="ignore", over="ignore"):
        s = (q @ k.T) / np.sqrt(128.0)
    seen = np.arange(k.shape[0])[None] <= np.asarray(last)[:, None]
    s = np.where(seen, s, -np.inf)
    m = s.max(-1, keepdims=True)
    e = np.where(seen, np.exp(s - m), 0.0)
    total = e.sum(-1, keepdims=True)
    p = e / total
    vz = np.where(np.isfinite(v), v, 0.0)
    out = p @ vz
    d = 2.0 ** -20 * np.where(seen, np.abs(q) @ np.abs(k).T, 0.0).max(-1, keepdims=True) / np.sqrt(128.0)
    rel = 2 * d + 2.0 ** -19
    mass = p @ np.abs(vz)
    # the kernel's reference value may lag the maximum by 2^8, never lead it
    tol = 2.0 ** -11 * np.abs(out) + (2.0 ** -11 + rel) * mass + 2.0 ** -25 * (seen @ np.abs(vz)) / total + 2.0 ** -25
    return out, p, (m + np.log(total))[:, 0], tol, rel


def logprobs(x, ids, top):
    """x [rows, vocab] fp16; (logprob, entropy, top logprob, top ids, T / S)."""
    x = x.astype(np.float64)
    rows, vocab = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = np.where(np.isnan(x).all(-1), np.nan, np.nanmax(np.where(np.isnan(x), -np.inf, x), -1))[:, None]
        nothing = (x == -np.inf).all(-1)
        d = np.where(nothing[:, None], -np.inf, x - np.where(np.isfinite(m), m, 0.0))
        e = np.exp(d)
        e = np.where((np.isnan(x) | (x == np.inf)).any(-1)[:, None], np.nan, e)
        total = e.sum(-1)
        t = np.where(e > 0, e * np.where(e > 0, d, 0.0), np.where(np.isnan(e), np.nan, 0.0)).sum(-1)
        lp = d - np.log(total)[:, None]
        lp = np.where(nothing[:, None], -np.inf, lp)
        entropy = np.where(nothing, 0.0, np.log(total) - t / total)
    out = np.array([lp[i, ids[i]] if 0 <= ids[i] < vocab else 0.0 for i in range(rows)])
    tl, ti = np.full((rows, top), np.nan), np.full((rows, top), -1)
    for i in range(rows):
        ok = np.flatnonzero(~np.isnan(x[i]))
        best = ok[np.argsort(-x[i, ok], kind="stable")][:top]  # stable: the lower index first
        ti[i, :best.size] = best
        tl[i, :best.size] = lp[i, best]
    return out, entropy, tl, ti, np.abs(np.where(nothing, 0.0, t / np.where(total == 0, 1, total)))
