"""GPU parity of log probabilities where rows are many and long: segments of 32768 logits (512 of them and more in a
call), and rows of more than 64 segments.  Definition: kv4_reference.logprobs.

Tolerances, with fp32 roundings of 2^-24: a probability is off by 2^-23 for the exponential and, its exponent t being
rounded, by |t| 2^-24 ln 2.  A sum S takes 64 additions in a lane, one of its two halves, six over lanes, then with the
factors that bring them to one maximum four waves, up to 2 (segments / 256 + 1) in a thread, six over lanes and four
waves again: n = 90 in all, so S and log S are off by e = (n + 2) 2^-24 + 2^-24 T' with T' = T / S below 2^4 here, and T
likewise, each term |t| p of it.  A log probability is x - m - log S with two roundings of its own size; the entropy
log S - T / S is off by e + 2 e |T / S|."""
import numpy as np
import pytest

import kv4_reference as ref
from test_gpu_logprobs import _logits, _run, _same, qe

pytestmark = pytest.mark.gpu


def _check(qe, x, ids, top, **layout):
    lp, ent, tl, ti, mean = ref.logprobs(x, ids, top)
    e = 92 * 2.0 ** -24 + 2.0 ** -24 * mean
    got = _run(qe, x, ids, top, **layout)
    with np.errstate(invalid="ignore"):
        _same(got[0], lp, e + 2.0 ** -22 * np.abs(lp), "logprob")
        _same(got[1], ent, e * (1 + 2 * mean) + 2.0 ** -22 * np.abs(ent), "entropy")
        if top:
            assert np.array_equal(got[3], ti), "top ids"
            _same(got[2], tl, e[:, None] + 2.0 ** -22 * np.abs(tl), "top logprob")


@pytest.mark.parametrize("rows,vocab,skew,extra,top", [
    (520, 2000, 0, 0, 5), (520, 2000, 3, 1, 32), (260, 40000, 0, 0, 0), (260, 40000, 5, 7, 20), (513, 20000, 1, 3, 1),
    (512, 32761, 0, 0, 8), (512, 32762, 7, 0, 8), (8, 2200000, 0, 0, 32), (8, 2200000, 6, 11, 5)])
def test_long_segments(qe, rows, vocab, skew, extra, top):
    rng = np.random.default_rng(rows + skew)
    x = _logits(rng, rows, vocab)
    x[:, 7] = 2.0
    ids = rng.integers(0, vocab, rows)
    ids[:4] = [0, vocab - 1, 7, -1]
    _check(qe, x, ids, top, skew=skew, stride=vocab + extra)


@pytest.mark.parametrize("skew", [0, 5])
@pytest.mark.parametrize("top", [1, 7, 32])
def test_rows_of_more_than_64_segments(qe, top, skew):
    rng = np.random.default_rng(top)
    x = _logits(rng, 3, 600001)
    x[1] = np.round(x[1])           # many equal alternatives
    x[2] = -np.inf
    x[2, [524287, 524288, 600000]] = 3.0
    _check(qe, x, [600000, 0, 524288], top, skew=skew)


@pytest.mark.parametrize("vocab", [20000, 40000])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_ties_orders_and_what_is_not_finite(qe, top, vocab):
    """The rows of test_ties_and_orders and test_infinities_and_nan, over and over until segments are long."""
    rng = np.random.default_rng(2)
    i = np.arange(vocab)
    kinds = [np.zeros(vocab), i / 8.0, -i / 8.0, np.where(i % 2, 0.0, -0.0), rng.integers(0, 3, vocab).astype(np.float64),
             np.full(vocab, -np.inf), np.full(vocab, 65504.0), np.where(i == vocab - 1, -5.0, -np.inf),
             np.where((i == 5) | (i == 12345), 65504.0, -65504.0), np.full(vocab, np.nan), np.where(i < 20, i, np.nan),
             np.where(i == vocab - 2, np.nan, 1.0), np.where(i == 3, np.inf, 0.0), np.where(i == 0, np.inf, np.nan),
             np.where(i % 7 == 0, 2.0, -np.inf), np.where(i < 32768, 1.0, 1.0 + (i % 2))]
    x = np.stack(kinds).astype(np.float16)
    rows = 520
    ids = rng.integers(0, vocab, len(kinds))
    lp, ent, tl, ti, mean = ref.logprobs(x, ids, top)
    pick = np.arange(rows) % len(kinds)
    got = _run(qe, x[pick], ids[pick], top)
    e = 92 * 2.0 ** -24 + 2.0 ** -24 * np.nan_to_num(mean)
    with np.errstate(invalid="ignore"):
        _same(got[0], lp[pick], (e + 2.0 ** -22 * np.abs(lp))[pick], "logprob")
        _same(got[1], ent[pick], (e * (1 + 2 * np.nan_to_num(mean)) + 2.0 ** -22 * np.abs(ent))[pick], "entropy")
        assert np.array_equal(got[3], ti[pick]), "top ids"
        _same(got[2], tl[pick], (e[:, None] + 2.0 ** -22 * np.abs(tl))[pick], "top logprob")
