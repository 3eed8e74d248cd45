"""GPU parity of token log probabilities, entropy and top alternatives with
their definition in 64 bits (kv4_reference.logprobs).

Tolerances: a sum of probabilities is at most 64 fp32 roundings in a row, 2^-18 of itself, so its logarithm is off by
2^-18; the exponent's own rounding adds less than that (|d| exp(d) <= 1/e); the subtraction rounds once more."""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from helpers import dev, empty, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    qe_amd.lib()
    return qe_amd


def _run(qe, x, ids, top, skew=0, stride=None):
    """x [rows, vocab] laid out with a row stride and `skew` elements past an aligned address; rubbish around it."""
    rows, vocab = x.shape
    stride = stride or vocab
    buf = np.full(skew + rows * stride + 64, np.float16(60000.0))
    for r in range(rows):
        buf[skew + r * stride:skew + r * stride + vocab] = x[r]
    d = dev(buf)
    ws = torch.full((qe.token_logprobs_workspace_bytes(rows, vocab, top),), 0xFF, dtype=torch.uint8, device="cuda")
    lp, ent = empty(rows, torch.float32), empty(rows, torch.float32)
    tl, ti = (empty((rows, top), torch.float32), empty((rows, top), torch.int32)) if top else (None, None)
    qe.launch_token_logprobs(d.data_ptr() + 2 * skew, dev(np.asarray(ids, np.int32)), lp, ent, tl, ti, ws, rows,
                             vocab_size=vocab, row_stride=stride, top_k=top)
    return host(lp), host(ent), host(tl) if top else None, host(ti) if top else None


def _same(got, want, tol, what):
    got = got.astype(np.float64)
    special = ~np.isfinite(want)
    assert np.array_equal(got[special], want[special], equal_nan=True), what
    err = np.abs(got[~special] - want[~special])
    limit = np.broadcast_to(tol, want.shape)[~special]
    assert np.all(err <= limit), f"{what}: {np.max(err / limit)} of the tolerance"


def _check(qe, x, ids, top, **layout):
    got = _run(qe, x, ids, top, **layout)
    lp, ent, tl, ti, mean = ref.logprobs(x, ids, top)
    with np.errstate(invalid="ignore"):
        _same(got[0], lp, 2.0 ** -17 + 2.0 ** -22 * np.abs(lp), "logprob")
        _same(got[1], ent, 2.0 ** -17 * (1 + mean), "entropy")
        if top:
            assert np.array_equal(got[3], ti), "top ids"
            _same(got[2], tl, 2.0 ** -17 + 2.0 ** -22 * np.abs(tl), "top logprob")


def _logits(rng, rows, vocab, banned=0.02):
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float16)
    x[rng.random((rows, vocab)) < banned] = -np.inf
    return x


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 33, 64, 65, 1000, 8185, 8186, 8192, 8193, 50257, 151936, 300001])
def test_vocabularies(qe, vocab):
    rng = np.random.default_rng(vocab)
    rows = 3
    x = _logits(rng, rows, vocab)
    x[:, 0] = 1.0
    ids = [0, vocab - 1, vocab // 2]
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
        _check(qe, x, ids, top)


@pytest.mark.parametrize("skew", range(8))
@pytest.mark.parametrize("vocab,extra", [(1000, 0), (1001, 0), (8190, 3), (513, 1000)])
def test_strides_and_alignments(qe, skew, vocab, extra):
    rng = np.random.default_rng(skew)
    x = _logits(rng, 5, vocab)
    _check(qe, x, rng.integers(0, vocab, 5), 8, skew=skew, stride=vocab + extra)


def test_many_rows(qe):
    rng = np.random.default_rng(1)
    x = _logits(rng, 300, 2000)
    _check(qe, x, rng.integers(0, 2000, 300), 5)


@pytest.mark.parametrize("top", [1, 5, 32])
def test_ties_and_orders(qe, top):
    vocab = 20000
    rng = np.random.default_rng(2)
    rows = [np.zeros(vocab), np.arange(vocab) / 4.0, -np.arange(vocab) / 4.0, np.where(np.arange(vocab) % 2, 0.0, -0.0),
            rng.integers(0, 3, vocab).astype(np.float64), np.full(vocab, -np.inf), np.full(vocab, 65504.0)]
    rows.append(np.full(vocab, -np.inf))
    rows[-1][19999] = -5.0
    rows.append(np.full(vocab, -65504.0))
    rows[-1][[5, 12345]] = 65504.0
    x = np.stack(rows).astype(np.float16)
    _check(qe, x, [7, 19999, 0, 5, 100, 3, 0, 19999, 12345], top)


@pytest.mark.parametrize("vocab", [40, 9000])
def test_infinities_and_nan(qe, vocab):
    rng = np.random.default_rng(3)
    x = _logits(rng, 5, vocab, banned=0)
    x[0, vocab - 2] = np.nan
    x[1, 3] = np.inf
    x[2] = np.nan
    x[3, 20:] = np.nan      # fewer numbers than alternatives asked for
    x[4, [0, vocab - 1]] = [np.inf, np.nan]
    _check(qe, x, [0, 3, 1, 2, 0], 32)


def test_ids_outside_and_no_ids(qe):
    rng = np.random.default_rng(4)
    x = _logits(rng, 4, 500, banned=0)
    got = _run(qe, x, [-1, 500, -100, 2**31 - 1], 0)
    assert np.all(got[0] == 0.0)
    ent = empty(4, torch.float32)
    ws = empty(qe.token_logprobs_workspace_bytes(4, 500, 0), torch.uint8)
    qe.launch_token_logprobs(dev(x), None, None, ent, None, None, ws, 4, vocab_size=500)
    assert np.array_equal(host(ent), got[1])


def test_agrees_with_the_greedy_sampler(qe):
    rng = np.random.default_rng(5)
    x = rng.integers(-3, 4, (1, 151936)).astype(np.float16)
    val, idx, tok = empty(256, torch.float32), empty(256, torch.int32), empty(1, torch.int32)
    qe.launch_sample_and_advance(dev(x[0]), val, idx, None, tok)
    assert _run(qe, x, [0], 1)[3][0, 0] == host(tok)[0]


def test_recorded_into_a_graph(qe):
    rng = np.random.default_rng(6)
    rows, vocab, top = 3, 30000, 5
    x, ids = torch.zeros((rows, vocab), dtype=torch.float16, device="cuda"), dev(np.array([1, 2, 29999], np.int32))
    out = [empty(rows, torch.float32), empty(rows, torch.float32), empty((rows, top), torch.float32),
           empty((rows, top), torch.int32)]
    ws = empty(qe.token_logprobs_workspace_bytes(rows, vocab, top), torch.uint8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        qe.launch_token_logprobs(x, ids, *out, ws, rows, vocab_size=vocab, top_k=top)
    for _ in range(4):
        new = _logits(rng, rows, vocab)
        x.copy_(dev(new))
        g.replay()
        torch.cuda.synchronize()
        want = _run(qe, new, [1, 2, 29999], top)
        assert all(np.array_equal(host(a), b) for a, b in zip(out, want))
