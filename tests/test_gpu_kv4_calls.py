"""Calls of the 4-bit cache kernels that their documentation allows and that reach other
code than the usual ones (definition and tolerances: kv4_reference.py)."""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from helpers import dev, empty, host
from test_gpu_kv4 import _cache, _check, _ctl, _decode, _prefill, qe, workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,base", [(1, 700), (40, 1200), (600, 300)])
def test_outputs_in_the_place_of_q(qe, workspace, T, base):
    rng = np.random.default_rng(T)
    nq, nkv, ms = 12, 2, 2048
    kv = _cache(rng, nkv, ms, base + T)
    q = rng.standard_normal((T, nq * 128)).astype(np.float16)
    apart, _ = _prefill(qe, kv, q, T, nq, base, None, ms)
    x = dev(q)
    qe.launch_attention_gqa_prefill_kv4(x, dev(kv[0]), dev(kv[1]), x, _ctl(base), None, T, num_q_heads=nq,
                                        num_kv_heads=nkv, max_seq_len=ms, hidden_size=nq * 128)
    assert np.array_equal(host(x).view(np.uint16), apart.view(np.uint16))
    _check(qe, kv, q, T, nq, base, [0] * nkv, ms, apart)
    one, ws = dev(q[-1]), empty(qe.kv4_decode_workspace_bytes(nq, ms), torch.uint8)
    qe.launch_attention_gqa_flash_decode_kv4(one, dev(kv[0]), dev(kv[1]), ws, one, _ctl(base + T - 1), None, None, nq, nkv,
                                             max_seq_len=ms)
    assert np.array_equal(host(one), _decode(qe, kv, q[-1], nq, base + T - 1, None, ms))


# ---- chunks of many rows ---------------------------------------------------------------------
# Blocks of eight waves (28 blocks of 256 rows and more), merges by one group with more than eight splits, sums of the
# key weights over four shares of the q rows and by the rule for many key blocks: test_kv4_variants.py says which.
def _chunk(qe, T, base, nq, nkv, ms, gone=None):
    """A chunk with key weights, then without: checked against the definition, and against each other.  (The weights'
    tolerance holds 66 fp32 roundings in a row: up to 50 tiles of q rows here, five steps over lanes, four waves, four
    shares and the weight before.)"""
    rng = np.random.default_rng(T + base)
    gone = gone or [9] * nkv
    pos = base + 9
    kv = _cache(rng, nkv, ms, min(pos - min(gone) + T, ms))
    q = (1.5 * rng.standard_normal((T, nq * 128))).astype(np.float16)
    w_in = rng.random((nkv, ms), np.float32)
    w = dev(np.full((nkv, ms), -7, np.float32))
    got, lse = _prefill(qe, kv, q, T, nq, pos, gone, ms, nq * 128 + 64, weights=w, w_in=dev(w_in))
    w = host(w)
    for h in range(nkv):
        assert np.all(w[h, min(max(pos - gone[h], 0) + T, ms):] == -7)
    _check(qe, kv, q, T, nq, pos, gone, ms, got, lse, w_in, w)
    again, _ = _prefill(qe, kv, q, T, nq, pos, gone, ms)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("T,base,nq,nkv,ms", [(600, 0, 12, 2, 1100), (598, 1000, 12, 2, 1700), (130, 1, 64, 32, 1100),
                                              (257, 100, 28, 28, 1100), (2400, 63, 4, 4, 2500), (100, 17, 128, 2, 1100),
                                              (640, 1300, 12, 2, 20000)])
def test_chunks_of_eight_waves(qe, T, base, nq, nkv, ms, split):
    if split:
        qe.gemm_reserve_workspace()
    try:
        _chunk(qe, T, base, nq, nkv, ms)
    finally:
        qe.gemm_release_workspace()


@pytest.mark.parametrize("T,base,nq,nkv", [(180, 5000, 12, 2), (200, 9000, 11, 1), (700, 6500, 3, 3)])
def test_rows_merged_from_more_than_eight_splits_by_one_group(qe, workspace, T, base, nq, nkv):
    _chunk(qe, T, base, nq, nkv, base + T + 3)


def test_eight_waves_and_more_than_eight_splits(qe, workspace):
    _chunk(qe, 512, 5000, 14, 2, 5600)


def test_eight_waves_with_heads_of_different_lengths_and_a_full_cache(qe, workspace):
    ms, base = 1500, 1700
    pos = base + 9
    # from rows 0, 509, 1059 and 1299 (the last tokens find no room), 899, 900 (exactly full), 1509 and 1709 (none does)
    gone = [pos, 1200, 650, 410, pos - 899, pos - 900, 200, 0]
    _chunk(qe, 600, base, 16, 8, ms, gone=gone)


def test_eight_waves_and_the_poison_of_a_later_token(qe, workspace):
    rng = np.random.default_rng(51)
    T, nq, nkv, base = 600, 12, 2, 700
    ms = base + T + 10
    for at in (0, 130, 599):
        kv = _cache(rng, nkv, ms, base + T)
        kv[0, :, base + at, 64:] = np.frombuffer(np.full(8, 0x7E00, np.uint16).tobytes(), np.uint8)
        kv[1, :, base + at] = 0
        q = rng.standard_normal((T, nq * 128)).astype(np.float16)
        w = dev(np.zeros((nkv, ms), np.float32))
        got, lse = _prefill(qe, kv, q, T, nq, base, None, ms, weights=w)
        assert np.all(np.isnan(got[at:])) and np.all(np.isnan(lse[at:]))
        if at:
            _check(qe, kv, q[:at], at, nq, base, [0, 0], ms, got[:at], lse[:at])
        w = host(w)
        assert np.all(np.isnan(w[:, :base + at + 1])) and np.all(w[:, base + T:] == 0)


def test_rows_whose_every_score_is_minus_infinity(qe, workspace):
    """A query with an infinity where every key is of the other sign: no softmax, so NaN, from every form alike."""
    rng = np.random.default_rng(61)
    nq, nkv, ms, ctx = 12, 2, 2048, 1500
    kv = _cache(rng, nkv, ms, ctx)
    k = rng.standard_normal((nkv, ctx, 128)) + 3.0
    group = np.clip(k, 0.5, None).reshape(nkv, ctx, 4, 32)  # every key value positive
    low = group.min(-1).astype(np.float16)
    scale = ((group.max(-1) - low) / 15).astype(np.float16)
    kv[0, :, :ctx] = ref.pack(np.clip(np.rint((group - low[..., None]) / scale[..., None]), 0, 15).reshape(nkv, ctx, 128),
                              scale, low)
    assert (ref.values(kv[0, :, :ctx]) > 0).all()
    for T, base in ((40, 1400), (40, 3), (600, 800)):  # splits, none, eight waves
        q = rng.standard_normal((T, nq * 128)).astype(np.float16)
        q[5, 4 * 128 + 9] = -np.inf
        out, lse = _prefill(qe, kv, q, T, nq, base, None, ms, lse=True)
        assert np.all(np.isnan(out[5, 4 * 128:5 * 128])) and lse[5, 4] == -np.inf
        out[5, 4 * 128:5 * 128] = 0
        assert np.all(np.isfinite(out))
    assert np.all(np.isnan(_decode(qe, kv, q[5], nq, 1000, None, ms)[4 * 128:5 * 128]))


def test_q8_of_a_head_that_is_nan(qe):
    """attn_out is NaN; Q8_1 cannot say so: zeros with the smallest scale, as the fp16 flash decode's epilogue."""
    rng = np.random.default_rng(62)
    nq, nkv, ms = 12, 2, 500
    kv = _cache(rng, nkv, ms, 400)
    clean = _decode(qe, kv, np.ones(nq * 128, np.float16), nq, 399, None, ms, q8=True)
    kv[0, 1, 250, 64:] = np.frombuffer(np.full(8, 0x7E00, np.uint16).tobytes(), np.uint8)
    out, q8, scale, sum8 = _decode(qe, kv, np.ones(nq * 128, np.float16), nq, 399, None, ms, q8=True)
    half = nq // 2 * 128
    assert np.all(np.isnan(out[half:])) and np.all(q8[half:] == 0) and np.all(sum8[half // 8:] == 0)
    assert np.all(scale[nq // 2:] == np.float32(1e-8))
    for got, want in zip((out, q8, scale, sum8), clean):
        assert np.array_equal(got[:got.size // 2], want[:want.size // 2])
