"""GPU parity of the 4-bit key/value cache (append, unpack, decode and prefill
attention with key weights, eviction) with its definition in 64 bits
(kv4_reference.py, where the tolerances are derived)."""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from helpers import dev, empty, host

pytestmark = pytest.mark.gpu
THETA = 1000000.0


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    qe_amd.lib()
    return qe_amd


@pytest.fixture
def workspace(qe):
    """The default stream holds a split workspace, as the engine's stream does."""
    qe.gemm_reserve_workspace()
    yield
    qe.gemm_release_workspace()


def _ctl(pos):
    raw = np.zeros(64, np.int32)
    raw[1] = pos
    return dev(raw)


def _i32(*v):
    return dev(np.array(v, np.int32))


# ---- append -------------------------------------------------------------------------
def _append(qe, q, k, v, biases, caches, pos, evicted, ms, rot, theta=THETA, q_out=None, stream=None):
    nq, nkv = q.shape[1] // 128, k.shape[1] // 128
    dq = dev(q)
    out = dq if q_out == "same" else empty(q.shape, torch.float16)
    qe.launch_qkv_bias_rope_kv4_append(dq, out, dev(k), dev(v), *[None if b is None else dev(b) for b in biases],
                                       caches[0], caches[1], _ctl(pos), None if evicted is None else _i32(*evicted),
                                       q.shape[0], stream, num_q_heads=nq, num_kv_heads=nkv, max_seq_len=ms,
                                       rotary_dim=rot, rope_theta=theta)
    return host(out)


@pytest.mark.parametrize("T,nq,nkv,pos,gone,rot,bias", [
    (1, 12, 2, 0, 0, 0, True), (1, 12, 2, 1000, 0, 128, True), (3, 1, 1, 5, 0, 64, False), (33, 5, 5, 7, 3, 96, True),
    (16, 28, 4, 131071, 131000, 16, False), (2, 7, 1, 1000000, 999990, 128, True), (70, 16, 8, 100, 0, 32, True),
    (5, 40, 40, 200000000, 199999999, 128, True)])
def test_append(qe, T, nq, nkv, pos, gone, rot, bias):
    rng = np.random.default_rng(T * 1000 + nq)
    ms = pos - gone + T + 5
    q, k, v = (rng.standard_normal((T, n * 128)).astype(np.float16) for n in (nq, nkv, nkv))
    k[:, :128] *= np.float16(0.01)
    b = [rng.standard_normal(n * 128).astype(np.float16) * np.float16(3) if bias else None for n in (nq, nkv, nkv)]
    before = rng.integers(0, 256, (2, nkv, ms, 80), dtype=np.uint8)
    kc, vc = dev(before[0]), dev(before[1])
    got_q = _append(qe, q, k, v, b, (kc, vc), pos, [gone] * nkv, ms, rot)
    x = [a.astype(np.float64).reshape(T, -1, 128) + (0 if c is None else c.astype(np.float64).reshape(-1, 128))
         for a, c in zip((q, k, v), b)]
    r = rot or 128
    # fp32 sums and products, sines and cosines of an angle rounded to fp32 in [-pi, pi]: 2^-20 of what is added up
    slack = [2.0 ** -20 * (np.abs(a) + np.roll(np.abs(a[..., :r]), r // 2, -1)
                           if r == 128 else np.abs(a) + np.abs(a).max(-1, keepdims=True)) + 2.0 ** -25 for a in x]
    eq, ek = (ref.rotate(a, pos, r, THETA) for a in x[:2])
    err = np.abs(got_q.reshape(T, nq, 128).astype(np.float64) - eq)
    assert np.all(err <= 2.0 ** -11 * np.abs(eq) + slack[0]), (err - slack[0]).max()
    for cache, old, exact, sl in ((kc, before[0], ek, slack[1]), (vc, before[1], x[2], slack[2])):
        got = host(cache)
        row0 = pos - gone
        assert np.array_equal(got[:, :row0], old[:, :row0]) and np.array_equal(got[:, row0 + T:], old[:, row0 + T:])
        n, scale, low = ref.parts(got[:, row0:row0 + T])
        e, s = exact.transpose(1, 0, 2).reshape(nkv, T, 4, 32), sl.transpose(1, 0, 2).reshape(nkv, T, 4, 32).max(-1)
        assert np.all(np.abs(low - e.min(-1)) <= 2.0 ** -11 * np.abs(low) + s)
        want = (e.max(-1) - low) / 15
        assert np.all(np.abs(scale - want) <= 2.0 ** -11 * np.abs(want) + s)
        n = n.reshape(e.shape)
        # every element within half a step of its own value
        off = np.abs(low[..., None] + n * scale[..., None] - e)
        assert np.all(off <= scale[..., None] * (0.5 + 15 * 2.0 ** -11) + s[..., None]), off.max()


def test_append_in_place_and_repeatable(qe):
    rng = np.random.default_rng(3)
    T, nq, nkv, ms = 9, 12, 2, 64
    q, k, v = (rng.standard_normal((T, n * 128)).astype(np.float16) for n in (nq, nkv, nkv))
    outs = []
    for mode in (None, "same"):
        kc, vc = qe.kv4_cache(nkv, ms), qe.kv4_cache(nkv, ms)
        outs.append((_append(qe, q, k, v, [None] * 3, (kc, vc), 11, None, ms, 0, q_out=mode), host(kc), host(vc)))
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*outs))


def test_append_of_one_token_at_a_time_equals_a_chunk(qe):
    rng = np.random.default_rng(4)
    T, nq, nkv, ms = 7, 6, 3, 32
    q, k, v = (rng.standard_normal((T, n * 128)).astype(np.float16) for n in (nq, nkv, nkv))
    a, b = [qe.kv4_cache(nkv, ms) for _ in range(2)], [qe.kv4_cache(nkv, ms) for _ in range(2)]
    whole = _append(qe, q, k, v, [None] * 3, a, 9, [2, 2, 2], ms, 0)
    single = [_append(qe, q[t:t + 1], k[t:t + 1], v[t:t + 1], [None] * 3, b, 9 + t, [2, 2, 2], ms, 0) for t in range(T)]
    assert np.array_equal(whole, np.concatenate(single))
    assert all(np.array_equal(host(x), host(y)) for x, y in zip(a, b))


def test_append_heads_with_rows_of_their_own_and_a_full_cache(qe):
    """Heads may have lost different numbers of rows; tokens past the last row are not stored."""
    rng = np.random.default_rng(5)
    T, nkv, ms, pos = 6, 3, 16, 20
    q, k, v = (rng.standard_normal((T, nkv * 128)).astype(np.float16) for _ in range(3))
    kc, vc = qe.kv4_cache(nkv, ms), qe.kv4_cache(nkv, ms)
    kc.fill_(7), vc.fill_(7)
    gone = [4, 8, 2]  # first rows 16 (full), 12 (four fit), 18 (beyond)
    _append(qe, q, k, v, [None] * 3, (kc, vc), pos, gone, ms, 0)
    for c in (kc, vc):
        got = host(c)
        assert np.all(got[0] == 7) and np.all(got[2] == 7) and np.all(got[1, :12] == 7)
        assert not np.any(np.all(got[1, 12:] == 7, -1))
    # a count beyond the position is taken as the position: row 0
    kc.fill_(7)
    _append(qe, q[:1], k[:1], v[:1], [None] * 3, (kc, vc), 3, [9, 3, 2**31 - 1], ms, 0)
    got = host(kc)
    assert all(not np.all(got[h, 0] == 7) and np.all(got[h, 1:] == 7) for h in range(3))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan, "overflow"])
def test_append_poisons_what_fp16_cannot_hold(qe, which, value):
    rng = np.random.default_rng(6)
    T, nkv, ms = 3, 2, 8
    q, k, v = (rng.standard_normal((T, nkv * 128)).astype(np.float16) for _ in range(3))
    biases = [None] * 3
    bad = k if which == "k" else v
    if value == "overflow":
        bad[1, 128 + 77] = 65504
        bias = np.zeros(nkv * 128, np.float16)
        bias[128 + 77] = 16  # 65520 rounds to infinity
        biases = [None, bias, None] if which == "k" else [None, None, bias]
    else:
        bad[1, 128 + 77] = value
    kc, vc = qe.kv4_cache(nkv, ms), qe.kv4_cache(nkv, ms)
    # position 0 for the odd token, whose rotation is the identity
    _append(qe, q[1:2], k[1:2], v[1:2], biases, (kc, vc), 0, None, ms, 0)
    kv, vv = ref.values(host(kc)[:, 0]), ref.values(host(vc)[:, 0])
    assert np.all(np.isfinite(kv[0])) and np.all(np.isnan(kv[1]))
    assert np.all(np.isfinite(vv)) and np.all(vv[1] == 0) and np.any(vv[0] != 0)


def test_append_flat_and_tiny_groups(qe):
    T, ms = 1, 4
    k = np.zeros((1, 128), np.float16)
    v = np.zeros((1, 128), np.float16)
    v[0, :32] = 2.5                                          # one value: scale 0
    v[0, 32:64] = np.arange(32) * 2.0 ** -24                 # subnormal
    v[0, 64:96] = np.linspace(-60000, 60000, 32)             # most of the range
    v[0, 96:] = -1
    v[0, 96] = -1.001
    kc, vc = qe.kv4_cache(1, ms), qe.kv4_cache(1, ms)
    _append(qe, np.zeros((1, 128), np.float16), k, v, [None] * 3, (kc, vc), 0, None, ms, 0)
    assert np.all(ref.values(host(kc)[:, 0]) == 0)
    got, want = ref.values(host(vc)[0, 0]), v[0].astype(np.float64)
    assert np.all(got[:32] == 2.5)
    assert np.all(np.abs(got[32:64] - want[32:64]) <= 2.0 ** -24 * 1.5)  # steps of 2^-24 or 2^-23
    assert np.all(np.abs(got[64:96] - want[64:96]) <= 4000 * (1 + 2.0 ** -10) + 32)
    assert np.all(np.abs(got[96:] - want[96:]) <= 0.001)


def test_append_near_the_largest_fp16(qe):
    """What is finite is stored finite, also where the scale rounds up and a nibble of 15 would pass 65504."""
    top = 65504.0
    pairs = [(-top, top), (0, top), (top, top), (-top, -top), (top - 32, top), (-top, top - 32), (-32768, top),
             (-1.5, top), (-top, 0), (-61440, top), (8192, top), (-40000, 65472), (30000, top), (-50016, top),
             (-12345, top), (60000, top)]
    rng = np.random.default_rng(20)
    x = np.zeros((len(pairs) // 4, 128))
    for i, (lo, hi) in enumerate(pairs):
        g = x[i // 4, 32 * (i % 4):32 * (i % 4) + 32]
        g[:] = rng.uniform(lo, hi, 32)
        g[5], g[17] = lo, hi
    x = x.astype(np.float16)
    for token in x:
        kc, vc = qe.kv4_cache(1, 4), qe.kv4_cache(1, 4)
        row = token[None]
        _append(qe, np.zeros_like(row), row, row, [None] * 3, (kc, vc), 0, None, 4, 0)  # position 0: no rotation
        for cache in (kc, vc):
            got, want = host(cache)[0, 0], token.astype(np.float64)
            _, scale, low = ref.parts(got)
            with np.errstate(over="ignore"):
                off = np.abs(ref.values(got) - want).reshape(4, 32)
            # the scale: rounded by 2^-11, then up to 2^-10 less; 15 of it leave 45 * 2^-11 of a step. low and the
            # value itself are rounded by 2^-11 of 65504 each.
            assert np.all(off <= scale[:, None] * (0.5 + 45 * 2.0 ** -11) + 2 * 32), (off.max(-1), scale, low)


# ---- unpack ----------------------------------------------------------------------------
@pytest.mark.parametrize("nkv,ms,row0,n", [(1, 1, 0, 1), (2, 40, 3, 17), (5, 100, 0, 100), (3, 33, 32, 1)])
def test_unpack_is_exact(qe, nkv, ms, row0, n):
    rng = np.random.default_rng(ms)
    rows = rng.integers(0, 256, (2, nkv, ms, 80), dtype=np.uint8)
    par = rows[..., 64:].view(np.float16)
    par[~np.isfinite(par)] = 1.5
    ok, ov = (torch.full((nkv, n, 128), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    qe.launch_kv4_unpack(dev(rows[0]), dev(rows[1]), ok, ov, row0, n, num_kv_heads=nkv, max_seq_len=ms)
    for got, r in ((ok, rows[0]), (ov, rows[1])):
        with np.errstate(over="ignore"):
            want = ref.values(r[:, row0:row0 + n]).astype(np.float16)
        assert np.array_equal(host(got), want)
    only = torch.empty_like(ok)
    qe.launch_kv4_unpack(None, dev(rows[1]), None, only, row0, n, num_kv_heads=nkv, max_seq_len=ms)
    assert np.array_equal(host(only), host(ov))


# ---- attention ---------------------------------------------------------------------------
def _cache(rng, nkv, ms, live):
    """Rows in use, and rubbish with infinities and NaN behind them."""
    kv = np.full((2, nkv, ms, 80), 0xFF, np.uint8)
    kv[0, :, :live] = ref.random_rows(rng, nkv, live)
    kv[1, :, :live] = ref.random_rows(rng, nkv, live, offset=0.2)
    return kv


def _check(qe, kv, q, T, nq, pos, gone, ms, got, lse=None, w_in=None, w_out=None, what=""):
    nkv, group = kv.shape[1], nq // kv.shape[1]
    q = q.astype(np.float64).reshape(T, nkv, group, 128)
    got = got.astype(np.float64).reshape(T, nkv, group, 128)
    for h in range(nkv):
        base = max(pos - gone[h], 0)
        ctx = min(base + T, ms)
        last = np.minimum(base + np.arange(T), ms - 1).repeat(group)
        k, v = (ref.values(kv[i, h, :ctx]) for i in range(2))
        out, p, log_sum, tol, rel = ref.attention(q[:, h].reshape(-1, 128), k, v, last)
        err = np.abs(got[:, h].reshape(-1, 128) - out)
        assert np.all(err <= tol), f"{what} head {h}: {np.max(err / tol)} of the tolerance"
        if lse is not None:
            e = np.abs(lse.reshape(T, nkv, group)[:, h].reshape(-1) - log_sum)
            assert np.all(e <= rel[:, 0] + 2.0 ** -22 * np.abs(log_sum) + 2.0 ** -20), e.max()
        if w_out is not None:
            was = np.zeros(ctx) if w_in is None else w_in[h, :ctx].astype(np.float64).copy()
            was[base:] = 0
            want = was + p.sum(0)
            e = np.abs(w_out[h, :ctx] - want)
            # the weights' own tolerance; with row sums of the chunk, the log sum's rounding once more
            limit = (p * (rel + 2.0 ** -18 + 2.0 ** -22 * np.abs(log_sum[:, None]))).sum(0) + 2.0 ** -23 * want + 1e-12
            assert np.all(e <= limit), f"{what} head {h} weights: {np.max(e / limit)} of the tolerance"


def _decode(qe, kv, q, nq, pos, gone, ms, weights=None, w_in=None, q8=False, stream=None, ws=None):
    nkv = kv.shape[1]
    if ws is None:
        ws = torch.full((qe.kv4_decode_workspace_bytes(nq, ms, weights is not None),), 0xFF, dtype=torch.uint8, device="cuda")
    out = empty(nq * 128, torch.float16)
    extra = [empty(nq * 128, torch.int8), empty(nq, torch.float32), empty(nq * 16, torch.int32)] if q8 else [None] * 3
    qe.launch_attention_gqa_flash_decode_kv4(dev(q), dev(kv[0]), dev(kv[1]), ws, out, _ctl(pos),
                                             None if gone is None else _i32(*gone), stream, nq, nkv, max_seq_len=ms,
                                             out_q8=extra[0], out_scale=extra[1], out_sum8=extra[2],
                                             key_weights_in=w_in, key_weights_out=weights)
    return (host(out), *[host(x) for x in extra]) if q8 else host(out)


@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 161, 300, 1000, 4097, 20001])
@pytest.mark.parametrize("nq,nkv", [(12, 2), (4, 4), (7, 1)])
def test_decode_lengths(qe, ctx, nq, nkv):
    rng = np.random.default_rng(ctx + nq)
    ms = ctx + 3
    kv = _cache(rng, nkv, ms, ctx)
    q = (1.5 * rng.standard_normal(nq * 128)).astype(np.float16)
    w_in = rng.random((nkv, ms), np.float32)
    w = dev(np.full((nkv, ms), -7, np.float32))
    got = _decode(qe, kv, q, nq, ctx + 4, [5] * nkv, ms, weights=w, w_in=dev(w_in))
    w = host(w)
    assert np.all(w[:, ctx:] == -7)
    _check(qe, kv, q, 1, nq, ctx + 4, [5] * nkv, ms, got, w_in=w_in, w_out=w)
    # without the weights: the same bits
    assert np.array_equal(_decode(qe, kv, q, nq, ctx - 1, None, ms), got)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (2, 1), (16, 1), (17, 1), (64, 1), (33, 3), (40, 40), (64, 8), (128, 64)])
@pytest.mark.parametrize("ctx,ms", [(50, 64), (700, 9000)])
def test_decode_heads(qe, nq, nkv, ctx, ms):
    rng = np.random.default_rng(nq)
    kv = _cache(rng, nkv, ms, ctx)
    q = rng.standard_normal(nq * 128).astype(np.float16)
    w = dev(np.zeros((nkv, ms), np.float32))
    got = _decode(qe, kv, q, nq, ctx - 1, None, ms, weights=w, w_in=w)
    _check(qe, kv, q, 1, nq, ctx - 1, [0] * nkv, ms, got, w_out=host(w))


@pytest.mark.parametrize("nq,nkv,ctx,ms", [(64, 1, 18000, 20000), (17, 1, 30001, 70000), (12, 2, 40000, 40000), (64, 4, 5000, 33000),
                                           (1, 1, 100, 1000000), (256, 32, 3000, 30000)])
def test_decode_long_caches(qe, nq, nkv, ctx, ms):
    """Blocks of sixteen waves, of which those without rows do nothing."""
    rng = np.random.default_rng(ctx)
    kv = np.full((2, nkv, ms, 80), 0xFF, np.uint8)
    kv[0, :, :ctx] = ref.random_rows(rng, nkv, ctx)
    kv[1, :, :ctx] = ref.random_rows(rng, nkv, ctx, offset=0.2)
    q = rng.standard_normal(nq * 128).astype(np.float16)
    w = dev(np.zeros((nkv, ms), np.float32))
    got = _decode(qe, kv, q, nq, ctx - 1, None, ms, weights=w, w_in=w)
    _check(qe, kv, q, 1, nq, ctx - 1, [0] * nkv, ms, got, w_out=host(w))


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_query_that_is_not_finite_spoils_its_own_head_only(qe, workspace, bad):
    rng = np.random.default_rng(13)
    nq, nkv, ms, T = 12, 2, 1500, 40
    kv = _cache(rng, nkv, ms, 1400)
    q = rng.standard_normal((T, nq * 128)).astype(np.float16)
    q[7, 3 * 128 + 5] = bad
    clean = q.copy()
    clean[7, 3 * 128 + 5] = 0
    for rows, run in ((q[7:8], lambda x: _decode(qe, kv, x[0], nq, 1300, None, ms).reshape(1, -1)),
                      (q, lambda x: _prefill(qe, kv, x, T, nq, 1300, None, ms)[0])):
        at = 0 if len(rows) == 1 else 7
        got, want = run(rows), run(clean[7:8] if len(rows) == 1 else clean)
        assert np.all(np.isnan(got[at, 3 * 128:4 * 128]))
        got[at, 3 * 128:4 * 128] = want[at, 3 * 128:4 * 128]
        assert np.array_equal(got, want)


def test_two_streams_at_once(qe):
    """Launches with workspaces of their own do not disturb each other."""
    rng = np.random.default_rng(14)
    nq, nkv, ms = 12, 2, 30000
    kv = _cache(rng, nkv, ms, 20000)
    dk, dv = dev(kv[0]), dev(kv[1])
    qs = [dev(rng.standard_normal(nq * 128).astype(np.float16)) for _ in range(2)]
    ctls = [_ctl(19000), _ctl(700)]
    n = qe.kv4_decode_workspace_bytes(nq, ms, True)
    ws = [empty(n, torch.uint8) for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def run(i, stream, out, w):
        qe.launch_attention_gqa_flash_decode_kv4(qs[i], dk, dv, ws[i], out, ctls[i], None, stream, nq, nkv, max_seq_len=ms,
                                                 key_weights_out=w)

    alone = []
    for i in range(2):
        out, w = empty(nq * 128, torch.float16), torch.zeros((nkv, ms), device="cuda")
        run(i, None, out, w)
        alone.append((host(out), host(w)))
    outs = [[(empty(nq * 128, torch.float16), torch.zeros((nkv, ms), device="cuda")) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    for k in range(20):
        for i in range(2):
            run(i, streams[i], *outs[i][k])
    torch.cuda.synchronize()
    for i in range(2):
        for out, w in outs[i]:
            assert np.array_equal(host(out), alone[i][0]) and np.array_equal(host(w), alone[i][1])


def test_decode_heads_of_different_lengths_and_a_full_cache(qe):
    rng = np.random.default_rng(8)
    nq, nkv, ms, pos = 8, 4, 300, 310
    gone = [310, 200, 11, 2]  # 1 row, 111, exactly full, beyond (the token is not stored)
    kv = _cache(rng, nkv, ms, ms)
    q = rng.standard_normal(nq * 128).astype(np.float16)
    w_in = rng.random((nkv, ms), np.float32)
    w = dev(w_in)
    got = _decode(qe, kv, q, nq, pos, gone, ms, weights=w, w_in=w)
    w = host(w)
    _check(qe, kv, q, 1, nq, pos, gone, ms, got, w_in=w_in, w_out=w)
    assert np.array_equal(w[0, 1:], w_in[0, 1:]) and np.array_equal(w[1, 111:], w_in[1, 111:])


def test_decode_poison_reaches_those_who_see_it(qe):
    rng = np.random.default_rng(9)
    nq, nkv, ms = 12, 2, 500
    kv = _cache(rng, nkv, ms, 400)
    kv[0, 1, 399, 64:] = np.frombuffer(np.full(8, 0x7E00, np.uint16).tobytes(), np.uint8)
    q = rng.standard_normal(nq * 128).astype(np.float16)
    _check(qe, kv, q, 1, nq, 398, [0, 0], ms, _decode(qe, kv, q, nq, 398, None, ms))
    got = _decode(qe, kv, q, nq, 399, None, ms).reshape(nq, 128)
    assert np.all(np.isfinite(got[:6])) and np.all(np.isnan(got[6:]))
    # a cache of poison only
    kv[0, :, :, 64:] = kv[0, 1, 399, 64:]
    w = dev(np.zeros((nkv, ms), np.float32))
    assert np.all(np.isnan(_decode(qe, kv, q, nq, 200, None, ms, weights=w)))
    assert np.all(np.isnan(host(w)[:, :201])) and np.all(host(w)[:, 201:] == 0)


def test_decode_q8_epilogue(qe):
    rng = np.random.default_rng(10)
    nq, nkv, ms = 12, 2, 2000
    kv = _cache(rng, nkv, ms, 1500)
    q = rng.standard_normal(nq * 128).astype(np.float16)
    out, q8, scale, sum8 = _decode(qe, kv, q, nq, 1499, None, ms, q8=True)
    o = out.astype(np.float64).reshape(nq, 128)
    # the head's largest value is known to half a step of fp16
    assert np.all(np.abs(scale - np.abs(o).max(-1) / 127) <= (2.0 ** -11 + 2.0 ** -22) * scale)
    assert np.all(np.abs(q8.reshape(nq, 128) - o / scale[:, None]) <= 0.5 + 127 * (2.0 ** -11 + 2.0 ** -22))
    assert np.array_equal(sum8.reshape(nq, 16), -8 * q8.reshape(nq, 16, 8).astype(np.int32).sum(-1))


def test_decode_large_scores(qe):
    """Scores of hundreds: one row takes everything, and no difference overflows."""
    rng = np.random.default_rng(11)
    nq, nkv, ms = 4, 2, 1000
    kv = _cache(rng, nkv, ms, 1000)
    kv[0, :, :] = ref.random_rows(rng, nkv, ms, spread=30.0, offset=40.0)
    q = (8 * rng.standard_normal(nq * 128)).astype(np.float16)
    _check(qe, kv, q, 1, nq, 999, [0, 0], ms, _decode(qe, kv, q, nq, 999, None, ms))


def test_decode_offsets_past_32_bits(qe):
    """A head whose rows begin more than 2^32 bytes into the cache, and a row as far into its head."""
    rng = np.random.default_rng(12)
    ctx = 300
    rows = ref.random_rows(rng, 2, ctx)
    q = rng.standard_normal(128).astype(np.float16)
    for nkv, ms, first in ((9, 6_800_000, 0), (1, 54_000_000, 53_999_700)):
        assert ((nkv - 1) * ms + first) * 80 > 2 ** 32
        caches = [torch.zeros(nkv * ms * 80, dtype=torch.uint8, device="cuda") for _ in range(2)]
        for c, r in zip(caches, rows):
            c.view(nkv, ms, 80)[nkv - 1, first:first + ctx] = dev(r)
        nq = nkv
        qs = np.zeros((nq, 128), np.float16)
        qs[-1] = q
        out = empty(nq * 128, torch.float16)
        pos = first + ctx - 1
        if first:  # the rows before give a score of 0 and V of 0: make them count for nothing
            qs[-1] *= np.float16(8)
        ws = empty(qe.kv4_decode_workspace_bytes(nq, ms), torch.uint8)
        qe.launch_attention_gqa_flash_decode_kv4(dev(qs.reshape(-1)), caches[0], caches[1], ws, out, _ctl(pos), None,
                                                 None, nq, nkv, max_seq_len=ms)
        got = host(out).reshape(nq, 128)[-1].astype(np.float64)
        k, v = ref.values(rows[0]), ref.values(rows[1])
        s = (qs[-1].astype(np.float64) @ k.T) / np.sqrt(128)
        m = max(s.max(), 0.0) if first else s.max()
        e = np.exp(s - m)
        total = e.sum() + first * np.exp(-m)
        p = e / total
        # as in kv4_reference.attention, from these inputs' own sums: p is off by 2 d + 2^-19 and rounded to fp16
        d = 2.0 ** -20 * (np.abs(qs[-1].astype(np.float64)) @ np.abs(k).T).max() / np.sqrt(128)
        tol = 2.0 ** -11 * np.abs(p @ v) + (2.0 ** -11 + 2 * d + 2.0 ** -19) * (p @ np.abs(v)) + 2.0 ** -24
        assert np.all(np.abs(got - p @ v) <= tol)
        assert not first or np.abs(got).max() > 0.05
        del caches
        torch.cuda.empty_cache()


def _prefill(qe, kv, q, T, nq, pos, gone, ms, hidden=None, weights=None, w_in=None, lse=False):
    nkv = kv.shape[1]
    hidden = hidden or nq * 128
    out = torch.full((T, hidden), 77.0, dtype=torch.float16, device="cuda")
    row_lse = empty((T, nq), torch.float32) if lse or weights is not None else None
    qe.launch_attention_gqa_prefill_kv4(dev(q), dev(kv[0]), dev(kv[1]), out, _ctl(pos),
                                        None if gone is None else _i32(*gone), T, num_q_heads=nq, num_kv_heads=nkv,
                                        max_seq_len=ms, hidden_size=hidden, key_weights_in=w_in, key_weights_out=weights,
                                        row_lse=row_lse)
    out = host(out)
    assert np.all(out[:, nq * 128:] == 77)
    return out[:, :nq * 128], (None if row_lse is None else host(row_lse))


@pytest.mark.parametrize("T,base,nq,nkv", [
    (1, 0, 12, 2), (1, 500, 12, 2), (2, 63, 12, 2), (17, 0, 12, 2), (21, 64, 6, 1), (22, 1, 12, 2), (64, 0, 4, 4),
    (65, 1000, 7, 1), (100, 37, 1, 1), (128, 129, 8, 2), (333, 0, 12, 2), (200, 2000, 12, 2), (43, 5000, 12, 2),
    (9, 30, 64, 1), (300, 700, 16, 8)])
@pytest.mark.parametrize("split", [False, True])
def test_prefill(qe, T, base, nq, nkv, split):
    rng = np.random.default_rng(T + base)
    ms = max(base + T + 2, 1100)
    kv = _cache(rng, nkv, ms, base + T)
    q = (1.5 * rng.standard_normal((T, nq * 128))).astype(np.float16)
    w_in = rng.random((nkv, ms), np.float32)
    if split:
        qe.gemm_reserve_workspace()
    try:
        w = dev(np.full((nkv, ms), -7, np.float32))
        got, lse = _prefill(qe, kv, q, T, nq, base + 9, [9] * nkv, ms, nq * 128 + 64, weights=w, w_in=dev(w_in))
        again, _ = _prefill(qe, kv, q, T, nq, base, None, ms)
    finally:
        qe.gemm_release_workspace()
    w = host(w)
    assert np.all(w[:, base + T:] == -7)
    _check(qe, kv, q, T, nq, base + 9, [9] * nkv, ms, got, lse, w_in, w)
    assert np.array_equal(got, again)


def test_prefill_heads_of_different_lengths_and_a_full_cache(qe, workspace):
    rng = np.random.default_rng(21)
    T, nq, nkv, ms, pos = 50, 8, 4, 1200, 1230
    gone = [1230, 600, 80, 10]  # from row 0; 630; exactly full; 30 tokens and more find no room
    kv = _cache(rng, nkv, ms, ms)
    q = rng.standard_normal((T, nq * 128)).astype(np.float16)
    w_in = rng.random((nkv, ms), np.float32)
    w = dev(w_in)
    got, lse = _prefill(qe, kv, q, T, nq, pos, gone, ms, weights=w, w_in=w)
    _check(qe, kv, q, T, nq, pos, gone, ms, got, lse, w_in, host(w))


@pytest.mark.parametrize("T", [20, 150])
def test_prefill_poison_of_a_later_token(qe, workspace, T):
    """A token with an infinity, stored as the append stores it: rows before it are exact, rows from it on NaN."""
    rng = np.random.default_rng(22)
    nq, nkv, ms, base, at = 12, 2, 1500, 1000, 13
    kv = _cache(rng, nkv, ms, base + T)
    kv[0, :, base + at, 64:] = np.frombuffer(np.full(8, 0x7E00, np.uint16).tobytes(), np.uint8)
    kv[1, :, base + at] = 0
    q = rng.standard_normal((T, nq * 128)).astype(np.float16)
    got, lse = _prefill(qe, kv, q, T, nq, base, None, ms, lse=True)
    assert np.all(np.isnan(got[at:])) and np.all(np.isnan(lse[at:]))
    _check(qe, kv, q[:at], at, nq, base, [0, 0], ms, got[:at], lse[:at])


def test_prefill_recorded_into_a_graph(qe, workspace):
    """Replayed with other positions and other rows, between eager launches that use the workspace."""
    rng = np.random.default_rng(23)
    T, nq, nkv, ms = 30, 12, 2, 2048
    kv = _cache(rng, nkv, ms, ms)
    q = rng.standard_normal((T, nq * 128)).astype(np.float16)
    dk, dv, dq, ctl, gone = dev(kv[0]), dev(kv[1]), dev(q), _ctl(0), _i32(0, 0)
    out, lse, w = empty((T, nq * 128), torch.float16), empty((T, nq), torch.float32), empty((nkv, ms), torch.float32)
    args = dict(num_q_heads=nq, num_kv_heads=nkv, max_seq_len=ms, hidden_size=nq * 128)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        qe.launch_attention_gqa_prefill_kv4(dq, dk, dv, out, ctl, gone, T, key_weights_out=w, row_lse=lse, **args)
    for pos, lost in ((0, (0, 0)), (1500, (3, 700)), (40, (40, 1)), (1900, (0, 900))):
        ctl.copy_(_ctl(pos)), gone.copy_(_i32(*lost))
        w.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check(qe, kv, q, T, nq, pos, list(lost), ms, host(out), host(lse), None, host(w), what=f"replay at {pos}")
        _prefill(qe, kv, q, T, nq, 1000, None, ms)


# ---- eviction ------------------------------------------------------------------------------
def _kept(w, n, keep, sinks, recent):
    if n <= keep:
        return np.arange(n)
    rank = np.where(np.isnan(w[:n]), -np.inf, w[:n]).astype(np.float64)
    # NaN below everything, -inf too
    rank = np.where(np.isnan(w[:n]), -1e300, np.where(np.isneginf(rank), -1e299, rank))
    mid = np.arange(sinks, n - recent)
    c = keep - sinks - recent
    best = mid[np.argsort(-rank[mid], kind="stable")][:c]
    return np.sort(np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)]))


def _evict(qe, kv, w, pos, gone, keep, sinks, recent, ms, in_place):
    nkv = w.shape[0]
    dk, dv, dw, dg = dev(kv[0]), dev(kv[1]), dev(w), _i32(*gone)
    kept = torch.full((nkv, keep), 99, dtype=torch.int32, device="cuda")
    if in_place:
        ok, ov, ow, og = dk, dv, dw, dg
    else:
        ok, ov, ow, og = torch.zeros_like(dk), torch.zeros_like(dv), torch.full_like(dw, -3), torch.zeros_like(dg)
    qe.launch_kv4_evict(dk, dv, dw, dg, ok, ov, ow, og, kept, _ctl(pos), keep, sinks, recent, num_kv_heads=nkv,
                        max_seq_len=ms)
    return [host(x) for x in (ok, ov, ow, og, kept)]


def _check_evict(kv, w, pos, gone, keep, sinks, recent, ms, got):
    ok, ov, ow, og, kept = got
    for h in range(w.shape[0]):
        n = min(max(pos - gone[h], 0), ms)
        want = _kept(w[h], n, keep, sinks, recent)
        m = want.size
        assert np.array_equal(kept[h, :m], want) and np.all(kept[h, m:] == -1), h
        assert np.array_equal(ok[h, :m], kv[0, h, want]) and np.array_equal(ov[h, :m], kv[1, h, want])
        assert np.array_equal(ow[h, :m].view(np.uint32), w[h, want].view(np.uint32)) and np.all(ow[h, m:n] == 0)
        assert og[h] == (pos - m if n else gone[h])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,keep,sinks,recent", [
    (1, 1, 0, 0), (2, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (10, 20, 4, 8), (20, 20, 4, 8), (21, 20, 4, 8), (100, 7, 3, 4),
    (100, 99, 0, 0), (1000, 500, 4, 100), (1025, 64, 0, 64), (4097, 4096, 1, 1), (5000, 4300, 4, 512), (9000, 100, 4, 3),
    (32768, 20000, 4, 10000), (40000, 9000, 4, 700)])
def test_evict(qe, n, keep, sinks, recent, in_place):
    rng = np.random.default_rng(n + keep)
    nkv, ms = 3, n + 6
    keep = min(keep, ms)
    kv = rng.integers(0, 256, (2, nkv, ms, 80), dtype=np.uint8)
    w = np.exp(2 * rng.standard_normal((nkv, ms))).astype(np.float32)
    w[1] = rng.integers(0, 3, ms)  # ties
    w[2] = 0.25                    # nothing but ties
    got = _evict(qe, kv, w, n + 11, [11] * nkv, keep, sinks, recent, ms, in_place)
    _check_evict(kv, w, n + 11, [11] * nkv, keep, sinks, recent, ms, got)


@pytest.mark.parametrize("n,keep,sinks,recent", [(32769, 32768, 0, 0), (33793, 1, 1, 0), (49153, 20000, 300, 1500),
                                                 (70001, 123, 4, 100), (131000, 65000, 4, 40000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_more_rows_than_lds_holds(qe, n, keep, sinks, recent, in_place):
    test_evict(qe, n, keep, sinks, recent, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_odd_weights_and_heads_of_their_own(qe, in_place):
    """NaN, infinities, negative weights, zeros of both signs, subnormals; heads with other lengths, none, and full ones."""
    rng = np.random.default_rng(31)
    nkv, ms, pos = 5, 700, 1000
    odd = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-40, -1e-40, 3.4e38, -1.0, 1.0], np.float32)
    w = odd[rng.integers(0, odd.size, (nkv, ms))]
    w[3] = np.nan
    gone = [500, 301, 998, 400, 100]  # 500 rows, 699, 2, 600, and more than there is room for
    kv = rng.integers(0, 256, (2, nkv, ms, 80), dtype=np.uint8)
    got = _evict(qe, kv, w, pos, gone, 333, 2, 50, ms, in_place)
    _check_evict(kv, w, pos, gone, 333, 2, 50, ms, got)
    # nothing yet
    got = _evict(qe, kv, w, 0, [0] * nkv, 333, 2, 50, ms, in_place)
    _check_evict(kv, w, 0, [0] * nkv, 333, 2, 50, ms, got)


# ---- together ---------------------------------------------------------------------------------
def _session(qe, rng, nq, nkv, ms, steps, budget, check_every):
    """Chunks, tokens and evictions of one layer, followed in numpy from the caches' own bytes: what each launch wrote
    is checked against what it read."""
    q_dim, kv_dim = nq * 128, nkv * 128
    kc, vc = qe.kv4_cache(nkv, ms), qe.kv4_cache(nkv, ms)
    w, gone = torch.zeros((nkv, ms), dtype=torch.float32, device="cuda"), _i32(*[0] * nkv)
    kept = empty((nkv, budget), torch.int32)
    ws = empty(qe.kv4_decode_workspace_bytes(nq, ms, True), torch.uint8)
    pos = 0
    for i, T in enumerate(steps):
        if T == "evict":
            before = [host(x).copy() for x in (kc, vc, w, gone)]
            qe.launch_kv4_evict(kc, vc, w, gone, kc, vc, w, gone, kept, _ctl(pos), budget, 2, 16, num_kv_heads=nkv,
                                max_seq_len=ms)
            _check_evict(np.stack(before[:2]), before[2], pos, before[3], budget, 2, 16, ms,
                         [host(x) for x in (kc, vc, w, gone, kept)])
            continue
        q, k, v = (rng.standard_normal((T, n)).astype(np.float16) for n in (q_dim, kv_dim, kv_dim))
        dq, out = dev(q), empty((T, q_dim), torch.float16)
        ctl = _ctl(pos)
        old_w, lost = host(w).copy(), list(host(gone))
        qe.launch_qkv_bias_rope_kv4_append(dq, dq, dev(k), dev(v), None, None, None, kc, vc, ctl, gone, T,
                                           num_q_heads=nq, num_kv_heads=nkv, max_seq_len=ms)
        if T == 1:
            qe.launch_attention_gqa_flash_decode_kv4(dq, kc, vc, ws, out, ctl, gone, None, nq, nkv, max_seq_len=ms,
                                                     key_weights_in=w, key_weights_out=w)
            lse = None
        else:
            lse = empty((T, nq), torch.float32)
            qe.launch_attention_gqa_prefill_kv4(dq, kc, vc, out, ctl, gone, T, num_q_heads=nq, num_kv_heads=nkv,
                                                max_seq_len=ms, hidden_size=q_dim, key_weights_in=w, key_weights_out=w,
                                                row_lse=lse)
        if i % check_every == 0 or T > 1:
            kv = np.stack([host(kc), host(vc)])
            _check(qe, kv, host(dq), T, nq, pos, lost, ms, host(out), None if lse is None else host(lse), old_w, host(w),
                   what=f"step {i}")
        pos += T
    return pos, host(gone)


def test_a_bounded_session(qe, workspace):
    rng = np.random.default_rng(41)
    steps = [300, 40] + [1] * 5 + ["evict"] + [1] * 70 + [33] + ["evict"] + [1] * 20 + ["evict", 90, "evict", 1, 1]
    pos, gone = _session(qe, rng, 12, 2, 400, steps, 256, 10)
    assert pos == 300 + 40 + 5 + 70 + 33 + 20 + 90 + 2 and np.all(gone == pos - 2 - 256)


def test_a_decode_step_replayed_from_a_graph_on_another_stream(qe):
    """Append, attention with weights and the advance of the position in one graph; eager eviction between replays."""
    rng = np.random.default_rng(42)
    nq, nkv, ms, keep = 12, 2, 160, 96
    q_dim = nq * 128
    src = [torch.zeros((1, n * 128), dtype=torch.float16, device="cuda") for n in (nq, nkv, nkv)]
    logits = torch.zeros(64, dtype=torch.float16, device="cuda")

    def state():
        return dict(kc=qe.kv4_cache(nkv, ms), vc=qe.kv4_cache(nkv, ms), w=torch.zeros((nkv, ms), device="cuda"),
                    gone=_i32(0, 0), ctl=_ctl(0), q=empty((1, q_dim), torch.float16), out=empty((1, q_dim), torch.float16),
                    ws=empty(qe.kv4_decode_workspace_bytes(nq, ms, True), torch.uint8), kept=empty((nkv, keep), torch.int32),
                    val=empty(256, torch.float32), idx=empty(256, torch.int32))

    def step(s):
        qe.launch_qkv_bias_rope_kv4_append(src[0], s["q"], src[1], src[2], None, None, None, s["kc"], s["vc"], s["ctl"],
                                           s["gone"], 1, max_seq_len=ms)
        qe.launch_attention_gqa_flash_decode_kv4(s["q"], s["kc"], s["vc"], s["ws"], s["out"], s["ctl"], s["gone"],
                                                 max_seq_len=ms, key_weights_in=s["w"], key_weights_out=s["w"])
        qe.launch_sample_and_advance(logits, s["val"], s["idx"], s["ctl"], None, vocab_size=64)

    a, b = state(), state()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(a)
    for x, y in zip(a.values(), state().values()):
        x.copy_(y)
    torch.cuda.synchronize()
    for i in range(230):
        for x in src:
            x.copy_(dev(rng.standard_normal(x.shape).astype(np.float16)))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        step(b)
        torch.cuda.synchronize()
        assert all(torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)) for k in ("out", "w", "gone", "ctl", "kc")), i
        if i in (120, 150, 200):
            for s in (a, b):
                qe.launch_kv4_evict(s["kc"], s["vc"], s["w"], s["gone"], s["kc"], s["vc"], s["w"], s["gone"], s["kept"],
                                    s["ctl"], keep, 4, 30, max_seq_len=ms)
            assert np.all(host(b["gone"]) == i + 1 - keep)
    assert np.all(np.isfinite(host(a["out"])))
