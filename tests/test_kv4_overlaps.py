"""Buffers of the 4-bit cache calls that share memory where kernels would read what others have written: refused on
the host before any HIP call (no GPU needed)."""
import ctypes

import pytest

MB = 1 << 20


@pytest.fixture(scope="module")
def L():
    import qe_amd
    return qe_amd.lib()


def _says(L, rc, text):
    assert rc == 1 and text in L.qe_last_error().decode(), (rc, L.qe_last_error())


def test_evict(L):
    """2 heads, 64 rows: caches of 10240 bytes, weights of 512, counts of 8, kept rows of 256.  Rows, weights and counts
    are moved by blocks that do not wait for each other: no two outputs meet, and an output meets no input but its own."""
    cache, weights = 2 * 64 * 80, 2 * 64 * 4
    inputs = dict(kc=MB, vc=2 * MB, w=3 * MB, gone=4 * MB)
    apart = dict(ok=5 * MB, ov=6 * MB, ow=7 * MB, og=8 * MB, kept=9 * MB)

    def evict(**kw):
        a = {**inputs, **apart, **kw}
        return L.qe_launch_kv4_evict(a["kc"], a["vc"], a["w"], a["gone"], a["ok"], a["ov"], a["ow"], a["og"], a["kept"],
                                     10 * MB, 32, 4, 8, None, 2, 128, 64)

    in_place = dict(ok=MB, ov=2 * MB, ow=3 * MB, og=4 * MB)
    last = dict(kc=cache - 16, vc=cache - 16, w=weights - 16, gone=4, ok=cache - 16, ov=cache - 16, ow=weights - 16, og=4,
                kept=252)
    # apart: each output on another's last bytes, and on the last bytes of an input that is not its own
    for out in apart:
        for other in (*inputs, *apart):
            if other == out or (out, other) in (("ok", "kc"), ("ov", "vc"), ("ow", "w")):
                continue
            if (out, other) == ("og", "gone"):  # may be it, but not part of it
                _says(L, evict(og=inputs["gone"] + 4), "overlap")
                continue
            at = {**inputs, **apart}[other] + last[other]
            _says(L, evict(**{out: at // 16 * 16 if out in ("ok", "ov") else at}), "overlap")
    # swapped: K moves to where V comes from
    _says(L, evict(ok=2 * MB, ov=MB, ow=7 * MB), "overlap")
    # in place: one cache for both, lists and counts inside what moves
    _says(L, evict(**{**in_place, "kc": MB, "vc": MB, "ok": MB, "ov": MB}), "overlap")
    for kw in (dict(kept=MB), dict(kept=2 * MB + cache - 4), dict(kept=3 * MB), dict(kept=4 * MB + 4), dict(og=2 * MB),
               dict(og=3 * MB + weights - 4), dict(og=4 * MB + 4)):
        _says(L, evict(**{**in_place, **kw}), "overlap")


def test_append(L):
    """3 tokens, 4 q heads, 2 kv heads, 64 rows.  Heads are rotated and stored by blocks that do not wait for each other:
    q_out may be q and meets nothing else that is read, the caches meet nothing."""
    q, kv, cache, counts = 3 * 4 * 256, 3 * 2 * 256, 2 * 64 * 80, 8
    at = dict(q=MB, k=2 * MB, v=3 * MB, qb=4 * MB, kb=5 * MB, vb=6 * MB, q_out=MB, kc=7 * MB, vc=8 * MB, gone=9 * MB)
    size = dict(q=q, k=kv, v=kv, qb=4 * 256, kb=2 * 256, vb=2 * 256, q_out=q, kc=cache, vc=cache, gone=counts)

    def append(T=3, **kw):
        a = {**at, **kw}
        return L.qe_launch_qkv_bias_rope_kv4_append(a["q"], a["q_out"], a["k"], a["v"], a["qb"], a["kb"], a["vb"], a["kc"],
                                                    a["vc"], None, a["gone"], T, None, 4, 2, 128, 64, 0,
                                                    ctypes.c_float(1e6))
    for out in ("q_out", "kc", "vc"):
        for other in at:
            if other in (out, "q_out") or (out, other) == ("q_out", "q"):
                continue
            _says(L, append(**{out: at[other] + (size[other] - 1) // 16 * 16}), "overlap")
            if out != "q_out" and other != "q":
                _says(L, append(**{out: at[other] + 16 - size[out]}), "overlap")
    _says(L, append(q_out=MB + 16), "overlap")
    _says(L, append(kc=MB, vc=7 * MB), "overlap")
    assert append(T=0, kc=MB) == 0


def test_attention(L):
    """Key weights are added in place or apart, never shifted; a chunk's outputs are its q rows or apart from them (a
    block writes its rows while others still read theirs)."""
    T, nq, nkv, rows = 3, 4, 2, 64
    weights, q = nkv * rows * 4, T * nq * 256

    def decode(w_in, w_out):
        return L.qe_launch_attention_gqa_flash_decode_kv4(MB, 2 * MB, 3 * MB, 4 * MB, 6 * MB, None, None, None, nq, nkv, 128,
                                                          rows, None, None, None, w_in, w_out)

    def prefill(out=6 * MB, w_in=None, w_out=None, hidden=nq * 128, lse=5 * MB, T=T):
        return L.qe_launch_attention_gqa_prefill_kv4(MB, 2 * MB, 3 * MB, out, None, None, T, None, nq, nkv, 128, rows,
                                                     hidden, w_in, w_out, lse)
    for shift in (4, weights - 4, -4, 4 - weights):
        _says(L, decode(7 * MB, 7 * MB + shift), "overlap")
        _says(L, prefill(w_in=7 * MB, w_out=7 * MB + shift), "overlap")
    for shift in (8, 256, q - 8, -8, 8 - q):
        _says(L, prefill(out=MB + shift), "attn_out overlaps q")
    _says(L, prefill(out=MB, hidden=nq * 128 + 4), "attn_out overlaps q")
    _says(L, prefill(out=MB - 8 - (T - 1) * 2 * 1024, hidden=1024), "attn_out overlaps q")
    assert prefill(out=MB + 8, T=0) == 0


def test_unpack(L):
    """Rows come out 3.2 times as wide, by blocks that do not wait for each other: outputs meet neither cache nor each
    other."""
    cache, out = 2 * 64 * 80, 2 * 10 * 256

    def unpack(kc=MB, vc=2 * MB, ok=3 * MB, ov=4 * MB, n=10):
        return L.qe_launch_kv4_unpack(kc, vc, ok, ov, 5, n, None, 2, 128, 64)
    for kw in (dict(ok=MB), dict(ok=2 * MB + cache - 16), dict(ov=MB + 16 - out), dict(ov=2 * MB), dict(ov=3 * MB + out - 16),
               dict(kc=None, ok=None, ov=2 * MB + 16), dict(vc=None, ov=None, ok=MB + cache - 16)):
        _says(L, unpack(**kw), "overlap")
    assert unpack(ok=MB, n=0) == 0
