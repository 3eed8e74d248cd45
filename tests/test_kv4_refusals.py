"""What the 4-bit cache and log probability entry points refuse, decided on the
host before any HIP call (no GPU needed), and their workspace sizes."""
import ctypes

import pytest

P = 0x100000  # an aligned address; nothing is launched
F = ctypes.c_float(1e6)


@pytest.fixture(scope="module")
def L():
    import qe_amd
    return qe_amd.lib()


def _says(L, rc, text, code=1):
    assert rc == code and text in L.qe_last_error().decode(), (rc, L.qe_last_error())


def _append(L, q=P, q_out=None, k=P, v=P, qb=None, kc=P, vc=P, T=1, nq=12, nkv=2, hd=128, ms=64, rot=0, theta=1e6):
    return L.qe_launch_qkv_bias_rope_kv4_append(q, q if q_out is None else q_out, k, v, qb, None, None, kc, vc, None,
                                                None, T, None, nq, nkv, hd, ms, rot, ctypes.c_float(theta))


def test_append(L):
    for bad in ({"q": None}, {"k": None}, {"v": None}, {"kc": None}, {"vc": None}):
        _says(L, _append(L, **bad), "NULL")
    for bad, text in (({"hd": 64}, "head_dim"), ({"nkv": 0}, "num_kv_heads"), ({"nq": 0}, "num_q_heads"),
                      ({"ms": 0}, "max_seq_len"), ({"rot": 24}, "rotary_dim"), ({"rot": 144}, "rotary_dim"),
                      ({"rot": -16}, "rotary_dim"), ({"theta": 0.0}, "rope_theta"), ({"theta": -1.0}, "rope_theta"),
                      ({"theta": float("nan")}, "rope_theta"), ({"theta": float("inf")}, "rope_theta"),
                      ({"kc": P + 8}, "aligned"), ({"vc": P + 4}, "aligned"), ({"q": P + 2}, "aligned"),
                      ({"k": P + 8}, "aligned"), ({"qb": P + 2}, "aligned"), ({"q_out": P + 256}, "overlaps")):
        _says(L, _append(L, **bad), text)
    assert _append(L, T=0) == 0 and _append(L, T=-3) == 0


def test_unpack(L):
    def unpack(kc=P, vc=P, ok=P, ov=P, r0=0, n=1, nkv=2, hd=128, ms=64):
        return L.qe_launch_kv4_unpack(kc, vc, ok, ov, r0, n, None, nkv, hd, ms)
    for bad in ({"ok": None}, {"kc": None}, {"ov": None}, {"kc": None, "ok": None, "vc": None, "ov": None}):
        _says(L, unpack(**bad), "together")
    for bad, text in (({"r0": -1}, "rows"), ({"r0": 64}, "rows"), ({"r0": 60, "n": 5}, "rows"), ({"n": 65}, "rows"),
                      ({"ok": P + 8}, "aligned"), ({"hd": 64}, "head_dim"), ({"kc": P + 4}, "aligned"),
                      ({"nkv": 65536}, "num_kv_heads"), ({"r0": 2**31 - 1, "n": 2**31 - 1}, "rows")):
        _says(L, unpack(**bad), text)
    assert unpack(n=0) == 0


def test_decode(L):
    def decode(q=P, kc=P, vc=P, ws=P, out=P, nq=12, nkv=2, hd=128, ms=64, w_in=None, w_out=None):
        return L.qe_launch_attention_gqa_flash_decode_kv4(q, kc, vc, ws, out, None, None, None, nq, nkv, hd, ms, None,
                                                          None, None, w_in, w_out)
    for bad in ({"q": None}, {"kc": None}, {"vc": None}, {"ws": None}, {"out": None}):
        _says(L, decode(**bad), "NULL")
    for bad, text in (({"nq": 13}, "13 q heads"), ({"nq": 0}, "q heads"), ({"nq": 130}, "at most 64"),
                      ({"nkv": -1}, "num_kv_heads"), ({"hd": 64}, "head_dim"), ({"ms": 0}, "max_seq_len"),
                      ({"q": P + 8}, "aligned"), ({"ws": P + 4}, "aligned"), ({"kc": P + 1}, "aligned"),
                      ({"w_in": P}, "key_weights_in without"), ({"ms": 2**31 - 1}, "max_seq_len")):
        _says(L, decode(**bad), text)


def test_prefill(L):
    def prefill(q=P, kc=P, vc=P, out=P, T=1, nq=12, nkv=2, hd=128, ms=64, hs=1536, w_in=None, w_out=None, lse=None):
        return L.qe_launch_attention_gqa_prefill_kv4(q, kc, vc, out, None, None, T, None, nq, nkv, hd, ms, hs, w_in,
                                                     w_out, lse)
    for bad in ({"q": None}, {"kc": None}, {"vc": None}, {"out": None}):
        _says(L, prefill(**bad), "NULL")
    for bad, text in (({"nq": 13}, "13 q heads"), ({"nq": 130, "hs": 130 * 128}, "at most 64"), ({"hd": 64}, "head_dim"),
                      ({"hs": 1535}, "hidden_size"), ({"hs": 1538}, "hidden_size"), ({"w_in": P}, "without"),
                      ({"w_out": P}, "row_lse"), ({"w_out": P, "lse": P}, "attn_out overlaps q"),
                      ({"w_out": P, "lse": P, "out": P + 4 * 1536 - 8, "T": 2}, "attn_out overlaps q"),
                      ({"w_out": P, "lse": P, "q": P + 7056, "T": 2, "hs": 2000}, "attn_out overlaps q"),
                      ({"out": P + 4}, "aligned"), ({"q": P + 8}, "aligned"),
                      ({"T": 2**31 - 1}, "num_tokens"), ({"ms": 2**30}, "max_seq_len")):
        _says(L, prefill(**bad), text)
    assert prefill(T=0) == 0


def test_evict(L):
    big = 0x10000000

    def evict(kc=P, vc=2 * P, w=3 * P, ok=None, ov=None, ow=None, oe=4 * P, kept=5 * P, ctl=6 * P, keep=32, sinks=4,
              recent=8, nkv=2, hd=128, ms=64):
        return L.qe_launch_kv4_evict(kc, vc, w, None, ok or kc, ov or vc, ow or w, oe, kept, ctl, keep, sinks, recent,
                                     None, nkv, hd, ms)
    for bad in ({"kc": None}, {"vc": None}, {"w": None}, {"oe": None}, {"kept": None}, {"ctl": None}):
        _says(L, evict(**bad), "NULL")
    for bad, text in (({"keep": 0}, "keep"), ({"keep": 65}, "keep"), ({"sinks": -1}, "sinks"), ({"recent": -1}, "recent"),
                      ({"sinks": 20, "recent": 13}, "do not fit"), ({"sinks": 2**31 - 1}, "do not fit"),
                      ({"ok": big}, "all in place"), ({"ov": big}, "all in place"), ({"ow": big}, "all in place"),
                      ({"ok": P + 16, "ov": big, "ow": 2 * big}, "overlaps"),
                      ({"ok": big, "ov": 2 * P + 80 * 64, "ow": 2 * big}, "overlaps"),
                      ({"ok": big, "ov": 2 * big, "ow": 3 * P + 4}, "overlaps"),
                      ({"ok": big + 8}, "aligned"), ({"hd": 96}, "head_dim"), ({"nkv": 65536}, "num_kv_heads")):
        _says(L, evict(**bad), text)


def test_logprobs(L):
    def lp(x=P, ids=P, out=P, ent=None, tl=None, ti=None, ws=P, rows=2, vocab=100, stride=100, top=0):
        return L.qe_launch_token_logprobs(x, ids, out, ent, tl, ti, ws, rows, vocab, ctypes.c_longlong(stride), top, None)
    for bad, text in (({"x": None}, "NULL"), ({"ws": None}, "NULL"), ({"ids": None}, "together"), ({"out": None}, "together"),
                      ({"vocab": 0}, "vocab_size"), ({"vocab": 2**31 - 1, "stride": 2**31}, "vocab_size"),
                      ({"stride": 99}, "row_stride"), ({"top": -1}, "top_k"), ({"top": 33, "ti": P}, "top_k"),
                      ({"top": 20, "ti": P, "vocab": 19}, "top_k"), ({"top": 4}, "without an output"),
                      ({"ti": P}, "top_k=0"), ({"x": P + 1}, "alignment"), ({"rows": 2**30, "vocab": 2**20, "stride": 2**20}, "num_rows")):
        _says(L, lp(**bad), text)
    assert lp(rows=0) == 0


def test_workspace_sizes(L):
    import qe_amd
    assert qe_amd.kv4_decode_workspace_bytes(12, 4096) == 12 * 128 * 130 * 4
    assert qe_amd.kv4_decode_workspace_bytes(12, 4095, True) == 12 * (128 * 130 + 4096) * 4
    assert qe_amd.token_logprobs_workspace_bytes(3, 151936, 20) == 3 * 19 * 23 * 4
    assert qe_amd.token_logprobs_workspace_bytes(0) == 0
    n = ctypes.c_size_t()
    _says(L, L.qe_kv4_decode_workspace_bytes(0, 64, 0, ctypes.byref(n)), "num_q_heads")
    _says(L, L.qe_kv4_decode_workspace_bytes(12, 64, 0, None), "NULL")
    _says(L, L.qe_token_logprobs_workspace_bytes(1, 0, 0, ctypes.byref(n)), "vocab_size")
    _says(L, L.qe_token_logprobs_workspace_bytes(1, 100, 33, ctypes.byref(n)), "top_k")


def test_tensors_in_host_memory():
    """The Python launchers, before the library is called."""
    import torch

    import qe_amd
    x = torch.zeros(4096, dtype=torch.uint8)
    calls = [lambda: qe_amd.launch_qkv_bias_rope_kv4_append(x, x, x, x, None, None, None, x, x, None, None, 1),
             lambda: qe_amd.launch_kv4_unpack(x, x, x, x, 0, 1), lambda: qe_amd.launch_kv4_unpack(None, x, None, x, 0, 1),
             lambda: qe_amd.launch_attention_gqa_flash_decode_kv4(x, x, x, x, x, None, None),
             lambda: qe_amd.launch_attention_gqa_prefill_kv4(x, x, x, x, None, None, 1),
             lambda: qe_amd.launch_kv4_evict(x, x, x, None, x, x, x, x, x, x, 1),
             lambda: qe_amd.launch_token_logprobs(x, None, None, x, None, None, x, 1, vocab_size=8)]
    for call in calls:
        with pytest.raises(RuntimeError, match="must be on a GPU"):
            call()
