"""What the paged cache's entry points refuse, decided on the host before any HIP call (no GPU needed), their
workspace sizes, and the rotary tables."""
import ctypes
import math
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import launch_recorder

P = 0x10000000  # aligned addresses far apart; nothing is launched
F = ctypes.c_float


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    return qe_amd


def _says(qe, rc, text, code=1):
    assert rc == code and text in qe.lib().qe_last_error().decode(), (rc, qe.lib().qe_last_error())


def _cache(qe, k=P, v=2 * P, stride=0, pages=16, size=16, heads=2, dim=128):
    return qe._PagedCache(k, v, stride, pages, size, heads, dim)


def _batch(qe, table=3 * P, starts=None, context=3 * P + 4096, seqs=4, tokens=4, max_pages=8):
    return qe._PagedBatch(table, starts, context, seqs, tokens, max_pages)


def _at(x):
    return None if x is None else ctypes.byref(x)


BAD_CACHE = [({"k": None}, "NULL"), ({"v": None}, "NULL"), ({"dim": 64}, "head_dim"), ({"size": 8}, "page_size"),
             ({"size": 48}, "page_size"), ({"size": 512}, "page_size"), ({"size": 0}, "page_size"), ({"pages": 0}, "num_pages"),
             ({"heads": 0}, "num_kv_heads"), ({"heads": 1025}, "num_kv_heads"), ({"stride": 4095}, "page_stride"),
             ({"stride": 4100}, "page_stride"), ({"stride": 2**41}, "page_stride"), ({"stride": -4096}, "page_stride"),
             ({"k": P + 8}, "aligned"), ({"v": 2 * P + 2}, "aligned")]
BAD_BATCH = [({"table": None}, "NULL"), ({"context": None}, "NULL"), ({"seqs": -1}, "num_seqs"), ({"tokens": -1}, "num_tokens"),
             ({"max_pages": 0}, "max_pages"), ({"max_pages": 2**26 + 1}, "max_pages"), ({"tokens": 5}, "without query_start"),
             ({"tokens": 2**24 + 1, "starts": 4 * P}, "num_tokens"), ({"seqs": 2**24 + 1, "starts": 4 * P}, "num_seqs"),
             ({"table": 3 * P + 2}, "aligned"), ({"context": 3 * P + 1}, "aligned"), ({"starts": 4 * P + 2}, "aligned")]


def _calls(qe):
    """Each entry point as a function of (cache, batch)."""
    L = qe.lib()
    return {
        "append": lambda c, b: L.qe_launch_qkv_norm_rope_paged_append(5 * P, 6 * P, 7 * P, 8 * P, None, None, None, None, None,
                                                                      None, c, b, None, 12, 0, 0, F(1e-6)),
        "decode": lambda c, b: L.qe_launch_attention_gqa_paged_decode(5 * P, c, b, 6 * P, 7 * P, None, None, 12, 0),
        "prefill": lambda c, b: L.qe_launch_attention_gqa_paged_prefill(5 * P, c, b, 6 * P, 7 * P, None, None, 12, 0),
        "bounds": lambda c, b: L.qe_launch_paged_key_bounds(c, b, 5 * P, 6 * P, None),
        "select": lambda c, b: L.qe_launch_paged_select(5 * P, c, b, 6 * P, 7 * P, 8 * P, 9 * P, None, 12, 4, 1, 1),
        "sparse": lambda c, b: L.qe_launch_attention_gqa_paged_sparse(5 * P, c, b, 6 * P, 7 * P, 8 * P, None, None, 12, 4),
    }


@pytest.mark.parametrize("name", ["append", "decode", "prefill", "bounds", "select", "sparse"])
def test_descriptions(qe, name):
    call = _calls(qe)[name]
    for bad, text in BAD_CACHE:
        _says(qe, call(_at(_cache(qe, **bad)), _at(_batch(qe))), text)
    for bad, text in BAD_BATCH:
        if name == "decode" and "starts" in bad:
            text = "query_start"
        _says(qe, call(_at(_cache(qe)), _at(_batch(qe, **bad))), text)
    _says(qe, call(None, _at(_batch(qe))), "NULL")
    _says(qe, call(_at(_cache(qe)), None), "NULL")
    for none in ({"seqs": 0, "tokens": 0}, {"tokens": 0, "starts": 4 * P}, {"seqs": 0, "starts": 4 * P}):
        if name != "decode" or "starts" not in none:
            assert call(_at(_cache(qe)), _at(_batch(qe, **none))) == 0


def test_append(qe):
    cache, batch = _cache(qe), _batch(qe)

    def append(q=5 * P, q_out=6 * P, k=7 * P, v=8 * P, qb=None, vb=None, qn=None, rope=None, nq=12, qs=0, ks=0, eps=1e-6, c=cache):
        return qe.lib().qe_launch_qkv_norm_rope_paged_append(q, q_out, k, v, qb, None, vb, qn, None, _at(rope), _at(c), _at(batch),
                                                             None, nq, qs, ks, F(eps))
    rope = lambda turns=9 * P, dim=128, scale=1.0: qe._Rope(turns, dim, 0, scale)  # noqa: E731
    for bad in ({"q": None}, {"q_out": None}, {"k": None}, {"v": None}):
        _says(qe, append(**bad), "NULL")
    for bad, text in (({"nq": 13}, "13 q heads"), ({"nq": 0}, "q heads"), ({"nq": 130}, "at most 64"), ({"qs": 1535}, "q_stride"),
                      ({"qs": 1540}, "q_stride"), ({"qs": -1536}, "q_stride"), ({"ks": 128}, "kv_stride"), ({"ks": 2**33}, "kv_stride"),
                      ({"eps": -1.0}, "norm_eps"), ({"eps": math.inf}, "norm_eps"), ({"eps": math.nan}, "norm_eps"),
                      ({"q": 5 * P + 8}, "aligned"), ({"v": 8 * P + 2}, "aligned"), ({"qn": 9 * P + 4}, "aligned"),
                      ({"qb": 9 * P + 8}, "aligned"), ({"rope": rope(turns=None)}, "turns"), ({"rope": rope(turns=9 * P + 4)}, "turns"),
                      ({"rope": rope(dim=24)}, "rotary_dim"), ({"rope": rope(dim=0)}, "rotary_dim"), ({"rope": rope(dim=144)}, "rotary_dim"),
                      ({"rope": rope(scale=math.nan)}, "scale"),
                      ({"q_out": 5 * P + 256}, "q_out overlaps q"), ({"q_out": 5 * P, "qs": 2048}, "q_out over q"),
                      ({"q_out": 7 * P + 16}, "q_out overlaps k"), ({"q_out": 8 * P}, "q_out overlaps v"),
                      ({"q_out": P}, "overlaps the K pages"), ({"q_out": 2 * P + 64}, "overlaps the V pages"),
                      ({"k": P + 4096}, "K pages overlaps k"), ({"v": 2 * P}, "V pages overlaps v"), ({"qn": P}, "K pages overlaps q_norm"),
                      ({"vb": 6 * P}, "q_out overlaps v_bias"), ({"rope": rope(turns=6 * P + 512)}, "q_out overlaps the rotation"),
                      ({"q_out": 3 * P}, "q_out overlaps block_table"), ({"q_out": 3 * P + 4096}, "q_out overlaps context_len"),
                      ({"c": _cache(qe, v=P + 64)}, "K pages overlap the V pages"),
                      ({"c": _cache(qe, v=P + 8192 * 3)}, "K pages overlap the V pages"),
                      ({"c": _cache(qe, stride=8192, v=P + 4096)}, "K pages overlap the V pages"),
                      ({"c": _cache(qe, stride=6144, v=P + 8192)}, "K pages overlap the V pages")):
        _says(qe, append(**bad), text)


def test_attention(qe):
    cache, batch, L = _cache(qe), _batch(qe), qe.lib()

    def decode(q=5 * P, ws=6 * P, out=7 * P, lse=None, nq=12, window=0, f=L.qe_launch_attention_gqa_paged_decode):
        return f(q, _at(cache), _at(batch), ws, out, lse, None, nq, window)

    def prefill(**a):
        return decode(f=L.qe_launch_attention_gqa_paged_prefill, **a)

    def sparse(sel=8 * P, num=4, q=5 * P, ws=6 * P, out=7 * P, lse=None, nq=12, window=0):
        return L.qe_launch_attention_gqa_paged_sparse(q, _at(cache), _at(batch), sel, ws, out, lse, None, nq, num)
    for call in (decode, prefill, sparse):
        for bad in ({"q": None}, {"ws": None}, {"out": None}):
            _says(qe, call(**bad), "NULL")
        for bad, text in (({"nq": 13}, "13 q heads"), ({"nq": 130}, "at most 64"), ({"q": 5 * P + 8}, "aligned"),
                          ({"ws": 6 * P + 8}, "aligned"), ({"out": 7 * P + 4}, "aligned"), ({"lse": 9 * P + 2}, "aligned"),
                          ({"out": 5 * P}, "attn_out overlaps q"), ({"out": 5 * P + 1536 * 8 - 8}, "attn_out overlaps q"),
                          ({"lse": 7 * P}, "attn_out overlaps row_lse"), ({"out": 6 * P + 4096}, "overlaps the workspace"),
                          ({"lse": 5 * P}, "row_lse overlaps q"), ({"ws": P}, "the workspace overlaps the K pages"),
                          ({"out": 2 * P}, "attn_out overlaps the V pages"), ({"out": 3 * P}, "overlaps block_table"),
                          ({"lse": 3 * P + 4096}, "overlaps context_len")):
            _says(qe, call(**bad), text)
    for call in (decode, prefill):
        _says(qe, call(window=-1), "window")
    for bad, text in (({"sel": None}, "NULL"), ({"num": 0}, "num_selected"), ({"num": 2**20 + 1}, "num_selected"), ({"sel": 8 * P + 2}, "aligned"),
                      ({"sel": 7 * P}, "attn_out overlaps selected"), ({"sel": 6 * P}, "the workspace overlaps selected")):
        _says(qe, sparse(**bad), text)
    _says(qe, L.qe_launch_attention_gqa_paged_decode(5 * P, _at(cache), _at(_batch(qe, starts=4 * P)), 6 * P, 7 * P, None, None, 12, 0),
          "query_start")
    many = _cache(qe, heads=1024, v=40 * P)
    _says(qe, L.qe_launch_attention_gqa_paged_sparse(100 * P, _at(many), _at(_batch(qe, seqs=1, tokens=2**21, starts=4 * P)), 8 * P, 6 * P,
                                                     7 * P, None, None, 1024, 4), "num_tokens")


def test_bounds_and_selection(qe):
    cache, batch, L = _cache(qe), _batch(qe), qe.lib()

    def bounds(b=5 * P, s=6 * P):
        return L.qe_launch_paged_key_bounds(_at(cache), _at(batch), b, s, None)

    def select(q=5 * P, b=6 * P, s=7 * P, sel=8 * P, ws=9 * P, nq=12, num=4, sinks=1, recent=1, bt=batch):
        return L.qe_launch_paged_select(q, _at(cache), _at(bt), b, s, sel, ws, None, nq, num, sinks, recent)
    for bad, text in (({"b": None}, "NULL"), ({"s": None}, "NULL"), ({"b": 5 * P + 8}, "aligned"), ({"s": 6 * P + 2}, "aligned"),
                      ({"s": 5 * P + 256}, "bounds overlaps bound_steps"), ({"b": P}, "bounds overlaps the K pages"),
                      ({"s": 3 * P}, "bound_steps overlaps block_table")):
        _says(qe, bounds(**bad), text)
    for bad in ({"q": None}, {"b": None}, {"s": None}, {"sel": None}, {"ws": None}):
        _says(qe, select(**bad), "NULL")
    for bad, text in (({"nq": 13}, "13 q heads"), ({"num": 0}, "num_selected"), ({"sinks": -1}, "do not fit"), ({"recent": -1}, "do not fit"),
                      ({"sinks": 2, "recent": 3}, "do not fit"), ({"sinks": 2**31 - 1, "recent": 2**31 - 1}, "do not fit"),
                      ({"q": 5 * P + 8}, "aligned"), ({"b": 6 * P + 8}, "aligned"), ({"ws": 9 * P + 2}, "aligned"),
                      ({"sel": 5 * P}, "selected overlaps q"), ({"ws": 8 * P}, "selected overlaps the workspace"),
                      ({"ws": 6 * P}, "the workspace overlaps bounds"), ({"sel": 7 * P}, "selected overlaps bound_steps"),
                      ({"bt": _batch(qe, seqs=2**24, tokens=2**24, max_pages=2**20)}, "num_tokens")):
        _says(qe, select(**bad), text)


def test_workspace_sizes(qe):
    assert qe.paged_decode_workspace_bytes(1) == qe.paged_decode_workspace_bytes(5000, 128, 2)
    assert qe.paged_prefill_workspace_bytes(1) % 16 == 0
    assert qe.paged_select_workspace_bytes(3, 2, 100) == 3 * 2 * 100 * 4
    assert qe.paged_select_workspace_bytes(0, 2, 100) == 0
    n = ctypes.c_size_t()
    L = qe.lib()
    for name in ("qe_paged_decode_workspace_bytes", "qe_paged_prefill_workspace_bytes"):
        _says(qe, getattr(L, name)(1, 12, 2, None), "NULL")
        _says(qe, getattr(L, name)(-1, 12, 2, ctypes.byref(n)), "num_tokens")
        _says(qe, getattr(L, name)(1, 13, 2, ctypes.byref(n)), "13 q heads")
    _says(qe, L.qe_paged_select_workspace_bytes(1, 2, 8, None), "NULL")
    _says(qe, L.qe_paged_select_workspace_bytes(2**24, 1024, 2**26, ctypes.byref(n)), "max_pages")
    _says(qe, L.qe_paged_select_workspace_bytes(1, 2, 0, ctypes.byref(n)), "max_pages")


def test_rope_turns(qe):
    """The tables against their formulas (double arithmetic on both sides: pow and log differ by a few ulp)."""
    i = np.arange(64)
    plain = 1e6 ** (-2.0 * i / 128) / (2 * np.pi)
    got, scale = qe.rope_turns()
    assert scale == 1.0 and np.allclose(got, plain, rtol=1e-14, atol=0)
    got, scale = qe.rope_turns(kind="linear", factor=4.0)
    assert scale == 1.0 and np.allclose(got, plain / 4, rtol=1e-14, atol=0)
    got, scale = qe.rope_turns(kind="bands", factor=8.0, original_positions=8192, low_turns=1, high_turns=4)
    r = np.clip((4 - 8192 * plain) / 3, 0, 1)
    assert scale == 1.0 and np.allclose(got, (1 - r) * plain + r * plain / 8, rtol=1e-13, atol=0)
    got, scale = qe.rope_turns(kind="ramp", factor=4.0, original_positions=32768)
    at = [128 * math.log(32768 / (n * 2 * math.pi)) / (2 * math.log(1e6)) for n in (32, 1)]
    first, last = math.floor(at[0]), math.ceil(at[1])
    r = np.clip((i - first) / (last - first), 0, 1)
    assert abs(scale - (0.1 * math.log(4) + 1)) < 1e-7 and np.allclose(got, (1 - r) * plain + r * plain / 4, rtol=1e-13, atol=0)
    assert np.allclose(got[:first + 1], plain[:first + 1], rtol=1e-14, atol=0) and np.allclose(got[last:], plain[last:] / 4, rtol=1e-14, atol=0)
    got, scale = qe.rope_turns(kind="ramp", factor=1.0)
    assert scale == 1.0 and np.allclose(got, plain, rtol=1e-14, atol=0)
    assert qe.rope_turns(rotary_dim=16, theta=1e4)[0].numel() == 8


def test_rope_turns_refusals(qe):
    for bad, text in (({"rotary_dim": 0}, "rotary_dim"), ({"rotary_dim": 24}, "rotary_dim"), ({"rotary_dim": 144}, "rotary_dim"),
                      ({"rotary_dim": -16}, "rotary_dim"), ({"theta": 1.0}, "theta"), ({"theta": math.inf}, "theta"), ({"theta": math.nan}, "theta"),
                      ({"kind": "linear", "factor": 0.5}, "factor"), ({"kind": "ramp", "factor": math.nan}, "factor"),
                      ({"kind": "ramp", "original_positions": 0}, "original_positions"), ({"kind": "bands", "low_turns": 0.0}, "low_turns"),
                      ({"kind": "bands", "low_turns": 32.0}, "low_turns"), ({"kind": "ramp", "high_turns": math.inf}, "low_turns"),
                      ({"kind": "spiral"}, "spiral")):
        with pytest.raises(RuntimeError, match=text):
            qe.rope_turns(**bad)
    L, turns = qe.lib(), (ctypes.c_double * 64)()
    _says(qe, L.qe_rope_turns(None, ctypes.byref(F()), 128, 1e6, 0, 1, 1, 1, 2), "NULL")
    _says(qe, L.qe_rope_turns(turns, None, 128, 1e6, 0, 1, 1, 1, 2), "NULL")
    _says(qe, L.qe_rope_turns(turns, ctypes.byref(F()), 128, 1e6, 4, 1, 1, 1, 2), "kind")


def test_python_descriptions(qe):
    """Shapes, types and places of the tensors, before the library is called."""
    import torch
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="meta")  # noqa: E731
    f16 = lambda *s: torch.zeros(s, dtype=torch.float16, device="meta")  # noqa: E731
    for call, text in ((lambda: qe.paged_cache(f16(4, 2, 16, 128).float(), f16(4, 2, 16, 128)), "float16"),
                       (lambda: qe.paged_cache(f16(4, 2, 16, 128), f16(5, 2, 16, 128)), "shapes"),
                       (lambda: qe.paged_cache(f16(2, 16, 128), f16(2, 16, 128)), "shapes"),
                       (lambda: qe.paged_cache(f16(4, 16, 2, 128).transpose(1, 2), f16(4, 2, 16, 128)), "strides"),
                       (lambda: qe.paged_cache(f16(4, 2, 2, 16, 128)[:, 0], f16(4, 2, 16, 128)), "strides"),
                       (lambda: qe.paged_batch(i32(3, 8).long(), i32(3)), "int32"),
                       (lambda: qe.paged_batch(i32(8, 3).T, i32(3)), "contiguous"),
                       (lambda: qe.paged_batch(i32(3, 8), i32(4)), "context_len"),
                       (lambda: qe.paged_batch(i32(3, 8), i32(3), i32(3), 9), "query_start"),
                       (lambda: qe.paged_batch(i32(3, 8), i32(3), i32(4)), "num_tokens"),
                       (lambda: qe.rope(torch.zeros(64)), "float64"),
                       (lambda: qe.rope(torch.zeros(128, dtype=torch.float64)[::2]), "contiguous"),
                       (lambda: qe.paged_cache(*[torch.zeros(4, 2, 16, 128, dtype=torch.float16)] * 2), "must be on a GPU"),
                       (lambda: qe.paged_batch(torch.zeros(3, 8, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)), "must be on a GPU")):
        with pytest.raises(RuntimeError, match=text):
            call()


CALLS = """
class Cache(ctypes.Structure):
    _fields_ = [("k", V), ("v", V), ("stride", ctypes.c_longlong), ("pages", I), ("size", I), ("heads", I), ("dim", I)]
class Batch(ctypes.Structure):
    _fields_ = [("table", V), ("starts", V), ("context", V), ("seqs", I), ("tokens", I), ("max_pages", I)]
def describe(tokens=4, starts=False, size=64, max_pages=64, heads=2):
    return (ctypes.byref(Cache(100 * P, 200 * P, 0, 16, size, heads, 128)),
            ctypes.byref(Batch(300 * P, 301 * P if starts else 0, 302 * P, 1 if starts else tokens, tokens, max_pages)))
def names():
    out = [e.kernel for e in events()]
    R.recorder_reset(0)
    return out
def near(got, *want):
    assert len(got) == len(want) and all(w in g for g, w in zip(got, want)), (got, want)
q, out, ws, a, b = (V(P * i) for i in (1000, 2000, 3000, 4000, 5000))
"""


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("recorder"))


def test_launches(recorder):
    """Which kernels the calls launch, on the stream they are given."""
    launch_recorder.run(recorder, CALLS + """
s = V(0x5000)
c, t = describe()
ok(L.qe_launch_qkv_norm_rope_paged_append(q, out, a, b, V(0), V(0), V(0), V(0), V(0), V(0), c, t, s, I(12), ctypes.c_longlong(0),
                                          ctypes.c_longlong(0), ctypes.c_float(1e-6)))
e = events()
near(names(), "paged_append")
assert e[0].grid == (4, 1, 1) and e[0].stream == 0x5000, e
ok(L.qe_launch_attention_gqa_paged_decode(q, c, t, ws, out, V(0), s, I(12), I(0)))
near(names(), "paged_decode_kernel", "paged_decode_merge")
ok(L.qe_launch_attention_gqa_paged_sparse(q, c, t, a, ws, out, V(0), s, I(12), I(32)))
near(names(), "paged_decode_kernel", "paged_decode_merge")
for size in (16, 32, 64, 256):
    c, t = describe(100, True, size)
    ok(L.qe_launch_attention_gqa_paged_prefill(q, c, t, ws, out, V(0), s, I(12), I(0)))
    e = events()
    near(names(), "paged_prefill_kernelILb%d" % (size >= 32), "paged_prefill_merge")
    assert all(x.stream == 0x5000 for x in e), e
ok(L.qe_launch_paged_key_bounds(c, t, a, b, s))
ok(L.qe_launch_paged_select(q, c, t, a, b, out, ws, s, I(12), I(8), I(1), I(1)))
near(names(), "paged_key_bounds", "paged_score", "paged_select")
""")


def test_launches_too_large(recorder):
    """A launch has fewer than 2^32 threads."""
    launch_recorder.run(recorder, CALLS + """
L.qe_last_error.restype = ctypes.c_char_p
def refused(rc, text):
    assert rc != 0 and text in L.qe_last_error(), L.qe_last_error()
    assert names() == []
refused(L.qe_launch_paged_select(q, *describe(tokens=1 << 21), a, b, out, ws, V(0), I(12), I(8), I(1), I(1)), b"num_tokens=2097152")
refused(L.qe_launch_paged_select(q, *describe(tokens=1 << 20, max_pages=1 << 14), a, b, out, ws, V(0), I(12), I(8), I(1), I(1)), b"max_pages=16384")
refused(L.qe_launch_paged_key_bounds(*describe(tokens=1 << 24), a, b, V(0)), b"below 2^24")
""")


def test_routes(recorder):
    """Which kernels take which sizes."""
    launch_recorder.run(recorder, CALLS + """
def decode(window=0, q_heads=12, **how):
    ok(L.qe_launch_attention_gqa_paged_decode(q, *describe(**how), ws, out, V(0), V(0), I(q_heads), I(window)))
    e = events()
    return e[0].grid[0], *names()
def sparse(n, **how):
    ok(L.qe_launch_attention_gqa_paged_sparse(q, *describe(**how), a, ws, out, V(0), V(0), I(12), I(n)))
    e = events()
    return e[0].grid[0], *names()
def is_short(got, blocks):
    assert got[0] == blocks and len(got) == 2 and "paged_short" in got[1], got
def is_shared(got):
    assert got[0] == 256 and len(got) == 3 and "paged_decode_kernel" in got[1] and "merge" in got[2], got
is_short(decode(max_pages=16), 8)                          # 1024 keys
is_shared(decode(max_pages=17))
is_short(decode(window=1024), 8)
is_shared(decode(window=1025))
is_short(decode(max_pages=16, q_heads=34), 16)             # two groups of 16 heads each
is_shared(decode(max_pages=32, tokens=95))
is_short(decode(max_pages=32, tokens=96), 192)             # 2048 keys
is_shared(decode(max_pages=33, tokens=96))
is_short(sparse(16), 8)
is_shared(sparse(17))
is_shared(sparse(500, tokens=95))
is_short(sparse(500, tokens=96), 192)
def merge(tokens, **how):
    return decode(tokens=tokens, **how)[2]
assert "Li32ELi1024E" in merge(7) and "Li4ELi256E" in merge(8)
def prefill(tokens, q_heads):
    ok(L.qe_launch_attention_gqa_paged_prefill(q, *describe(tokens, True), ws, out, V(0), V(0), I(q_heads), I(0)))
    e = events()
    return e[0].grid[0], names()[0]
for tokens, q_heads, waves, few in ((2, 12, 4, 1), (3, 12, 4, 0), (85, 12, 4, 0), (86, 12, 8, 0), (16, 2, 4, 1), (512, 2, 8, 0)):
    blocks, name = prefill(tokens, q_heads)
    assert blocks == 2048 // waves and "Li%dELb%d" % (waves, few) in name, (tokens, q_heads, blocks, name)
def chunk_merge(tokens, max_pages):
    ok(L.qe_launch_attention_gqa_paged_prefill(q, *describe(tokens, True, max_pages=max_pages), ws, out, V(0), V(0), I(12), I(0)))
    return names()[1]
assert "Li4ELi4E" in chunk_merge(80, 17) and "Li4ELi1E" in chunk_merge(80, 16) and "Li8ELi4E" in chunk_merge(86, 17)
assert "Li8ELi1E" in chunk_merge(171, 17)
def select(max_pages):
    ok(L.qe_launch_paged_select(q, *describe(max_pages=max_pages), a, b, out, ws, V(0), I(12), I(8), I(1), I(1)))
    return names()[1]
for pages, name in ((1, "Li256ELi8E"), (2048, "Li256ELi8E"), (2049, "Li512ELi8E"), (4096, "Li512ELi8E"), (4097, "Li1024ELi16E"),
                    (16384, "Li1024ELi16E"), (16385, "select_long")):
    assert name in select(pages), (pages, select(pages))
""")


@pytest.mark.parametrize("kernel", ["paged_prefill_kernel"])
def test_tiles_read_at_turned_addresses_are_aligned_for_it(kernel, tmp_path):
    """Its LDS addresses are turned by exclusive or of 16 to 240."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    root, out = launch_recorder.ROOT, str(tmp_path / "variables.ll")
    csrc = os.path.join(root, "qwen-engine_amd", "csrc")
    r = subprocess.run([hipcc, "-std=c++17", "--offload-arch=gfx950", "--offload-device-only", "-S", "-emit-llvm", "-O1", "-Xclang",
                        "-disable-llvm-passes", f"-I{root}/include", f"-I{csrc}", os.path.join(csrc, "attention_paged.hip"),
                        "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    found = re.findall(rf"^@\S*\d{kernel}\S*4smem = .*addrspace\(3\) global .*align (\d+)", open(out).read(), re.M)
    assert len(found) == 8 and all(int(a) >= 256 for a in found), found


def test_cpp_mirror_compiles():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    root = launch_recorder.ROOT
    r = subprocess.run([hipcc, "-std=c++20", "-fsyntax-only", "-x", "hip", "--offload-arch=gfx950", f"-I{root}/include",
                        os.path.join(root, "tests", "cpp", "paged_call_shapes.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
