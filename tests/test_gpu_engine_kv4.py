"""The engine on a 4-bit key/value cache (qe_set_tuning("engine_kv4", 1) before create)."""
import numpy as np
import pytest

import kv4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qe():
    import qe_amd
    qe_amd.lib()
    return qe_amd


def _cfg(qe, chunk=64, fused=1, max_seq=256):
    c = qe.default_config()
    c.num_layers, c.hidden_size, c.intermediate_size = 3, 768, 1024
    c.num_q_heads, c.num_kv_heads, c.vocab_size = 6, 2, 4096
    c.max_seq_len, c.prefill_chunk, c.fused_decode = max_seq, chunk, fused
    return c


def _engine(qe, kv4, **kw):
    qe.set_tuning("engine_kv4", kv4)
    try:
        return qe.Engine(_cfg(qe, **kw), seed=7)
    finally:
        qe.set_tuning("engine_kv4", 0)


PROMPT = [(i * 37 % 3000) + 100 for i in range(150)]


def test_graph_matches_eager_and_the_unfused_sequence(qe, orc):
    a, b, c = _engine(qe, 1), _engine(qe, 1), _engine(qe, 1, fused=0)
    first = a.prefill(PROMPT)
    tokens = a.decode(20, use_graph=True)
    assert b.prefill(PROMPT) == first and b.decode(20, use_graph=False) == tokens
    assert c.prefill(PROMPT) == first and c.decode(20) == tokens
    assert np.isfinite(a.logits().astype(np.float32)).all()
    assert tokens[-1] == orc.argmax_f16(a.logits())
    for e in (b, c):
        assert np.array_equal(a.logits().view(np.uint16), e.logits().view(np.uint16))
    a.reset()
    assert a.prefill(PROMPT) == first and a.decode(20) == tokens
    for e in (a, b, c):
        e.close()


@pytest.mark.parametrize("chunk", [64, 256])
def test_first_layer_caches_are_the_fp16_ones_in_4_bits(qe, chunk):
    """The first layer's K and V depend on nothing that attention wrote: each stored value is within half a step of
    the fp16 engine's (whose angles are in fp32: 2^-24 of 150 positions, relative to what is rotated)."""
    n, steps = len(PROMPT), 9
    e4, e16 = _engine(qe, 1, chunk=chunk), _engine(qe, 0, chunk=chunk)
    e4.prefill(PROMPT)
    e16.prefill(PROMPT)
    for name in ("kcache", "vcache"):
        rows = e4.read(name, np.uint8, 2 * 256 * 80).reshape(2, 256, 80)[:, :n]
        want = e16.read(name, np.float16, 2 * 256 * 128).reshape(2, 256, 128)[:, :n].astype(np.float64)
        _, scale, _ = ref.parts(rows)
        got = ref.values(rows).reshape(2, n, 4, 32)
        want = want.reshape(2, n, 4, 32)
        off = np.abs(got - want)
        size = np.abs(want).max((-1, -2), keepdims=True)
        # half a step, the fp16 engine's rounding and this value's, the angle's and the fp32 sums'
        assert np.all(off <= scale[..., None] * (0.5 + 15 * 2.0 ** -11) + size * (2.0 ** -10 + 150 * 2.0 ** -22)), name
        assert np.abs(got).max() > 0
    e4.decode(steps)
    k = e4.read("kcache", np.uint8, 2 * 256 * 80).reshape(2, 256, 80)
    assert np.all(k[:, n + steps:] == 0) and np.all(np.any(k[:, :n + steps] != 0, -1))
    e4.close()
    e16.close()


def test_arena_is_smaller_and_buffers_do_not_overlap(qe):
    sizes = []
    for kv4 in (0, 1):
        e = _engine(qe, kv4, max_seq=4096)
        spans, total = e.arena_spans()
        e.close()
        end = 0
        for off, size in spans:
            assert off % 256 == 0 and size > 0 and off >= end
            end = off + size
        assert end <= total
        sizes.append(total)
    caches = 2 * 3 * 2 * 4096  # K and V, layers, heads, rows
    assert sizes[0] - sizes[1] == caches * (256 - 80) - 6 * 128 * 130 * 4


def test_context_limit(qe):
    e = _engine(qe, 1)
    with pytest.raises(RuntimeError, match="context window"):
        e.prefill(list(range(256)))
    e.prefill(list(range(250)))
    e.decode(6)
    with pytest.raises(RuntimeError, match="context window"):
        e.decode(1)
    e.close()


def test_file_round_trip(qe, tmp_path):
    """An engine read from a file holds 4-bit rows too, and says the same."""
    a = _engine(qe, 1)
    first = a.prefill(PROMPT)
    tokens = a.decode(10)
    path = str(tmp_path / "kv4.qwenbin")
    a.save_qwenbin(path)
    qe.set_tuning("engine_kv4", 1)
    try:
        b = qe.Engine.from_qwenbin(path, max_seq_len=256, prefill_chunk=64)
    finally:
        qe.set_tuning("engine_kv4", 0)
    assert b.prefill(PROMPT) == first and b.decode(10) == tokens
    assert np.array_equal(a.logits().view(np.uint16), b.logits().view(np.uint16))
    rows = [e.read("kcache", np.uint8, 2 * 256 * ref.ROW) for e in (a, b)]
    assert np.array_equal(*rows) and rows[0].any()
    a.close(), b.close()


def test_what_an_engine_says_and_how_likely_it_was(qe):
    """Tokens of an engine on a 4-bit cache are the most likely ones of its logits, with the probability of the definition."""
    import torch

    e = _engine(qe, 1)
    token = e.prefill(PROMPT)
    for _ in range(5):
        logits = e.logits()
        x = torch.from_numpy(logits.copy()).cuda()
        ids = torch.tensor([token], dtype=torch.int32, device="cuda")
        lp, entropy = (torch.empty(1, device="cuda") for _ in range(2))
        top, top_ids = torch.empty((1, 8), device="cuda"), torch.empty((1, 8), dtype=torch.int32, device="cuda")
        ws = torch.empty(qe.token_logprobs_workspace_bytes(1, x.numel(), 8), dtype=torch.uint8, device="cuda")
        qe.launch_token_logprobs(x, ids, lp, entropy, top, top_ids, ws, 1, vocab_size=x.numel(), top_k=8)
        want, want_entropy, want_top, want_ids, spread = ref.logprobs(logits[None], [token], 8)
        assert int(top_ids[0, 0]) == token and np.array_equal(top_ids.cpu().numpy(), want_ids)
        # fp32: the logit, the maximum and the logarithm are added with three roundings; sums of 4096 terms
        size = np.abs(logits.astype(np.float64)).max() + 20
        assert abs(float(lp) - want[0]) <= 2.0 ** -20 * size
        assert abs(float(entropy) - want_entropy[0]) <= 2.0 ** -20 * (size + spread[0])
        assert float(top[0, 0]) == float(lp)
        token = e.decode(1)[0]
    e.close()
