"""The largest and smallest sizes that the 4-bit cache and log probability entry points take: what their kernels'
32-bit indices can count, and no rows.  Decided on the host before any HIP call (no GPU needed)."""
import ctypes

import pytest

P = 0x100000  # an aligned address; nothing is launched
INT_MAX = 2**31 - 1


@pytest.fixture(scope="module")
def L():
    import qe_amd
    return qe_amd.lib()


def _says(L, rc, text):
    assert rc == 1 and text in L.qe_last_error().decode(), (rc, L.qe_last_error())


def test_vocabularies_whose_last_segment_ends_past_32_bits(L):
    """Segments of up to 32768 logits begin up to 7 logits before the row, and a thread counts its chunk's end: the
    last segment's end has to be an int.  vocab + 7 + 32767 is the sum that says how many segments there are."""
    n = ctypes.c_size_t()
    for vocab in (INT_MAX - 32768, INT_MAX - 32773):
        last = (vocab + 6) // 32768 * 32768
        assert vocab + 7 + 32767 > INT_MAX and last + 32768 > INT_MAX
        _says(L, L.qe_token_logprobs_workspace_bytes(1, vocab, 0, ctypes.byref(n)), "vocab_size")
        _says(L, L.qe_launch_token_logprobs(P, P, P, None, None, None, P, 1, vocab, ctypes.c_longlong(vocab), 0, None),
              "vocab_size")
    assert L.qe_token_logprobs_workspace_bytes(1, INT_MAX - 32775, 0, ctypes.byref(n)) == 0
    assert n.value == -(-(INT_MAX - 32775 + 7) // 8192) * 3 * 4


def test_caches_whose_runs_end_past_32_bits(L):
    """Decode cuts a cache into up to 128 runs, each rounded up to 32 rows: the end of the last one, up to 128 * 32 rows
    behind the cache, and a wave's next 32 * 16 rows have to be ints."""
    n = ctypes.c_size_t()
    for rows in (INT_MAX - 31, INT_MAX - 4094):
        run = -(-(-(-rows // 128)) // 32) * 32
        assert rows + 127 > INT_MAX or 128 * run > INT_MAX
        for weights in (0, 1):
            _says(L, L.qe_kv4_decode_workspace_bytes(1, rows, weights, ctypes.byref(n)), "max_seq_len")
        _says(L, L.qe_launch_attention_gqa_flash_decode_kv4(P, P, P, P, P, None, None, None, 1, 1, 128, rows, None, None,
                                                            None, None, None), "max_seq_len")
    rows = INT_MAX - 8191
    assert L.qe_kv4_decode_workspace_bytes(1, rows, 1, ctypes.byref(n)) == 0
    assert n.value == (128 * 130 + rows + (-rows) % 32) * 4


def test_key_weights_of_more_heads_than_a_tile_of_q_rows_can_address(L):
    """A tile of q rows holds the 128 // group tokens that 128 rows of one kv head hold; their places in q are byte
    offsets of 32 bits from the tile's first."""
    def prefill(nq, nkv, T=128):
        far = P + T * nq * 256
        return L.qe_launch_attention_gqa_prefill_kv4(P, P, P, far, None, None, T, None, nq, nkv, 128, 64, nq * 128, None,
                                                     P, P)
    for nq, nkv in ((131073, 131073), (2 * 131073, 131073), (64 * 131073, 131073)):
        group = nq // nkv
        assert (128 // group) * nq * 256 > 2**32
        _says(L, prefill(nq, nkv), "num_q_heads")


def test_rows_of_outputs_shorter_than_the_q_heads_past_32_bits(L):
    """128 values of 2^25 heads are 2^32, which an int would take for 0."""
    rc = L.qe_launch_attention_gqa_prefill_kv4(P, P, P, 1 << 45, None, None, 1, None, 1 << 25, 1 << 25, 128, 64, 128, None,
                                               None, None)
    _says(L, rc, "hidden_size")


def test_no_rows(L):
    """The size query says 0 bytes for no rows, and an allocation of none may be NULL, as that of no logits."""
    n = ctypes.c_size_t(1)
    assert L.qe_token_logprobs_workspace_bytes(0, 100, 5, ctypes.byref(n)) == 0 and n.value == 0

    def lp(x, ws, rows):
        return L.qe_launch_token_logprobs(x, P, P, None, None, None, ws, rows, 100, ctypes.c_longlong(100), 0, None)
    assert lp(None, None, 0) == 0 and lp(P, None, 0) == 0 and lp(None, P, 0) == 0
    assert L.qe_launch_token_logprobs(*[None] * 7, 0, 100, ctypes.c_longlong(100), 5, None) == 0
    for x, ws in ((None, P), (P, None)):
        _says(L, lp(x, ws, 1), "NULL")
