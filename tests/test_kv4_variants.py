"""Which forms of the 4-bit prefill and log probability kernels a call takes, on both sides of each rule, checked
without a GPU on the recording stand-in for the HIP runtime (launch_recorder.py): the sizes of the GPU tests that mean
to reach a form, and the borders."""
import textwrap

import pytest

import launch_recorder
from test_kv4_routes import CALLS


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("recorder"))


def _run(recorder, snippet):
    launch_recorder.run(recorder, CALLS + textwrap.dedent(snippet))


def test_eight_waves_from_28_blocks_of_256_rows_on(recorder):
    _run(recorder, """
        def block(T, nq, nkv):
            prefill(T, nq=nq, nkv=nkv)
            e = events()
            assert len(e) == 1, e
            R.recorder_reset(0)
            return e[0].block, e[0].grid[0]
        assert block(554, 12, 2) == (256, 2 * 26)   # 3324 rows: 13 blocks of 256, 26 of 128 a kv head
        assert block(555, 12, 2) == (512, 2 * 14)   # 3330: 14
        assert block(256, 27, 27) == (256, 27 * 2)
        assert block(256, 28, 28) == (512, 28)
        assert block(6912, 1, 1) == (256, 54)
        assert block(6913, 1, 1) == (512, 28)
        # what test_gpu_kv4_calls.py runs
        for T, nq, nkv in ((600, 12, 2), (598, 12, 2), (130, 64, 32), (257, 28, 28), (2400, 4, 4), (100, 128, 2), (640, 12, 2),
                           (512, 14, 2), (600, 16, 8)):
            assert block(T, nq, nkv)[0] == 512, (T, nq, nkv)
    """)


def test_splits_and_their_merges(recorder):
    _run(recorder, """
        s = 0x5000
        def split(T, ms, nq=12, nkv=2):
            prefill(T, s, nq=nq, nkv=nkv, ms=ms)
            a, b = events()
            R.recorder_reset(0)
            waves = a.block // 64
            row_blocks = -(-T * (nq // nkv) // (32 * waves)) * nkv
            return waves, a.grid[0] // row_blocks, b.block
        reserve(s)
        assert split(170, 4096)[2] == 1024 and split(171, 4096)[2] == 256   # 2040, 2052 rows in all
        for T, ms, nq, nkv in ((180, 5183, 12, 2), (200, 9203, 11, 1), (700, 7203, 3, 3)):
            waves, splits, merge = split(T, ms, nq, nkv)
            assert waves == 4 and splits > 8 and merge == 256, (waves, splits, merge)
        assert split(512, 5600, 14, 2) == (8, 9, 256)
    """)


def test_shares_of_the_q_rows_of_key_weights(recorder):
    _run(recorder, """
        s = 0x5000
        reserve(s)
        def shares(T, ms, nq=12, nkv=2):
            prefill(T, s, nq=nq, nkv=nkv, ms=ms, weights=True)
            e = [x for x in events() if "prefill_weights_kernel" in x.kernel]
            merge = [x for x in events() if "weights_merge" in x.kernel]
            R.recorder_reset(0)
            n = e[0].grid[0] // (-(-ms // 64) * nkv)
            assert len(merge) == (n > 1)
            return n
        assert [shares(T, 4096) for T in (170, 171, 256, 341, 342, 2000)] == [1, 2, 3, 3, 4, 4]
        # more than two blocks a CU for the keys alone: shares of 1024 rows
        assert [shares(T, 16384) for T in (341, 342)] == [3, 4]
        assert [shares(T, 16448) for T in (341, 342, 682, 683)] == [1, 2, 3, 4]
        assert shares(640, 20000) == 3 and shares(2400, 2500, 4, 4) == 4
    """)


def test_long_segments_of_logits_from_two_a_cu_on(recorder):
    _run(recorder, """
        def chunks(rows, vocab):
            logprobs(rows, vocab)
            e = events()
            R.recorder_reset(0)
            assert e[1].grid[0] == rows
            return e[0].grid[0] // rows, "ILi16E" in e[0].kernel
        assert chunks(511, 2000) == (1, False) and chunks(512, 2000) == (1, True)
        assert chunks(255, 40000) == (5, False) and chunks(256, 40000) == (2, True)
        assert chunks(2, 600001) == (74, False) and chunks(8, 2200000) == (68, True)
        for rows, vocab in ((520, 2000), (260, 40000), (513, 20000), (515, 9000), (512, 32761), (512, 32762)):
            assert chunks(rows, vocab)[1], (rows, vocab)
    """)
