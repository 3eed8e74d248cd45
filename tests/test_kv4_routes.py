"""Which kernels the 4-bit cache and log probability calls launch, checked
without a GPU on the recording stand-in for the HIP runtime (launch_recorder.py)."""
import pytest

import launch_recorder

CALLS = """
def decode(stream=0, nq=12, nkv=2, ms=4096, weights=False):
    ok(L.qe_launch_attention_gqa_flash_decode_kv4(V(P), V(P), V(P), V(P), V(P), V(0), V(0), V(stream), I(nq), I(nkv), I(128),
                                                  I(ms), V(0), V(0), V(0), V(0), V(P if weights else 0)))
def prefill(T, stream=0, nq=12, nkv=2, ms=4096, weights=False):
    w = V(P if weights else 0)
    ok(L.qe_launch_attention_gqa_prefill_kv4(V(P), V(P), V(P), V(P << 20), V(0), V(0), I(T), V(stream), I(nq), I(nkv), I(128), I(ms),
                                             I(nq * 128), w, w, w))
def evict(in_place, nkv=2, ms=4096, keep=1000):
    a, b, c, d = (V(P * k) for k in (1, 100, 200, 300))
    out = (a, b, c) if in_place else (V(P * 400), V(P * 500), V(P * 600))
    ok(L.qe_launch_kv4_evict(a, b, c, V(0), *out, d, V(P * 700), V(P), I(keep), I(4), I(8), V(0), I(nkv), I(128), I(ms)))
def logprobs(rows, vocab=151936, top=5):
    p = V(P if top else 0)
    ok(L.qe_launch_token_logprobs(V(P), V(P), V(P), V(P), p, p, V(P), I(rows), I(vocab), ctypes.c_longlong(vocab), I(top), V(0)))
def names():
    out = [e.kernel for e in events()]
    R.recorder_reset(0)
    return out
def near(got, *want):
    assert len(got) == len(want) and all(w in g for g, w in zip(got, want)), (got, want)
"""


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("recorder"))


def _run(recorder, snippet):
    import textwrap
    launch_recorder.run(recorder, CALLS + textwrap.dedent(snippet))


def test_decode_is_two_launches(recorder):
    _run(recorder, """
        decode()
        e = events()
        near(names(), "kv4_decode_kernel", "kv4_decode_merge")
        assert e[0].block == 256 and e[0].grid[0] == 2 * 32 and e[1].grid[0] == 12, e  # 32 runs of 128 rows
        decode(ms=131072, weights=True)
        e = events()
        assert e[0].block == 1024 and e[0].grid[0] == 2 * 128 and e[1].grid[0] == 12 + 2 * 256, e
        R.recorder_reset(0)
        decode(nq=128, nkv=2)  # groups of more than 16 q heads take several blocks a run
        assert events()[0].grid[0] == 2 * 4 * 32, events()
    """)


def test_prefill_splits_only_with_a_workspace_and_not_when_recorded(recorder):
    _run(recorder, """
        s = 0x5000
        prefill(100, s)
        near(names(), "kv4_prefill_kernel")
        reserve(s)
        prefill(100, s)
        near(names(), "kv4_prefill_kernel", "kv4_prefill_merge")
        prefill(100, s, weights=True)
        near(names(), "kv4_prefill_kernel", "kv4_prefill_merge", "kv4_prefill_weights")
        prefill(1000, s, weights=True)  # the q rows' sums are split too
        near(names(), "kv4_prefill_kernel", "kv4_prefill_merge", "weights_kernel", "weights_merge")
        prefill(100, s, ms=512)  # too short to split
        near(names(), "kv4_prefill_kernel")
        R.recorder_set_capturing(V(s), I(1))
        prefill(1000, s, weights=True)
        near(names(), "kv4_prefill_kernel", "kv4_prefill_weights")
        R.recorder_set_capturing(V(s), I(0))
        tune("gemm_split_k", 0)
        prefill(100, s)
        near(names(), "kv4_prefill_kernel")
    """)


def test_prefill_row_blocks(recorder):
    """Eight waves a block from 32 blocks of 256 rows on."""
    _run(recorder, """
        prefill(100)
        prefill(1000)
        a, b = events()
        assert (a.block, a.grid[0]) == (256, 2 * 5) and (b.block, b.grid[0]) == (512, 2 * 24), (a, b)
    """)


def test_prefill_partials_and_their_merge_stay_together(recorder):
    _run(recorder, """
        s = 0x5000
        reserve(s)
        R.recorder_reset(2000)
        go = threading.Barrier(3)
        def work(k):
            go.wait()
            for i in range(4):
                if k == 2: prefill(100, s, weights=True)
                elif k == 1: gemm(128, 1536, 8960, s)
                else: attention(s)
        threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        e = events()
        assert len(e) == 4 * (3 + 2 + 2), e
        i = 0
        while i < len(e):  # launches come in whole groups of one thread
            n = 3 if "kv4_prefill_kernel" in e[i].kernel else 2
            assert len({x.thread for x in e[i:i + n]}) == 1, e[i:i + n]
            i += n
    """)


def test_evict_and_logprobs(recorder):
    _run(recorder, """
        evict(False)
        near(names(), "kv4_evict_select", "kv4_evict_copy")
        evict(True)
        near(names(), "kv4_evict_select", "kv4_evict_move")
        logprobs(1)
        e = events()
        near(names(), "token_logprobs_segment", "token_logprobs_row")
        assert e[0].grid[0] == 19 and e[1].grid[0] == 1, e
        logprobs(1024, top=0)
        assert events()[0].grid[0] == 1024 * 5, events()
    """)


def test_cpp_mirror_compiles():
    import os
    import shutil
    import subprocess
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    root = launch_recorder.ROOT
    r = subprocess.run([hipcc, "-std=c++20", "-fsyntax-only", "-x", "hip", "--offload-arch=gfx950", f"-I{root}/include",
                        os.path.join(root, "tests", "cpp", "kv4_call_shapes.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
