"""The C++ mirror of the 4-bit cache and log probability calls: what its defaults hand on (no GPU needed)."""
import os
import shutil
import subprocess

import pytest

import launch_recorder

ROOT = launch_recorder.ROOT


def _seen(source, tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "seen")
    r = subprocess.run([hipcc, "-std=c++20", f"-I{ROOT}/include", os.path.join(ROOT, "tests", "cpp", source), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    return r.stdout.split()


def test_rows_of_logits_lie_behind_each_other_unless_said_otherwise(tmp_path):
    """The row stride follows the vocabulary of the call: with the default model's for a smaller vocabulary every row
    but the first would be read from behind it."""
    assert _seen("logprobs_default_stride.cpp", tmp_path) == ["151936", "1000", "1000", "1024", "999", "-5", "200000"]


def test_rows_of_outputs_lie_behind_each_other_unless_said_otherwise(tmp_path):
    """The width of an output row follows the q heads of the call: with the default model's 1536 for fewer heads every
    row but the first would be written behind them."""
    assert _seen("prefill_default_stride.cpp", tmp_path) == ["1536", "768", "3584", "768", "1536", "512"]


def test_rows_of_outputs_in_python(monkeypatch):
    import qe_amd
    calls = []
    monkeypatch.setattr(qe_amd, "_call", lambda name, *args: calls.append(args[12]))
    for heads, given in (((12, 2), {}), ((6, 2), {}), ((28, 4), {}), ((6, 2), {"hidden_size": 1536}),
                         ((6, 2), {"hidden_size": 512})):
        qe_amd.launch_attention_gqa_prefill_kv4(16, 16, 16, 16, None, None, 7, 0x5000, *heads, **given)
    assert calls == [1536, 768, 3584, 1536, 512]
