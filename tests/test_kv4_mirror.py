"""The C++ mirror of the 4-bit cache and log probability calls: what its defaults hand on (no GPU needed)."""
import os
import shutil
import subprocess

import pytest

import launch_recorder

ROOT = launch_recorder.ROOT


def test_rows_of_logits_lie_behind_each_other_unless_said_otherwise(tmp_path):
    """The row stride follows the vocabulary of the call: with the default model's for a smaller vocabulary every row
    but the first would be read from behind it."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "stride")
    r = subprocess.run([hipcc, "-std=c++20", f"-I{ROOT}/include",
                        os.path.join(ROOT, "tests", "cpp", "logprobs_default_stride.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["151936", "1000", "1000", "1024", "999", "-5", "200000"]
