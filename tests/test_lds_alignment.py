"""Kernels that turn bits of absolute LDS addresses (address ^ 16 .. 224) need their buffer aligned to 256 bytes; where
it stands otherwise depends on what other shared variables a kernel has (no GPU needed)."""
import os
import re
import shutil
import subprocess

import pytest

import launch_recorder

CSRC = os.path.join(launch_recorder.ROOT, "qwen-engine_amd", "csrc")


@pytest.mark.parametrize("source,kernels", [("attention_kv4.hip", ["kv4_prefill_kernel", "kv4_prefill_weights_kernel"]),
                                            ("attention.hip", ["prefill_attention_kernel"])])
def test_buffers_read_at_turned_addresses_are_aligned_for_it(source, kernels, tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    out = str(tmp_path / "variables.ll")  # what the compiler is told of each variable, nothing optimized
    r = subprocess.run([hipcc, "-std=c++17", "--offload-arch=gfx950", "--offload-device-only", "-S", "-emit-llvm", "-O1",
                        "-Xclang", "-disable-llvm-passes", f"-I{launch_recorder.ROOT}/include", f"-I{CSRC}",
                        os.path.join(CSRC, source), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    for kernel in kernels:
        found = re.findall(rf"^@\S*\d{kernel}\S*4smem = .*addrspace\(3\) global .*align (\d+)", open(out).read(), re.M)
        assert found and all(int(a) >= 256 for a in found), (kernel, found)
