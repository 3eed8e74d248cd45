"""The compiled chunk kernels: at a barrier behind which a tile of LDS may be filled again, every read of it has arrived."""
import os
import re
import shutil
import subprocess

import pytest

import launch_recorder


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    root, out = launch_recorder.ROOT, str(tmp_path_factory.mktemp("listing") / "attention_paged.s")
    csrc = os.path.join(root, "qwen-engine_amd", "csrc")
    r = subprocess.run([hipcc, "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "--offload-device-only", "-S", f"-I{root}/include", f"-I{csrc}", os.path.join(csrc, "attention_paged.hip"),
                        "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    found = dict(re.findall(r"^(\S*paged_prefill_kernel\S*):\s*;.*?\n(.*?)^\.Lfunc_end", open(out).read(), re.M | re.S))
    assert len(found) == 8, list(found)
    return found


def reads_open_at_barriers(body):
    """Barriers that a path reaches with an LDS read behind its last full wait for LDS."""
    code, label = [], {}
    for line in body.splitlines():
        line = line.split(";")[0].strip()
        if re.match(r"\.?\w+:$", line):
            label[line[:-1]] = len(code)
        elif line and not line.startswith("."):
            code.append(line)
    seen, found = {}, set()
    barriers = sum(line.startswith("s_barrier") for line in code)
    todo = [(0, False)]
    while todo:
        i, pending = todo.pop()
        while i < len(code) and not (i in seen and (seen[i] or not pending)):
            seen[i] = pending
            op, *args = code[i].replace(",", " ").split()
            if op.startswith("ds_read"):
                pending = True
            elif op == "s_waitcnt" and "lgkmcnt(0)" in args:
                pending = False
            elif op == "s_barrier" and pending:
                found.add(i)
            elif op == "s_endpgm":
                break
            elif op.startswith("s_cbranch"):
                todo.append((label[args[0]], pending))
            elif op == "s_branch":
                i = label[args[0]]
                continue
            i += 1
    return found, barriers


def test_no_read_is_on_its_way_at_a_barrier(listing):
    for name, body in listing.items():
        found, barriers = reads_open_at_barriers(body)
        assert barriers >= 4 and not found, (name, found)


def test_the_barrier_of_tiles_waits_for_reads_itself(listing):
    """Not only because the compiler happens to use what was read before it."""
    for name, body in listing.items():
        waits = [w for w in re.findall(r"#ASMSTART\s*\n(.*?)#ASMEND", body, re.S) if "s_waitcnt" in w]
        assert len(waits) >= 4 and all("vmcnt(0)" in w and "lgkmcnt(0)" in w for w in waits), (name, waits)


def test_an_open_read_is_found():
    text = "k:\n ds_read_b64_tr_b16 v[0:1], v2\n s_waitcnt lgkmcnt(1)\n s_cbranch_scc1 .L\n s_waitcnt lgkmcnt(0)\n s_barrier\n.L:\n s_barrier\n s_endpgm\n"
    assert reads_open_at_barriers(text) == ({5}, 2)
