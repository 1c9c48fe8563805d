"""The waits of the many-row attention kernel's loading warps, walked on the CPU: tests/cpp/attn_ring_check.cpp includes the kernel's own
rules (leviathan_b200/csrc/lev_attn_ring.h) and runs loading and MMA warps under random schedules with one warp held up at a time, over
pairs, two tiles, page boxes of every height and copies.  Without the arrivals of warps that fetch nothing, the walk must get stuck."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_no_warp_waits_for_a_phase_that_is_over(tmp_path):
    exe = os.path.join(str(tmp_path), "attn_ring_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "leviathan_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "attn_ring_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:]
    assert out.stdout.strip().endswith("ok")
    before = subprocess.run([exe, "before"], capture_output=True, text=True, timeout=300)
    assert before.returncode == 1 and "does not end" in before.stdout
