"""The intervals of keys and rows that the scored attention kernels walk and mask by, checked on the CPU against the rule in
64-bit arithmetic at sizes up to the largest that the entry points accept (tests/host/scored_bounds_main.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAIN = os.path.join(ROOT, "tests", "host", "scored_bounds_main.cpp")


def test_intervals_against_64_bits(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not (os.path.exists(hipcc) and os.path.exists(MAIN)):
        pytest.skip("needs hipcc and the test program's source")
    exe = str(tmp_path / "bounds")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-std=c++17", "-O1", "-fwrapv", "-Wno-unused-result", MAIN, "-o",
                    exe], check=True, capture_output=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=300).stdout.splitlines()
    checks, broken = map(int, out[-1].split())
    assert checks > 1_000_000 and broken == 0, out
