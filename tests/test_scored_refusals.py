"""Arguments that the rotary and scored-attention entry points refuse, checked without a device (tests/host/
scored_refusals_main.cpp calls the library on a context that has none: every check comes before a launch)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "onemodel-csharp_amd", "lib")
MAIN = os.path.join(ROOT, "tests", "host", "scored_refusals_main.cpp")


def test_refusals(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not (os.path.exists(hipcc) and os.path.exists(MAIN) and os.path.exists(os.path.join(LIB, "libom_hip.so"))):
        pytest.skip("needs hipcc, the test program's source and the built library")
    exe = str(tmp_path / "refusals")
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-std=c++17", "-O1", "-Wno-unused-result", MAIN, "-o", exe,
                    "-L", LIB, "-lom_hip", "-Wl,-rpath," + LIB], check=True, capture_output=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout.splitlines()
    assert len(out) == 58, len(out)
    for line in out:
        name, status, message = (line.split(" ", 2) + [""])[:3]
        assert "DEVICE" not in line
        if name.startswith("ok-"):
            assert status == "0", line
        else:  # OM_E_ARG with a message that names the entry point
            assert status == "1" and message.startswith("om_rope_" if name.startswith("rope") else "om_attention_"), line
