"""Sizes on both sides of what the entry points of the 8-bit tensors take (tests/host/packed8_limits_main.cpp calls the library on a
context whose device does not exist, so that a call that is taken ends before anything is launched)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "onemodel-csharp_amd", "lib")
MAIN = os.path.join(ROOT, "tests", "host", "packed8_limits_main.cpp")
OK, E_ARG, E_DEVICE = "0", "1", "3"


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not (os.path.exists(hipcc) and os.path.exists(MAIN) and os.path.exists(os.path.join(LIB, "libom_hip.so"))):
        pytest.skip("needs hipcc, the test program's source and the built library")
    exe = str(tmp_path_factory.mktemp("limits") / "limits")
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-std=c++17", "-O1", "-Wno-unused-result", MAIN, "-o", exe,
                    "-L", LIB, "-lom_hip", "-Wl,-rpath," + LIB], check=True, capture_output=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout.splitlines()
    return [(line.split(" ", 2) + [""])[:3] for line in out]


def _check(lines, part, count):
    mine = [line for line in lines if part in line[0]]
    assert len(mine) == count, mine
    for name, status, message in mine:
        if name.startswith("ok-"):
            assert status == OK, (name, status, message)
        elif name.startswith("take-"):  # as far as the device
            assert status == E_DEVICE and message.startswith("hipSetDevice"), (name, status, message)
        else:  # refused by the entry point that the name begins with
            assert status == E_ARG and message.startswith(name.split("-")[0] + ":"), (name, status, message)


def test_products(lines):
    _check([line for line in lines if "no-rows" not in line[0]], "gemm", 6)


def test_weight_gradients(lines):
    _check([line for line in lines if "-dw-" in line[0] or line[0].startswith("om_linear")], "", 4)


def test_packing(lines):
    _check([line for line in lines if "pack" in line[0]], "", 10)


def test_gelu(lines):
    _check(lines, "gelu", 4)


def test_layernorm_forward(lines):
    _check([line for line in lines if line[0] in ("take-norm", "om_layernorm_fwd_x8-norm")], "", 16)


def test_layernorm_backward(lines):
    _check([line for line in lines if "norm-bwd" in line[0] or line[0].startswith("om_layernorm_bwd")], "", 5)


def test_no_rows(lines):
    _check(lines, "no-rows", 5)
