"""Arguments that the entry points of the 8-bit tensors refuse, checked without a device (tests/host/
packed8_refusals_main.cpp calls the library on a context that has none: every check comes before a launch); and the plain
forms that the GPU tests compare with, against torch's own 8-bit floats."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import packed8_ref as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "onemodel-csharp_amd", "lib")
MAIN = os.path.join(ROOT, "tests", "host", "packed8_refusals_main.cpp")
ENTRY = {"pack": "om_pack8", "unpack": "om_unpack8", "gemm": "om_gemm8", "linear": "om_linear_bwd_x8", "gelu": "om_gelu_",
         "norm": "om_layernorm_", "null": "om_pack8"}


def test_refusals(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not (os.path.exists(hipcc) and os.path.exists(MAIN) and os.path.exists(os.path.join(LIB, "libom_hip.so"))):
        pytest.skip("needs hipcc, the test program's source and the built library")
    exe = str(tmp_path / "refusals")
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-std=c++17", "-O1", "-Wno-unused-result", MAIN, "-o", exe,
                    "-L", LIB, "-lom_hip", "-Wl,-rpath," + LIB], check=True, capture_output=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout.splitlines()
    assert len(out) == 72, len(out)
    for line in out:
        name, status, message = (line.split(" ", 2) + [""])[:3]
        assert "DEVICE" not in line
        if name.startswith("ok-"):
            assert status == "0", line
        else:  # OM_E_ARG with a message that names the entry point
            assert status == "1" and message.startswith(ENTRY[name.split("-")[0]]), line


def test_codes_and_rounding_against_torch():
    torch = pytest.importorskip("torch")
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(codes, P.CODES.astype(np.float32), equal_nan=True)
    rng = np.random.default_rng(0)
    v = np.concatenate([448 * rng.uniform(-1, 1, 20000), np.exp2(rng.uniform(-12, 8, 20000)),
                        (P.CODES[0:126] + P.CODES[1:127]) / 2]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(P.round_e4m3(v.astype(np.float64)), want)


def test_scale_is_the_least_that_holds():
    rng = np.random.default_rng(1)
    x = (rng.normal(size=(50, 300)) * np.exp2(rng.integers(-140, 127, (50, 1)).astype(np.float64))).astype(np.float32)
    x[0], x[1, :128] = 0.0, np.float32(448.0)
    e = P.exponents(x)
    for b in range(3):
        top = np.abs(x[:, 128 * b:128 * b + 128].astype(np.float64)).max(1)
        assert (top <= 448.0 * np.exp2(e[:, b].astype(np.float64))).all()
        assert ((e[:, b] == -127) | (top > 448.0 * np.exp2(e[:, b] - 1.0))).all()
    assert (e[0] == -127).all() and e[1, 0] == 0


def test_bytes_round_trip():
    rng = np.random.default_rng(2)
    for rows, cols in ((1, 1), (3, 130), (2, 600)):
        x = rng.normal(size=(rows, cols)).astype(np.float32)
        raw = P.encode(x)
        assert raw.size == P.nbytes(rows, cols)
        assert np.array_equal(P.decode(raw, rows, cols)[0], P.value(x))


def test_gradients_of_the_plain_forms_against_differences():
    """GELU's slope and LayerNorm's backward in float64, against central differences."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=40)
    h = 1e-5
    # a central difference is off by h^2 / 6 times the third derivative (below 2) and by rounding, 1e-16 / h
    assert np.abs((P.gelu(x + h) - P.gelu(x - h)) / (2 * h) - P.gelu_slope(x)).max() < 1e-9
    z, gamma, g = rng.normal(size=(1, 9)), rng.normal(size=9), rng.normal(size=(1, 9))

    def f(v):  # in float64 throughout
        m = v.mean(1, keepdims=True)
        return (v - m) / np.sqrt(np.square(v - m).mean(1, keepdims=True) + 1e-5)

    rstd = 1 / np.sqrt(z.var(1, keepdims=True) + 1e-5)
    dx, dgamma, dbeta = P.layernorm_bwd(g, f(z), gamma, rstd)
    num = np.zeros_like(z)
    for i in range(9):
        d = np.zeros_like(z)
        d[0, i] = h
        num[0, i] = ((g * gamma * (f(z + d) - f(z - d))).sum()) / (2 * h)
    assert np.abs(num - dx).max() <= 1e-8
    assert np.allclose(dgamma, (g * f(z))[0]) and np.allclose(dbeta, g[0])
