"""Which kernels the sizes of the 8-bit tensors' GPU tests reach (host code alone: the choice by sizes, compiled from the library's
own header): every kernel of the products and the weight gradients, with k in one part and in several and with more blocks of it
than the kernel has in flight. A refit of the choice that moves sizes away from a kernel fails here."""
import os
import shutil
import subprocess

import pytest

import packed8_shapes as S
import test_packed8_gpu as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "onemodel-csharp_amd", "lib")
MAIN = os.path.join(ROOT, "tests", "host", "packed8_choice_main.cpp")


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not (os.path.exists(hipcc) and os.path.exists(MAIN) and os.path.exists(os.path.join(LIB, "libom_hip.so"))):
        pytest.skip("needs hipcc, the test program's source and the built library")
    exe = str(tmp_path_factory.mktemp("choice") / "choice")
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-std=c++17", "-O1", "-Wno-unused-result", MAIN, "-o", exe,
                    "-L", LIB, "-lom_hip", "-Wl,-rpath," + LIB], check=True, capture_output=True)

    def run(what, shapes):
        """Kernel, as packed8_shapes names it, and the blocks of its longest part, of each shape."""
        text = "".join("%s %d %d %d %d\n" % (what, S.CUS, *s) for s in shapes)
        out = []
        for line in subprocess.run([exe], input=text, check=True, capture_output=True, text=True, timeout=60).stdout.splitlines():
            kind, a, b, parts, per, _ = line.split()
            k = (kind, int(a), int(b)) if kind == "thin" else (kind, int(a))
            out.append((k + (("split",) if int(parts) > 1 else ()), int(per)))
        assert len(out) == len(shapes)
        return out

    return run


@pytest.mark.parametrize("name,what", [("PRODUCTS", "gemm"), ("SPECIAL_PRODUCTS", "gemm"), ("WEIGHT_GRADIENTS", "dw"),
                                       ("SPECIAL_WEIGHT_GRADIENTS", "dw")])
def test_shapes_reach_the_kernel_they_name(choose, name, what):
    cases = getattr(S, name)
    for (shape, want), (got, _) in zip(cases, choose(what, [c[0] for c in cases])):
        assert got == want, (shape, got, want)


def test_special_values_go_through_every_kernel():
    both = {("tile", t) + p for t in range(6) for p in ((), ("split",))} | {("thin", n, r) for n in (4, 8) for r in (1, 2, 3)}
    assert {k for _, k in S.SPECIAL_PRODUCTS} == both
    assert {k for _, k in S.SPECIAL_WEIGHT_GRADIENTS} == {("dw", t) + p for t in range(4) for p in ((), ("split",))}


# blocks of 128 of k from which on each kernel loads over what it has read: stages in flight, or its wavefronts' first ones
MANY = {("tile", 0): 3, ("tile", 1): 3, ("tile", 2): 3, ("tile", 3): 3, ("tile", 4): 5, ("tile", 5): 9, ("thin", 4): 5, ("thin", 8): 9,
        ("dw", 0): 4, ("dw", 1): 4, ("dw", 2): 5, ("dw", 3): 5}


@pytest.mark.parametrize("what,shapes", [("gemm", G.PRODUCTS + [s for s, _ in S.PRODUCTS]),
                                         ("dw", G.DW + [s for s, _ in S.WEIGHT_GRADIENTS])])
def test_every_kernel_is_reached(choose, what, shapes):
    longest = {}
    for k, per in choose(what, shapes):
        longest[k] = max(longest.get(k, 0), per)
    kernels = {("tile", t) + p for t in range(6) for p in ((), ("split",))} | {("thin", n, r) for n in (4, 8) for r in (1, 2, 3)} \
        if what == "gemm" else {("dw", t) + p for t in range(4) for p in ((), ("split",))}
    assert set(longest) == kernels
    for k, per in longest.items():
        assert per >= MANY[k[:2]], (k, per)


def test_blocks_whose_parts_share_scratch(choose):
    for rows, width, hidden in S.SPLIT_BLOCKS:
        assert choose("dw", [(rows, width, hidden)])[0][0][-1] == "split"
        assert choose("gemm", [(width, hidden, rows)])[0][0][-1] == "split"
