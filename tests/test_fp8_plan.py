"""The plans of the linear layer on 8-bit rows (csrc/fp8_plan.h), asked for on the CPU through
tests/native/fp8_plan_shape.cpp: the shape that each GPU test of one is there for, what was measured
fastest where kernels come close, and for sizes at random that a plan covers its product."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import test_gpu_fp8_shapes as shapes
from fp8_ref import BF16, F32

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "fp8_plan_shape")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-Wall", "-Werror", "-I", os.path.join(ROOT, "anima-on-android_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "fp8_plan_shape.cpp"), "-o", exe],
                   check=True)

    def ask(cases):
        lines = "".join(f"{M} {N} {-(-K // 128)} {int(t == F32)}\n" for t, M, N, K in cases)
        run = subprocess.run([exe], input=lines, capture_output=True, text=True, timeout=100)
        assert run.returncode == 0, run.stdout[-200:] + run.stderr
        return [line.rpartition(" ")[0] for line in run.stdout.splitlines()]
    return ask


def test_gpu_cases_reach_their_shapes(plans):
    want = [c[4] for c in shapes.SHAPES]
    assert plans([c[:4] for c in shapes.SHAPES]) == want
    for t in (BF16, F32):
        have = {c[4].rpartition(" ")[0] for c in shapes.SHAPES if c[0] == t and "tile" in c[4]}
        assert have == {f"tile {i}" for i in range(10)}
        assert {c[4] for c in shapes.SHAPES if c[0] == t} >= {f"few {w}" for w in (1, 2, 4, 8)}


# GPU time of whole calls (us), the fastest kernel and others.
@pytest.mark.parametrize("dtype,M,N,K,want", [
    (BF16, 1, 2048, 2048, "few 8"),        # 4.1
    (BF16, 1, 2048, 8192, "tile 9 8"),     # 8.7, few 9.9
    (BF16, 1, 8192, 2048, "few 4"),        # 6.2, tiles 6.8
    (BF16, 4608, 8192, 2048, "tile 1 1"),  # 73.6, 256 x 256 tiles 80
    (F32, 8, 6144, 2048, "few 8"),         # 6.9
])
def test_what_was_measured_fastest(plans, dtype, M, N, K, want):
    assert plans([(dtype, M, N, K)]) == [want]


def test_plans_cover_their_products(plans):
    rng = np.random.default_rng(1)
    sizes = np.exp2(rng.uniform(0, (16, 16, 15), (4000, 3))).astype(int)
    cases = [(t, *map(int, s)) for s in sizes for t in (BF16, F32)]
    top = 2 ** 30
    cases += [(t, *s) for t in (BF16, F32)
              for s in ((1, 1, 1), (top, 1, 128), (1, top, 128), (1, 1, top), (top, 1, 4096),
                        (2 ** 16, 2 ** 16, 4096), (1, 1, 2 ** 22), (1, 1, 2 ** 22 + 1), (7, 9, 0),
                        (2 ** 20, 2 ** 14, 128), (top, 1, 0))]
    assert len(plans(cases)) == len(cases)
