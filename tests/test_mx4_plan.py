"""The plans of the 4-bit operators (csrc/mx4_plan.h), asked for on the CPU through
tests/native/mx4_plan_shape.cpp: what was measured fastest where two kernels come close, and the
kernel that each case of the GPU tests of one shape is there for."""
import os
import shutil
import subprocess

import pytest

import test_gpu_mx4_shapes as shapes
from mx4_ref import BF16, F32

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "mx4_plan_shape")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-Wall", "-Werror", "-I", os.path.join(ROOT, "anima-on-android_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "mx4_plan_shape.cpp"), "-o", exe],
                   check=True)

    def ask(*words):
        line = " ".join(str(int(w) if isinstance(w, bool) else w) for w in words) + "\n"
        run = subprocess.run([exe], input=line, capture_output=True, text=True, timeout=60)
        assert run.returncode == 0, run.stdout + run.stderr
        return run.stdout.strip()
    return ask


@pytest.mark.parametrize("dtype,M,N,K,want", shapes.LINEAR)
def test_linear_cases_reach_their_kernels(plan, dtype, M, N, K, want):
    assert plan("linear", M, N, K, dtype == F32, True).startswith(want)


@pytest.mark.parametrize("dtype,Bn,S_q,H,H_kv,D,S,causal,want", shapes.ATTEND)
def test_attention_cases_reach_their_kernels(plan, dtype, Bn, S_q, H, H_kv, D, S, causal, want):
    assert plan("attend", Bn, S_q, H, H_kv, D, S, dtype == F32, causal).startswith(want)


@pytest.mark.parametrize("args", [(5, 300, 32, 32, 64, 140), (5, 300, 32, 32, 128, 140),
                                  (1, 300, 64, 64, 64, 130), (1, 300, 64, 64, 64, 64),
                                  (1, 300, 64, 64, 128, 64)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_tile_tests_reach_the_tile_kernel(plan, args, f32, causal):
    assert plan("attend", *args, f32, causal).startswith("tile")


# GPU time of whole calls (us), the fastest kernel and the next.
@pytest.mark.parametrize("dtype,M,N,K,want", [
    (BF16, 16, 2048, 2048, "few"),        # 5.5, staged 7.4
    (BF16, 16, 2048, 8192, "staged"),     # 9.8, few 12.5
    (F32, 4, 2048, 8192, "few"),          # 12.2, staged 15.2
    (F32, 16, 2048, 2048, "staged"),      # 8.8, few 13.1
    (BF16, 24, 2048, 8192, "staged 5 8"),  # 10.1
    (BF16, 333, 2048, 2048, "staged 4 1"),  # 12.1, 64 x 128 tiles 14.8
    (BF16, 1024, 8192, 2048, "staged 1 1"),  # 30.5, 192 x 256 tiles 36.7
    (BF16, 4608, 8192, 2048, "staged 0 1"),
    (F32, 333, 2048, 1024, "staged 3 1"),  # 16.0, 64 x 128 in two splits 19.0
    (F32, 2048, 8192, 2048, "staged 0 1")])  # 170, 128 x 256 tiles 182
def test_measured_linear(plan, dtype, M, N, K, want):
    assert plan("linear", M, N, K, dtype == F32, True).startswith(want)


@pytest.mark.parametrize("f32,B,S_q,H,H_kv,D,S,causal,want", [
    (False, 1, 1, 16, 16, 128, 200, True, "token 1"),     # 7.5, two splits 9.8
    (False, 16, 1, 16, 4, 128, 16384, True, "token 8"),   # 30.3, four splits 35
    (False, 1, 512, 16, 4, 128, 512, True, "token 1"),    # 10.8, tile 18.7
    (False, 2, 1000, 16, 16, 128, 1200, True, "tile 1"),  # 37, token 47
    (False, 2, 4096, 16, 16, 128, 512, False, "tile 1"),
    (True, 2, 2048, 16, 16, 128, 2048, True, "token 1")])  # 141, tile 172
def test_measured_attention(plan, f32, B, S_q, H, H_kv, D, S, causal, want):
    assert plan("attend", B, S_q, H, H_kv, D, S, f32, causal) == want


def test_plans_cover_their_work(plan):
    """Splits hold every chunk of K and no empty one, whatever the size."""
    for M in (17, 100, 1000, 70000):
        for N in (1, 300, 9000):
            for K in (1, 127, 128, 1000, 4096, 1 << 23):
                for f32 in (0, 1):
                    for staged in (0, 1):
                        p = plan("linear", M, N, K, f32, staged).split()
                        assert p[0] in ("few", "tiles", "pad", "staged")
                        assert p[0] == "few" or 1 <= int(p[2]) <= 16
