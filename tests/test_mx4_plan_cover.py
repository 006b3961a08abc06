"""The 4-bit linear layer's launch plans (csrc/mx4_plan.h, on the CPU) share out all of K and leave no
share empty, their scratch parts do not meet, and the GPU tests reach every staged kernel there is."""
import os
import shutil
import subprocess

import pytest

import test_gpu_mx4_limits as limits
import test_gpu_mx4_shapes as shapes
from mx4_ref import BF16, F32

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")

SOURCE = """
#include "mx4_plan.h"
#include <iostream>
using namespace anima_hip::mx4_plan;
int main()
{
    int M, N, K, f32, staged;
    while (std::cin >> M >> N >> K >> f32 >> staged) {
        const LinPlan p = lin_plan(M, N, K, f32, staged);
        const LinScratch s = lin_scratch(p, M, N, K, f32);
        const TileShape *t = p.kernel == kTiles ? kTileShapes : f32 ? kF32Shapes : kBf16Shapes;
        std::cout << p.kernel << " " << p.pad << " " << p.pairs << " " << p.shape << " " << p.tiles_m
                  << " " << p.tiles_n << " " << p.splits << " " << p.per_split << " " << p.chunks << " "
                  << t[p.shape].bm << " " << t[p.shape].bn << " " << s.a << " " << s.codes << " "
                  << s.scales << " " << s.planes << " " << s.bytes << "\\n";
    }
}
"""
FEW, TILES, STAGED = 0, 1, 2
NAMES = ("kernel pad pairs shape tiles_m tiles_n splits per_split chunks bm bn a codes scales planes "
         "bytes").split()


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("cover")
    (d / "p.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "anima-on-android_amd", "csrc"), str(d / "p.cpp"), "-o",
                    str(d / "p")], check=True)

    def ask(cases):
        text = "\n".join(" ".join(str(int(x)) for x in c) for c in cases)
        out = subprocess.run([str(d / "p")], input=text, capture_output=True, text=True, timeout=60,
                             check=True).stdout.splitlines()
        assert len(out) == len(cases)
        return [dict(zip(NAMES, map(int, line.split()))) for line in out]
    return ask


def test_shares_hold_every_chunk(plans):
    cases = [(M, N, K, f32, staged) for M in (17, 33, 100, 333, 1000, 4608, 70000)
             for N in (1, 64, 300, 2048, 9000)
             for K in (1, 64, 127, 128, 256, 384, 640, 1000, 1152, 4096, 11008, 1 << 22, 1 << 23)
             for f32 in (0, 1) for staged in (0, 1)]
    for (M, N, K, f32, staged), p in zip(cases, plans(cases)):
        at = (M, N, K, f32, staged, p)
        assert p["kernel"] in (TILES, STAGED), at
        kp = -(-K // 128) * 128 if p["pad"] else K
        chunk = 64 if p["kernel"] == TILES or f32 else 128
        assert p["chunks"] == -(-kp // chunk), at
        assert p["tiles_m"] == -(-M // p["bm"]) and p["tiles_n"] == -(-N // p["bn"]), at
        assert (p["splits"] - 1) * p["per_split"] < p["chunks"] <= p["splits"] * p["per_split"], at
        assert p["splits"] <= 16, at
        if p["kernel"] == STAGED:
            assert (staged or p["pad"]) and kp % 128 == 0, at
        if p["pairs"]:
            assert p["kernel"] == STAGED and p["chunks"] % 2 == 0 and p["per_split"] % 2 == 0, at
        size = 4 if f32 else 2
        if p["pad"]:
            assert p["codes"] >= M * kp * size and p["scales"] - p["codes"] >= N * kp // 2, at
            assert p["planes"] - p["scales"] >= N * kp // 32, at
            assert all(p[x] % 256 == 0 for x in ("a", "codes", "scales", "planes")), at
        need = p["splits"] * M * N * 4 if p["splits"] > 1 else 0
        assert p["bytes"] - p["planes"] == need, at


def test_gpu_tests_reach_every_staged_kernel(plans):
    """Kernels by type, shape and whether a stage holds two chunks; K is a multiple of 128, two
    chunks in f32, so its small shapes always take both."""
    odd = [m for m in limits.test_linear_odd_and_even_chunks.pytestmark if m.args[0] == "M,N,K"][0]
    cases = [(M, N, K, dtype == F32, 1) for dtype, M, N, K, _ in shapes.LINEAR]
    cases += [(*c, dtype == F32, 1) for c in odd.args[1] for dtype in (F32, BF16)]
    seen = {(c[3], p["shape"], p["pairs"]) for c, p in zip(cases, plans(cases))
            if p["kernel"] == STAGED and not p["pad"]}
    want = {(False, i, 0) for i in range(6)} | {(False, i, 1) for i in (3, 4, 5)}
    want |= {(True, 0, 0), (True, 1, 0), (True, 2, 1), (True, 3, 1)}
    assert seen == want, (want - seen, seen - want)


@pytest.mark.parametrize("dtype,M,N,K,plan", [c for c in shapes.LINEAR if " " in c[4]])
def test_named_plans_word_by_word(plans, dtype, M, N, K, plan):
    p, = plans([(M, N, K, dtype == F32, 1)])
    assert plan == f"staged {p['shape']} {p['splits']}"
