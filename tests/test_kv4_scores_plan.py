"""The cases of tests/test_gpu_kv4_scores.py reach the kernel, row blocks and splits they name
(csrc/mx4_plan.h, on the CPU)."""
import os
import shutil
import subprocess

import pytest

import test_gpu_kv4_scores as scores
from mx4_ref import F32

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")

SOURCE = """
#include "mx4_plan.h"
#include <iostream>
int main()
{
    int B, S_q, H, H_kv, D, S_max, f32;
    while (std::cin >> B >> S_q >> H >> H_kv >> D >> S_max >> f32) {
        const auto p = anima_hip::mx4_plan::attn_plan(B, S_q, H, H_kv, D, S_max, f32, false);
        std::cout << (p.tile ? "tile " : "token ") << p.row_blocks << " " << p.splits << "\\n";
    }
}
"""


def test_cases_reach_their_kernels(tmp_path):
    (tmp_path / "p.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I",
                    os.path.join(ROOT, "anima-on-android_amd", "csrc"), str(tmp_path / "p.cpp"),
                    "-o", str(tmp_path / "p")], check=True)
    text = "\n".join(" ".join(map(str, [*c[1:7], int(c[0] == F32)])) for c in scores.SHAPES)
    out = subprocess.run([str(tmp_path / "p")], input=text, capture_output=True, text=True,
                         timeout=60, check=True).stdout.splitlines()
    assert len(out) == len(scores.SHAPES)
    for c, line in zip(scores.SHAPES, out):
        assert line == f"{c[7]} {c[8]} {c[9]}", (c, line)
