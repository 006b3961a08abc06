"""Where the token kernel of the 4-bit cache attention takes two blocks of query rows
(csrc/mx4_plan.h, on the CPU): the cases of tests/test_gpu_kv4_blocks.py, and never for one block of
rows or for f32 at D = 128, whose registers do not hold two."""
import os
import shutil
import subprocess

import pytest

import test_gpu_kv4_blocks as blocks
from mx4_ref import F32

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")

SOURCE = """
#include "mx4_plan.h"
#include <iostream>
int main()
{
    int B, S_q, H, H_kv, D, S_max, f32, causal;
    while (std::cin >> B >> S_q >> H >> H_kv >> D >> S_max >> f32 >> causal) {
        const auto p = anima_hip::mx4_plan::attn_plan(B, S_q, H, H_kv, D, S_max, f32, causal);
        std::cout << p.tile << " " << p.row_blocks << " " << p.tiles << "\\n";
    }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("blocks")
    (d / "p.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I",
                    os.path.join(ROOT, "anima-on-android_amd", "csrc"), str(d / "p.cpp"), "-o",
                    str(d / "p")], check=True)

    def ask(cases):
        text = "\n".join(" ".join(str(int(x)) for x in c) for c in cases)
        out = subprocess.run([str(d / "p")], input=text, capture_output=True, text=True, timeout=60,
                             check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return ask


def test_cases_take_two_blocks(plans):
    cases = [(B, S_q, H, H_kv, D, S, dtype == F32, causal)
             for B, S_q, H, H_kv, S in blocks.CASES for D in (64, 128) for dtype in blocks.TYPES
             for causal in (0, 1)]
    for c, (tile, row_blocks, tiles) in zip(cases, plans(cases)):
        assert not tile and row_blocks == (1 if c[6] and c[4] == 128 else 2), c
        rows = c[1] * (c[2] // c[3])
        assert tiles == -(-rows // (16 * row_blocks))


def test_one_block_of_rows(plans):
    cases = [(B, S_q, H, H_kv, D, S, f32, 1)
             for B in (1, 16, 100) for S_q, H, H_kv in ((1, 16, 16), (1, 16, 1), (4, 32, 8), (16, 4, 4))
             for S in (100, 9000) for D in (64, 128) for f32 in (0, 1)]
    assert all(not tile and row_blocks == 1 and tiles == 1 for tile, row_blocks, tiles in plans(cases))
