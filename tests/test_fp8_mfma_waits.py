"""The compiled linear layer on 8-bit rows: whatever touches the result of an fp8 MFMA, on any path, but
the next one on the same accumulators, comes when it has been written.

The compiler waits for 8 passes behind `v_mfma_scale_f32_32x32x64_f8f6f4`, which takes 16: a vector
instruction may follow 18 wait states later at the soonest.  csrc/fp8_linear.hip puts its own wait behind
its MFMAs; a copy of an accumulator that the compiler moves in front of that would read old values, and
only now and then."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")

STATES = 18  # behind a 16-pass MFMA


def registers(line):
    """(file, first, last) of every vector register operand, the result's first."""
    out = []
    for r in re.finditer(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)", line):
        a = int(r.group(2) or r.group(4))
        out.append((r.group(1), a, int(r.group(3) or a)))
    return out


def kernels(asm):
    """{symbol: (instructions, {label: index})} of the kernels with fp8 MFMAs."""
    out = {}
    for m in re.finditer(r"^(_ZN\S*fp8_\S*kernel\S*):(.*?)\.Lfunc_end", asm, re.S | re.M):
        code, labels = [], {}
        for line in m.group(2).splitlines():
            line = line.split(";")[0].strip()
            if re.match(r"\.LBB\S+:", line):
                labels[line[:-1]] = len(code)
            elif line and not line.startswith("."):
                code.append(line)
        if any(line.startswith("v_mfma_scale") for line in code):
            out[m.group(1)] = code, labels
    return out


def early_uses(code, labels):
    bad = []
    for i, mfma in enumerate(code):
        if not mfma.startswith("v_mfma_scale"):
            continue
        result = registers(mfma)[0]
        paths, seen = [(i + 1, 0)], {}
        while paths:
            at, states = paths.pop()
            while at < len(code) and states < STATES and seen.get(at, STATES) > states:
                seen[at] = states
                line = code[at]
                op = line.split()[0]
                used = any(f == result[0] and a <= result[2] and b >= result[1]
                           for f, a, b in registers(line))
                if used and op.startswith("v_mfma_scale") and registers(line)[0] == result:
                    break  # the accumulators' next MFMA: the hardware's own order
                if used:
                    bad.append(f"{states} states after {mfma}: {line}")
                    break
                if op.startswith("s_cbranch"):
                    paths.append((labels[line.split()[1]], states + 1))
                elif op == "s_branch":
                    at, states = labels[line.split()[1]], states + 1
                    continue
                elif op == "s_endpgm":
                    break
                elif op == "s_nop":
                    states += int(line.split()[1])
                states += 1
                at += 1
    return bad


def test_the_check_sees_early_uses():
    code = ["v_mfma_scale_f32_32x32x64_f8f6f4 v[0:15], v[20:27], v[30:37], v[0:15], v40, v41",
            "s_nop 7", "s_cbranch_scc1 .LBB0_1", "s_nop 15", "v_mov_b32 v50, v15", "s_endpgm",
            "v_mov_b32 v50, v15", "s_endpgm"]
    assert len(early_uses(code, {".LBB0_1": 6})) == 1
    assert not early_uses(code[:6], {".LBB0_1": 3})
    code[1] = "s_nop 0"
    assert len(early_uses(code, {".LBB0_1": 0})) == 0 and len(early_uses(code, {".LBB0_1": 4})) == 1


def test_results_are_waited_for(tmp_path):
    out = str(tmp_path / "fp8_linear.s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-w", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "-I",
                    os.path.join(ROOT, "include"), "--cuda-device-only", "-S",
                    os.path.join(ROOT, "anima-on-android_amd", "csrc", "fp8_linear.hip"), "-o", out],
                   check=True, capture_output=True, timeout=600)
    with open(out) as f:
        found = kernels(f.read())
    assert len(found) == 14  # ten tile shapes, four sizes of the few-rows kernel
    for name, (code, labels) in found.items():
        assert not early_uses(code, labels), name
