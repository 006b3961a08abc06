"""The whole wait behind the fp8 MFMAs in the compiled linear layer on 8-bit rows: 32 states, the two
`s_nop 15` that csrc/fp8_linear.hip puts there, on every path to a use of the result."""
import test_fp8_mfma_waits as waits
from test_fp8_mfma_waits import pytestmark  # noqa: F401


def test_results_are_waited_for_as_written(tmp_path, monkeypatch):
    monkeypatch.setattr(waits, "STATES", 32)
    short = ["v_mfma_scale_f32_32x32x64_f8f6f4 v[0:15], v[20:27], v[30:37], v[0:15], v40, v41",
             "s_nop 15", "s_nop 14", "v_mov_b32 v50, v15", "s_endpgm"]
    assert len(waits.early_uses(short, {})) == 1
    short[2] = "s_nop 15"
    assert not waits.early_uses(short, {})
    waits.test_results_are_waited_for(tmp_path)
