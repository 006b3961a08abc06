"""The 4-bit entries without a GPU: what they refuse, before any device work, and their sizes."""
import ctypes as ct

import numpy as np
import pytest

import mx4_ref as ref
from anima_hip import _lib

P = 4096  # a 16-byte aligned address that is never read


def refused(ok, word):
    assert not ok
    assert word in _lib.last_error(), _lib.last_error()


PACK = dict(x=P, ldx=64, dtype=ref.F32, codes=P, scales=P, rows=4, K=64)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"),
    (dict(K=-1), "K"), (dict(K=2 ** 30 + 1), "2^30"), (dict(ldx=63), "stride"),
    (dict(ldx=-64), "stride"), (dict(x=None), "null"), (dict(codes=None), "null"),
    (dict(scales=None), "null"), (dict(codes=P + 8), "16-byte"), (dict(scales=P + 2), "4-byte"),
    (dict(x=P + 2), "aligned to their type"), (dict(x=P + 1, dtype=ref.BF16), "aligned"),
])
def test_pack_and_unpack_refusals(change, word):
    a = {**PACK, **change}
    lib = _lib.load()
    refused(lib.anima_hip_mx4_pack_dev(a["x"], a["ldx"], a["dtype"], a["codes"], a["scales"],
                                       a["rows"], a["K"], None), word)
    refused(lib.anima_hip_mx4_unpack_dev(a["codes"], a["scales"], a["x"], a["ldx"], a["dtype"],
                                         a["rows"], a["K"], None), word)


LINEAR = dict(a=P, lda=64, codes=P, scales=P, c=P, ldc=32, M=4, N=32, K=64, dtype=ref.F32)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(M=-1), "M, N and K"), (dict(N=-1), "M, N and K"),
    (dict(K=-1), "M, N and K"), (dict(K=2 ** 30 + 1), "2^30"), (dict(lda=63), "stride"),
    (dict(ldc=31), "stride"), (dict(a=None), "null"), (dict(c=None), "null"),
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=P + 4), "16-byte"),
    (dict(scales=P + 1), "4-byte"), (dict(a=P + 2), "aligned"), (dict(c=P + 1), "aligned"),
])
def test_linear_refusals(change, word):
    a = {**LINEAR, **change}
    refused(_lib.load().anima_hip_linear_mx4_dev(
        a["a"], a["lda"], a["codes"], a["scales"], a["c"], a["ldc"], a["M"], a["N"], a["K"],
        a["dtype"], None, 0, None), word)


APPEND = dict(k=P, v=P, dtype=ref.F32, kc=P, ks=P, vc=P, vs=P, starts=P, B=2, S_new=3, H_kv=2,
              D=128, S_max=16)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(B=-1), "negative"), (dict(S_new=-1), "negative"),
    (dict(H_kv=-1), "negative"), (dict(H_kv=0), "H_kv"), (dict(D=96), "D must"),
    (dict(D=256), "D must"), (dict(S_max=-1), "negative"), (dict(S_max=2 ** 30 + 1), "S_max"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(starts=None), "null"),
    (dict(kc=None), "null"), (dict(ks=None), "null"), (dict(vc=None), "null"),
    (dict(vs=None), "null"), (dict(kc=P + 8), "16-byte"), (dict(vc=P + 8), "16-byte"),
    (dict(vs=P + 2), "4-byte"), (dict(v=P + 2), "aligned to their type"),
])
def test_append_refusals(change, word):
    a = {**APPEND, **change}
    refused(_lib.load().anima_hip_kv4_append_dev(
        a["k"], a["v"], a["dtype"], None, None, a["kc"], a["ks"], a["vc"], a["vs"], a["starts"],
        None, a["B"], a["S_new"], a["H_kv"], a["D"], a["S_max"], None), word)


ATTEND = dict(q=P, dtype=ref.F32, kc=P, ks=P, vc=P, vs=P, lens=P, out=P, B=2, Bk=2, S_q=1, H=4,
              H_kv=2, D=128, S_max=16, scale=0.1)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(B=-1), "negative"), (dict(S_q=-1), "negative"),
    (dict(H=-4), "negative"), (dict(H_kv=0), "H_kv"), (dict(H_kv=3), "multiple"),
    (dict(D=80), "D must"), (dict(S_max=-1), "negative"), (dict(Bk=3), "one sequence"),
    (dict(Bk=0), "one sequence"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(S_q=2 ** 29), "2^30"), (dict(q=None), "null"),
    (dict(out=None), "null"), (dict(lens=None), "null"), (dict(kc=None), "null"),
    (dict(vs=None), "null"), (dict(vc=P + 8), "16-byte"), (dict(ks=P + 2), "4-byte"),
    (dict(q=P + 2), "aligned"), (dict(out=P + 1), "aligned"),
])
def test_attention_refusals(change, word):
    a = {**ATTEND, **change}
    refused(_lib.load().anima_hip_kv4_attention_dev(
        a["q"], a["dtype"], None, a["kc"], a["ks"], a["vc"], a["vs"], a["lens"], None, a["out"],
        None, a["B"], a["Bk"], a["S_q"], a["H"], a["H_kv"], a["D"], a["S_max"],
        ct.c_float(a["scale"]), True, None, 0, None), word)


def test_scratch_sizes_of_calls_without_work():
    lib = _lib.load()
    assert lib.anima_hip_linear_mx4_scratch_bytes(0, 64, 64, ref.F32) == 0
    assert lib.anima_hip_linear_mx4_scratch_bytes(-1, 64, 64, ref.F32) == 0
    assert lib.anima_hip_linear_mx4_scratch_bytes(64, 64, 64, 1) == 0
    assert lib.anima_hip_kv4_attention_scratch_bytes(1, 0, 4, 2, 128, 64, ref.F32) == 0
    assert lib.anima_hip_kv4_attention_scratch_bytes(1, 1, 4, 3, 128, 64, ref.F32) == 0


def test_reference_packing_is_nearest():
    """The numpy packing the GPU tests compare with: each value goes to the nearest magnitude of
    its group's scale, and a saturated one is off by at most 1 (of 6 ... 7) units."""
    rng = np.random.default_rng(0)
    x = np.float32(rng.standard_normal((64, 96)) * np.exp(rng.standard_normal((64, 1)) * 4))
    codes, scales = ref.pack(x.astype(np.float64))
    y = ref.unpack(codes, scales, 96)
    unit = np.exp2(np.repeat(scales, 32, -1).astype(float) - 127)
    mag = np.abs(x) / unit
    nearest = np.abs(mag[..., None] - ref.STEPS).min(-1)
    np.testing.assert_array_equal(np.abs(np.abs(y) / unit - mag), nearest)
    assert nearest.max() <= 1.0 and mag.max() <= 7.0
