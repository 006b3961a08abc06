"""The 8-bit entries and the rotation by axes without a GPU: what they refuse, before any device
work, and their sizes."""
import ctypes as ct

import numpy as np
import pytest

import fp8_ref as ref
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
    refused(lib.anima_hip_fp8_pack_dev(a["x"], a["ldx"], a["dtype"], a["codes"], a["scales"],
                                       a["rows"], a["K"], None), word)
    refused(lib.anima_hip_fp8_unpack_dev(a["codes"], a["scales"], a["x"], a["ldx"], a["dtype"],
                                         a["rows"], a["K"], None), word)


NORM = dict(x=P, ldx=64, r=P, ldr=64, w=P, eps=1e-6, dtype=ref.F32, sum=P, ldsum=64, y=2 * P,
            ldy=64, codes=P, scales=P, rows=4, K=64)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(rows=-1), "rows"), (dict(K=-1), "K"),
    (dict(K=2 ** 30 + 1), "2^30"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(codes=None), "together"),
    (dict(scales=None), "together"), (dict(sum=None, y=None, codes=None, scales=None), "no output"),
    (dict(x=None), "null"), (dict(ldx=63), "stride of x"), (dict(ldr=63), "stride of residual"),
    (dict(ldsum=63), "stride of sum"), (dict(ldy=63), "stride of y"), (dict(x=P + 2), "x must be"),
    (dict(r=P + 2), "residual must be"), (dict(sum=P + 1), "sum must be"),
    (dict(y=P + 3), "y must be"), (dict(w=P + 2), "w must be"), (dict(y=P), "different"),
    (dict(codes=P + 8), "16-byte"), (dict(scales=P + 2), "4-byte"),
])
def test_norm_refusals(change, word):
    a = {**NORM, **change}
    refused(_lib.load().anima_hip_add_rmsnorm_fp8_dev(
        a["x"], a["ldx"], a["r"], a["ldr"], a["w"], ct.c_float(a["eps"]), a["dtype"], a["sum"],
        a["ldsum"], a["y"], a["ldy"], a["codes"], a["scales"], a["rows"], a["K"], None), word)


LINEAR = dict(ac=P, sa=P, wc=P, ws=P, c=P, ldc=32, M=4, N=32, K=64, dtype=ref.F32)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(M=-1), "M, N and K"), (dict(N=-1), "M, N and K"),
    (dict(K=-1), "M, N and K"), (dict(K=2 ** 30 + 1), "2^30"), (dict(ldc=31), "stride"),
    (dict(c=None), "null"), (dict(ac=None), "null"), (dict(sa=None), "null"),
    (dict(wc=None), "null"), (dict(ws=None), "null"), (dict(ac=P + 4), "16-byte"),
    (dict(wc=P + 8), "16-byte"), (dict(sa=P + 1), "4-byte"), (dict(ws=P + 2), "4-byte"),
    (dict(c=P + 2), "aligned"), (dict(c=P + 1, dtype=ref.BF16), "aligned"),
])
def test_linear_refusals(change, word):
    a = {**LINEAR, **change}
    refused(_lib.load().anima_hip_linear_fp8_dev(
        a["ac"], a["sa"], a["wc"], a["ws"], a["c"], a["ldc"], a["M"], a["N"], a["K"], a["dtype"],
        None, 0, None), word)


ROPE = dict(q=P, qs=None, qo=P, qos=None, H_q=4, k=P, ks=None, ko=P, kos=None, H_k=2, pos=P,
            counts=P, freqs=P, axis=P, axes=3, pairs=32, B=2, S=5, D=64, dtype=ref.F32)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=1), "dtype"), (dict(B=-1), "negative"), (dict(S=-1), "negative"),
    (dict(H_q=-1), "negative"), (dict(H_k=-1), "negative"), (dict(H_q=2049), "2048"),
    (dict(D=1), "D must"), (dict(D=1025), "D must"), (dict(pairs=0), "pairs"),
    (dict(pairs=33), "pairs"), (dict(axes=0), "axes"), (dict(axes=257), "axes"),
    (dict(q=None), "null"), (dict(qo=None), "null"), (dict(k=None), "null"),
    (dict(ko=None), "null"), (dict(pos=None), "null"), (dict(freqs=None), "null"),
    (dict(q=P + 2), "aligned"), (dict(ko=P + 1), "aligned"), (dict(pos=P + 2), "aligned"),
    (dict(counts=P + 1), "aligned"), (dict(freqs=P + 4), "aligned"),
    (dict(qos=(0, 320, 64)), "overlap"), (dict(kos=(640, 63, 64)), "overlap"),
    (dict(qos=(1280, 320, -63)), "overlap"),
])
def test_rope_refusals(change, word):
    a = {**ROPE, **change}
    refused(_lib.load().anima_hip_rope_axes_dev(
        a["q"], _lib.strides(a["qs"]), a["qo"], _lib.strides(a["qos"]), a["H_q"], a["k"],
        _lib.strides(a["ks"]), a["ko"], _lib.strides(a["kos"]), a["H_k"], a["pos"], 15,
        a["counts"], a["freqs"], a["axis"], a["axes"], a["pairs"], a["B"], a["S"], a["D"],
        a["dtype"], False, False, None), word)


def test_scratch_sizes_of_calls_without_work():
    size = _lib.load().anima_hip_linear_fp8_scratch_bytes
    assert size(0, 64, 64, ref.F32) == 0 and size(64, -1, 64, ref.F32) == 0
    assert size(64, 64, 0, ref.BF16) == 0 and size(64, 64, 64, 1) == 0


def test_reference_packing_is_nearest():
    """The numpy packing the GPU tests compare with: the smallest scale that holds each group, and
    of it the nearest number to each value."""
    rng = np.random.default_rng(0)
    x = np.float32(rng.standard_normal((64, 300)) * np.exp(rng.standard_normal((64, 1)) * 4))
    codes, scales = ref.pack(x.astype(np.float64))
    y = ref.unpack(codes, scales, 300)
    unit = np.exp2(np.repeat(scales[:, :3], 128, -1)[:, :300].astype(float) - 127)
    mag = np.abs(x) / unit
    nearest = np.abs(mag[..., None] - ref.NUMBERS).min(-1)
    np.testing.assert_array_equal(np.abs(np.abs(y) / unit - mag), nearest)
    for g in range(3):
        top = mag[:, 128 * g:128 * g + 128].max(-1)
        assert (top <= 448).all() and (top > 224).all()
    assert (codes[:, 300:] == 0).all() and (scales[:, 3:] == 0).all()


@pytest.mark.parametrize("change", [dict(sum=P, ldsum=65), dict(sum=2 * P, ldsum=80), dict(y=P, ldy=96),
                                    dict(y=2 * P, ldy=65)])
def test_norm_in_place_at_another_stride_is_refused(change):
    """Rows would land on rows that are still to be read."""
    a = {**NORM, **dict(r=2 * P, sum=3 * P, y=4 * P), **change}
    refused(_lib.load().anima_hip_add_rmsnorm_fp8_dev(
        a["x"], a["ldx"], a["r"], a["ldr"], a["w"], ct.c_float(a["eps"]), a["dtype"], a["sum"],
        a["ldsum"], a["y"], a["ldy"], a["codes"], a["scales"], a["rows"], a["K"], None), "in place")


@pytest.mark.parametrize("change,word", [
    (dict(qo=P, qos=(1280, 64, 256)), "in place"), (dict(ko=2 * P, ks=(640, 64, 128)), "in place"),
    (dict(qo=3 * P, ko=3 * P), "overlap"), (dict(qo=2 * P), "overlap"), (dict(ko=P), "overlap")])
def test_rope_overlaps_are_refused(change, word):
    a = {**ROPE, **dict(k=2 * P, qo=3 * P, ko=4 * P), **change}
    refused(_lib.load().anima_hip_rope_axes_dev(
        a["q"], _lib.strides(a["qs"]), a["qo"], _lib.strides(a["qos"]), a["H_q"], a["k"],
        _lib.strides(a["ks"]), a["ko"], _lib.strides(a["kos"]), a["H_k"], a["pos"], 15,
        a["counts"], a["freqs"], a["axis"], a["axes"], a["pairs"], a["B"], a["S"], a["D"],
        a["dtype"], False, False, None), word)
