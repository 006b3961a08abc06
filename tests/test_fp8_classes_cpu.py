"""FP8Linear and `rotate` without a GPU: what they hand to the library and what they refuse, over
device arrays held in host memory and a library that notes its calls."""
import threading
import time

import numpy as np
import pytest

from anima_hip import _lib, fp8, mx4, rope_axes
from anima_hip.rope import generate_rope_freqs
from test_mx4_classes_cpu import HostArray, in_threads


class Library:
    """Every entry succeeds; names and arguments are noted."""

    def __init__(self):
        self.seen, self.inside, self.most = [], 0, 0

    def __getattr__(self, name):
        def call(*args):
            self.inside += 1
            self.most = max(self.most, self.inside)
            time.sleep(0.002)
            self.seen.append((name, args, threading.get_ident()))
            self.inside -= 1
            return True
        return call

    def anima_hip_linear_fp8_scratch_bytes(self, M, N, K, dtype):
        return 64 * M


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    for module in (mx4, fp8):
        monkeypatch.setattr(module, "DeviceArray", HostArray)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    return lib


def test_linear_calls(lib):
    lin = fp8.FP8Linear(np.zeros((48, 300), np.float32))
    assert lin.shape == (48, 300)
    name, args, _ = lib.seen[0]
    assert name == "anima_hip_fp8_pack_dev" and args[1:3] == (300, 0) and args[5:] == (48, 300, None)
    lib.seen.clear()
    y = lin(np.zeros((2, 5, 300), np.uint16))
    assert y.shape == (2, 5, 48) and y.dtype == np.uint16
    (a, pack, _), (b, mul, _) = lib.seen
    assert (a, b) == ("anima_hip_fp8_pack_dev", "anima_hip_linear_fp8_dev")
    assert pack[1:3] == (300, 2) and pack[5:] == (10, 300, None)
    assert mul[:2] == pack[3:5] and mul[5:10] == (48, 10, 48, 300, 2) and mul[11] == 640
    lib.seen.clear()
    y, h = lin.after_norm(np.zeros((3, 300), np.float32), eps=1e-5)
    assert y.shape == (3, 48) and h.shape == (3, 300)
    norm = lib.seen[0][1]
    assert norm[2] is None and norm[4] is None and norm[9] is None and norm[13:] == (3, 300, None)
    assert abs(norm[5].value - 1e-5) < 1e-11 and norm[11:13] == lib.seen[1][1][:2]


@pytest.mark.parametrize("call", [
    lambda lin, x: lin(x[:, 1:]), lambda lin, x: lin(np.float32(3)),
    lambda lin, x: lin.after_norm(x, x[:1]), lambda lin, x: lin.after_norm(x, np.uint16(x)),
    lambda lin, x: lin.after_norm(x, None, np.ones(299)), lambda lin, x: fp8.pack(x[0]),
    lambda lin, x: fp8.FP8Linear(x[0]),
    lambda lin, x: fp8.add_rmsnorm(x, x[:, :1]),
    lambda lin, x: fp8.unpack(np.zeros((2, 256)), np.zeros((2, 4)), 300),
    lambda lin, x: fp8.unpack(np.zeros((2, 384)), np.zeros((2, 3)), 300)])
def test_refusals(lib, call):
    lin = fp8.FP8Linear(np.zeros((48, 300), np.float32))
    lib.seen.clear()
    with pytest.raises(ValueError):
        call(lin, np.zeros((4, 300), np.float32))
    assert not lib.seen


def test_one_call_at_a_time(lib):
    """A call's pack and product come together, whatever other threads do."""
    lin = fp8.FP8Linear(np.zeros((48, 300), np.float32))
    lib.seen.clear()
    got = in_threads(5, lambda i: lin(np.zeros((1 + 7 * i, 300), np.float32)).shape)
    assert got == [(1 + 7 * i, 48) for i in range(5)]
    assert lib.most == 1
    for a, b in zip(lib.seen[::2], lib.seen[1::2]):
        assert a[2] == b[2] and a[1][5] == b[1][6]


def test_rotate_calls(lib):
    q, k = np.zeros((2, 5, 4, 64), np.uint16), np.zeros((2, 5, 1, 64), np.uint16)
    freqs = np.ones(20)
    rope_axes.rotate(q, k, np.zeros((2, 5, 3), int), freqs, np.arange(20) % 3, True, True)
    name, a, _ = lib.seen[0]
    assert name == "anima_hip_rope_axes_dev"
    assert (list(a[1]), a[4], list(a[6]), a[9]) == ([1280, 64, 256], 4, [320, 64, 64], 1)
    assert a[0] == a[2] and a[5] == a[7] and a[11] == 15 and a[12] is None
    assert a[15:] == (3, 20, 2, 5, 64, 2, True, True, None)
    rope_axes.rotate(q, None, np.zeros((1, 5, 1), int), freqs)
    a = lib.seen[1][1]
    assert a[9] == 0 and a[11] == 0 and a[14] is None


def test_grid_axes_are_the_tables_angles():
    """Angles from positions, frequencies and axes against the table's (rounded to f32: 7 * 2^-24 at
    most, its frequencies by some 2^-22 of the angle)."""
    T, H, W, D = 2, 3, 7, 128
    pos, freqs, axis = rope_axes.grid_axes(H, W, T, D)
    assert pos.dtype == np.int32 and axis.dtype == np.uint8 and freqs.dtype == np.float64
    angle = pos[0][:, axis] * freqs
    table = generate_rope_freqs(H, W, T, D)
    np.testing.assert_allclose(np.cos(angle), table[:, :, 0, 0], rtol=0, atol=7 * 2.0 ** -21)
    np.testing.assert_allclose(np.sin(angle), table[:, :, 1, 0], rtol=0, atol=7 * 2.0 ** -21)
    with pytest.raises(ValueError, match="even"):
        rope_axes.grid_axes(2, 2, 1, 63)
