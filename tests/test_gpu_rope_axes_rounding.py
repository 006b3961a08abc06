"""The rotation by several axes in f32, held to the roundings that it has, and its gradient against
differences.

Angles are products in 64 bits, in turns: off by less than 2^-51 of themselves and 2^-50.  Cosine and
sine are rounded to f32 once (2^-24 of them), the two products and their sum at most once each.  So
a c - b s is off by at most 3 * 2^-24 (|a c| + |b s|), and by what the angle's own error moves it."""
import numpy as np
import pytest

import fp8_ref as ref
import test_gpu_rope_axes as ropet
from anima_hip import rt

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


def pairs_of(x, P, interleaved):
    return (x[..., 0:2 * P:2], x[..., 1:2 * P:2]) if interleaved else (x[..., :P], x[..., P:2 * P])


@pytest.mark.parametrize("B,S,H,D,axes,P,far", [
    (2, 500, (16, 4), 128, 3, 64, 200), (1, 3000, (3, 3), 80, 4, 17, 200),
    (3, 700, (4, 1), 64, 2, 32, 2 ** 31), (1, 900, (2, 1), 1023, 2, 300, 1 << 20),
    (9000, 3, (2, 1), 40, 3, 20, 1 << 20)])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, False), (False, True),
                                                 (True, True)])
def test_f32_is_rounded_as_stated(B, S, H, D, axes, P, far, interleaved, inverse):
    raw, val, pos, freqs, axis = ropet.inputs(B, S, H, D, axes, P, ref.F32, D, far)
    got = ropet.rope(*raw, pos, freqs, axis, ref.F32, interleaved, inverse)
    theta = (pos[..., axis].astype(np.longdouble) * freqs.astype(np.longdouble))[:, :, None]
    c, s = np.abs(np.cos(theta)).astype(float), np.abs(np.sin(theta)).astype(float)
    turn = np.abs(theta).astype(float) * 2.0 ** -51 + 2.0 ** -50
    for g, v in zip(got, val):
        want = ref.rotate(v, pos, freqs, axis, interleaved, inverse)
        np.testing.assert_array_equal(g[..., 2 * P:], v[..., 2 * P:])
        a, b = (np.abs(x) for x in pairs_of(v, P, interleaved))
        err = [np.abs(x) for x in pairs_of(g - want, P, interleaved)]
        for e, tol in zip(err, (a * c + b * s, b * c + a * s)):
            assert (e <= 3 * STEP * (1 + 2.0 ** -20) * tol + (a + b) * turn + 1e-44).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_gradient_against_differences(interleaved, inverse):
    """f(x) = <g, R x>: its gradient is R^-1 g, the call with `inverse` turned over, and its
    differences (f(x + e) - f(x - e)) / 2e one element at a time are those of a linear function, with
    no error but the roundings."""
    S, H, D, P, axes, e = 2, (2, 1), 12, 5, 3, 1.0
    raw, val, pos, freqs, axis = ropet.inputs(1, S, H, D, axes, P, ref.F32, 11, 1 << 20)
    rng = np.random.default_rng(12)
    g = [np.float32(rng.standard_normal(r.shape)) for r in raw]
    grad = ropet.rope(*g, pos, freqs, axis, ref.F32, interleaved, not inverse)
    assert len(set(axis)) > 1
    for i in range(2):
        # Multiples of 2^-10, so that adding e is exact.
        x = np.round(val[i] * 1024) / 1024
        n = x.size
        moved = np.concatenate([x + e * np.eye(n).reshape(n, *x.shape[1:]),
                                x - e * np.eye(n).reshape(n, *x.shape[1:])])
        y = ropet.rope(np.float32(moved), np.float32(moved[:, :, :0]), pos, freqs, axis, ref.F32,
                       interleaved, inverse, shared=True)[0].astype(float)
        f = (g[i].astype(float) * y).sum((1, 2, 3))
        difference = ((f[:n] - f[n:]) / (2 * e)).reshape(x.shape)
        # Each y by 3 STEP (|a| + |b|), and far positions' angles by 2^20 * 2^-51.
        size = 2 * np.abs(moved).max()
        tol = (3 * STEP + 2.0 ** -31) * (np.abs(g[i]).sum() * size / e + 2 * np.abs(g[i]).max())
        assert np.abs(difference - grad[i]).max() <= tol
        assert np.abs(grad[i]).max() > 1000 * tol
