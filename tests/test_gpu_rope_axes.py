"""The rotation by several axes on the GPU against 64-bit numpy.

Cosine and sine are f32 functions of an f32 part of a turn: 2 ulp of theirs and the part's rounding,
together below 2^-21 of 1; two products and one sum round three times.  So a turned value is off by
at most TOL = 2^-20 of |a| + |b|, and by half a step of its type.  Angles are rounded in 64 bits,
relative to the angle: far positions add |theta| * 2^-51.
"""
import numpy as np
import pytest

import fp8_ref as ref
from anima_hip import _lib, rt
from anima_hip.rope import generate_rope_freqs

pytestmark = pytest.mark.gpu

TYPES = [ref.F32, ref.BF16]
TOL = 2.0 ** -20


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


def np_type(dtype):
    return np.float32 if dtype == ref.F32 else np.uint16


class View:
    """A [B, S, H, D] array in a flat device buffer, its axes in memory in `order`, D innermost and
    rows `pad` elements longer."""

    def __init__(self, raw, order="bsh", pad=0, shift=0, fill=None):
        from devmem import DevBuf
        self.shape, self.dtype, self.shift = raw.shape, raw.dtype, shift
        B, S, H, D = raw.shape
        size = {"b": B, "s": S, "h": H}
        step, self.st = D + pad, {}
        for x in reversed(order):
            self.st[x] = step
            step *= size[x]
        self.n = shift + step
        flat = np.full(self.n, 3, raw.dtype)
        self.index = shift + sum(np.arange(size[x]).reshape([-1 if y == x else 1 for y in "bsh"] + [1])
                                 * self.st[x] for x in "bsh") + np.arange(D)
        if fill is None:
            flat[self.index] = raw
        self.buf = DevBuf.of(flat)

    @property
    def addr(self):
        return self.buf.addr + self.shift * self.dtype.itemsize

    @property
    def strides(self):
        return _lib.strides([self.st[x] for x in "bhs"])

    def get(self):
        flat = self.buf.get((self.n,), self.dtype)
        rest = np.ones(self.n, bool)
        rest[self.index] = False
        assert (flat[rest] == 3).all()
        return flat[self.index]


def rope(q, k, positions, freqs, axis, dtype, interleaved=False, inverse=False, counts=None,
         layout=("bsh", 0, 0), in_place=False, shared=False, axes=None):
    """(q_out, k_out) raw [B, S, H, D]."""
    from devmem import DevBuf
    B, S, _, D = q.shape
    order, pad, shift = layout
    vq, vk = View(q, order, pad, shift), View(k, order, pad, shift)
    oq = vq if in_place else View(q, "bhs", pad, shift, fill=3)
    ok = vk if in_place else View(k, "bhs", pad, shift, fill=3)
    A = positions.shape[-1]
    pd = DevBuf.of(positions.astype(np.int32))
    fd, ad = DevBuf.of(freqs.astype(np.float64)), DevBuf.of(axis.astype(np.uint8))
    cd = None if counts is None else DevBuf.of(np.asarray(counts, np.int32))
    _lib.check(_lib.load().anima_hip_rope_axes_dev(
        vq.addr, vq.strides, oq.addr, oq.strides, q.shape[2], vk.addr, vk.strides, ok.addr,
        ok.strides, k.shape[2], pd.addr, 0 if shared else S * A, cd.addr if cd else None, fd.addr,
        ad.addr, A, len(freqs), B, S, D, dtype, interleaved, inverse, None), "rope_axes")
    return oq.get(), ok.get()


def check(got, x, positions, freqs, axis, dtype, interleaved, inverse, counts=None):
    B, S = x.shape[:2]
    want = ref.rotate(x, positions, freqs, axis, interleaved, inverse)
    P = len(freqs)
    theta = np.abs(positions[..., np.minimum(axis, positions.shape[-1] - 1)] * freqs)[:, :, None]
    a = np.abs(x[..., 0:2 * P:2] if interleaved else x[..., :P])
    b = np.abs(x[..., 1:2 * P:2] if interleaved else x[..., P:2 * P])
    tol = (a + b) * (TOL + theta * 2.0 ** -51)
    both = np.stack([tol, tol], -1).reshape(*x.shape[:3], -1) if interleaved else \
        np.concatenate([tol, tol], -1)
    full = np.zeros(x.shape)
    full[..., :2 * P] = both + ref.HALF[dtype] * np.abs(want[..., :2 * P]) if dtype == ref.BF16 \
        else both
    seen = np.ones((B, S), bool) if counts is None else \
        np.arange(S) < np.asarray(counts)[:, None]
    val = ref.untyped(got, dtype)
    err = np.abs(val - want)
    assert (err <= full)[seen].all(), (err - full)[seen].max()
    assert (got[~seen] == 3).all()


def inputs(B, S, H, D, axes, P, dtype, seed, far=200):
    rng = np.random.default_rng(seed)
    q, qv = ref.typed(rng.standard_normal((B, S, H[0], D)), dtype)
    k, kv = ref.typed(rng.standard_normal((B, S, H[1], D)), dtype)
    pos = rng.integers(-far, far, (B, S, axes)).astype(np.int64)
    freqs = 10.0 ** -(4.0 * rng.permutation(P) / P)
    return (q, k), (qv, kv), pos, freqs, rng.integers(0, axes, P)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,H,D,axes,P,layout", [
    (1, 1, (1, 1), 2, 1, 1, ("bsh", 0, 0)),
    (8, 1, (16, 4), 128, 1, 64, ("bsh", 0, 0)),
    (2, 77, (16, 16), 128, 3, 64, ("bsh", 0, 0)),
    (3, 33, (5, 1), 64, 3, 24, ("bhs", 8, 8)),
    (2, 19, (4, 2), 44, 2, 22, ("shb", 0, 0)),
    (1, 130, (3, 3), 80, 4, 17, ("bsh", 1, 3)),
    (2, 9, (24, 1), 256, 3, 128, ("hbs", 0, 0)),
    (1, 3, (2, 1), 1024, 3, 512, ("bsh", 0, 0)),
    (1, 5, (2, 1), 1023, 2, 300, ("bsh", 0, 0)),
    (1, 600, (1, 1), 8, 1, 4, ("bsh", 0, 0))])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, False), (False, True),
                                                 (True, True)])
def test_rope(B, S, H, D, axes, P, layout, interleaved, inverse, dtype):
    raw, val, pos, freqs, axis = inputs(B, S, H, D, axes, P, dtype, S + D)
    got = rope(*raw, pos, freqs, axis, dtype, interleaved, inverse, layout=layout)
    for g, v in zip(got, val):
        check(g, v, pos, freqs, axis, dtype, interleaved, inverse)
    again = rope(*raw, pos, freqs, axis, dtype, interleaved, inverse, layout=layout, in_place=True)
    for g, w in zip(again, got):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("dtype", TYPES)
def test_counts_shared_positions_and_missing_heads(dtype):
    raw, val, pos, freqs, axis = inputs(3, 11, (4, 2), 64, 2, 32, dtype, 1)
    counts = [11, 0, 4]
    got = rope(*raw, pos, freqs, axis, dtype, counts=counts)
    for g, v in zip(got, val):
        check(g, v, pos, freqs, axis, dtype, False, False, counts)
    got = rope(*raw, pos[:1], freqs, axis, dtype, shared=True)
    for g, v in zip(got, val):
        check(g, v, np.repeat(pos[:1], 3, 0), freqs, axis, dtype, False, False)
    none = raw[1][:, :, :0]
    got = rope(raw[0], none, pos, freqs, axis, dtype)
    check(got[0], val[0], pos, freqs, axis, dtype, False, False)
    got = rope(none, raw[1], pos, freqs, axis, dtype)
    check(got[1], val[1], pos, freqs, axis, dtype, False, False)


def test_far_positions_and_axes_past_the_last():
    raw, val, pos, freqs, axis = inputs(2, 40, (3, 1), 64, 3, 32, ref.F32, 2, far=2 ** 31)
    pos[0, 0], pos[0, 1] = 2 ** 31 - 1, -2 ** 31
    axis[5] = 200  # counts as the last axis
    got = rope(*raw, pos, freqs, axis, ref.F32)
    for g, v in zip(got, val):
        check(g, v, pos, freqs, axis, ref.F32, False, False)


def test_infinities_and_nan_stay_in_their_pairs():
    raw, val, pos, freqs, axis = inputs(1, 4, (2, 1), 64, 1, 32, ref.F32, 3)
    clean = rope(*raw, pos, freqs, axis, ref.F32)
    raw[0][0, 1, 1, 7], raw[0][0, 2, 0, 40] = np.inf, np.nan
    got = rope(*raw, pos, freqs, axis, ref.F32)
    bad = np.zeros(raw[0].shape, bool)
    bad[0, 1, 1, [7, 39]] = bad[0, 2, 0, [40, 8]] = True
    assert not np.isfinite(got[0][bad]).any()
    np.testing.assert_array_equal(got[0][~bad], clean[0][~bad])
    np.testing.assert_array_equal(got[1], clean[1])


def test_turn_and_back_and_gradient():
    """The inverse undoes the turn, and is its transpose: <y, R x> = <R^-1 y, x>."""
    raw, val, pos, freqs, axis = inputs(2, 30, (4, 2), 64, 3, 20, ref.F32, 4)
    there = rope(*raw, pos, freqs, axis, ref.F32)
    back = rope(*there, pos, freqs, axis, ref.F32, inverse=True)
    for b, v in zip(back, val):
        # |R x| <= |a| + |b| elementwise, off by TOL of it twice.
        assert np.abs(b - v).max() <= 2 * 2 * TOL * 2 * np.abs(v).max()
    rng = np.random.default_rng(8)
    g = [np.float32(rng.standard_normal(r.shape)) for r in raw]
    grad = rope(*g, pos, freqs, axis, ref.F32, inverse=True)
    for i in range(2):
        a = np.sum(g[i].astype(np.float64) * there[i])
        b = np.sum(grad[i].astype(np.float64) * raw[i])
        size = np.sum(np.abs(g[i]) * np.abs(raw[i])) * 2
        assert abs(a - b) <= 4 * TOL * size


def test_equals_the_table_of_an_image_grid():
    """The DiT's own 3D table on a (t, h, w) grid: the prologue's rotation, which reads it, and this
    one, from the grid's positions.  The table's angles are rounded to f32: 24 * 2^-24 at most, and
    its frequencies by some 2^-22 of them."""
    from devmem import DevBuf
    T, Hh, W, D, heads = 2, 5, 7, 128, 3
    table = generate_rope_freqs(Hh, W, T, D)
    S = T * Hh * W
    rng = np.random.default_rng(6)
    q = np.float32(rng.standard_normal((1, S, heads, D)))
    xd, od, fd = DevBuf.of(q), DevBuf(q.nbytes), DevBuf.of(table)
    st = _lib.strides([S * heads * D, D, heads * D])
    import ctypes as ct
    _lib.check(_lib.load().anima_hip_qk_prologue_dev(xd.addr, od.addr, None, fd.addr, 1, S, heads, D,
                                                     st, st, ct.c_float(1e-6), 0, None), "prologue")
    want = od.get(q.shape)
    dh = D // 6 * 2
    dt = D - 2 * dh
    sp = 1e4 * 4.0 ** (dh / (dh - 2))
    freqs = np.concatenate([1e4 ** -(np.arange(0, dt, 2) / dt), sp ** -(np.arange(0, dh, 2) / dh),
                            sp ** -(np.arange(0, dh, 2) / dh)])
    axis = np.repeat([0, 1, 2], [dt // 2, dh // 2, dh // 2])
    pos = np.stack(np.meshgrid(np.arange(T), np.arange(Hh), np.arange(W), indexing="ij"),
                   -1).reshape(1, S, 3)
    got, _ = rope(q, q[:, :, :0], pos, freqs, axis, ref.F32)
    np.testing.assert_allclose(got, want, rtol=0, atol=2 * np.abs(q).max() * (TOL + 7 * 2.0 ** -21))
