"""The 8-bit operators together, as a program uses them: the residual's addition and norm into 8-bit
rows, one product for queries, keys and values, their rotation in place in its columns, keys and
values into the 4-bit cache, attention, the output packed and projected; and the numpy classes.

Tolerances: each step is held to 64-bit numpy on the step's own inputs with the bounds of
test_gpu_fp8.py, test_gpu_rope_axes.py and test_gpu_kv4.py, or the whole chain to its eager run bit
for bit.
"""
import ctypes as ct

import numpy as np
import pytest

import fp8_ref as ref
import mx4_ref
import test_gpu_fp8 as fp8t
import test_gpu_kv4 as kv4
import test_gpu_rope_axes as ropet
from anima_hip import FP8Linear, _lib, fp8, rope_axes, rt
from anima_hip.rope import generate_rope_freqs
from test_mx4_classes_cpu import in_threads

pytestmark = pytest.mark.gpu

W, H, H_KV, D, P = 640, 4, 2, 128, 48  # model width, heads, K/V heads, head width, pairs turned
QKV = (H + 2 * H_KV) * D
EPS = 1e-6
FREQS = 1e4 ** (-np.arange(P) / P)
AXIS = (np.arange(P) % 3).astype(np.uint8)


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


class Layer:
    """One layer's weights, cache and buffers; step() enqueues one token of every sequence."""

    def __init__(self, dtype, B, S_max, seed):
        from devmem import DevBuf
        rng = np.random.default_rng(seed)
        self.dtype, self.B, self.S_max, self.lib = dtype, B, S_max, _lib.load()
        self.size = 4 if dtype == ref.F32 else 2
        self.w = {}
        for name, n, k in (("qkv", QKV, W), ("o", W, H * D)):
            packed = ref.pack(np.float32(rng.standard_normal((n, k)) * 0.04).astype(float))
            self.w[name] = (*(DevBuf.of(a) for a in packed), n, k, packed)
        self.norm_w = np.float32(1 + 0.2 * rng.standard_normal(W))
        self.cache = kv4.Cache(B, H_KV, S_max, D)
        self.nw, self.freqs, self.axis = (DevBuf.of(a) for a in (self.norm_w, FREQS, AXIS))
        self.x, self.stream_ = DevBuf(B * W * self.size), DevBuf(B * W * self.size)
        self.rows = {n: [DevBuf(B * b) for b in ref.sizes(k)] for n, k in (("x", W), ("att", H * D))}
        self.qkv, self.att = DevBuf(B * QKV * self.size), DevBuf(B * H * D * self.size)
        self.turned = DevBuf(B * H * D * self.size)
        self.pos = DevBuf(B * 3 * 4)
        self.starts, self.lens = kv4.ints([0] * B), kv4.ints([0] * B)
        self.need = max([self.lib.anima_hip_linear_fp8_scratch_bytes(B, w[2], w[3], dtype)
                         for w in self.w.values()]
                        + [self.lib.anima_hip_kv4_attention_scratch_bytes(B, 1, H, H_KV, D, S_max,
                                                                          dtype)])
        self.scratch = DevBuf(max(self.need, 16))

    def linear(self, name, rows, dst, stream):
        codes, scales, n, k, _ = self.w[name]
        _lib.check(self.lib.anima_hip_linear_fp8_dev(
            rows[0].addr, rows[1].addr, codes.addr, scales.addr, dst.addr, n, self.B, n, k,
            self.dtype, self.scratch.addr, self.need, stream), "linear")

    def step(self, stream=None):
        """x + stream -> stream; its norm -> qkv -> rotation -> cache -> attention -> x."""
        B, e = self.B, self.size
        _lib.check(self.lib.anima_hip_add_rmsnorm_fp8_dev(
            self.x.addr, W, self.stream_.addr, W, self.nw.addr, ct.c_float(EPS), self.dtype,
            self.stream_.addr, W, None, W, *(b.addr for b in self.rows["x"]), B, W, stream), "norm")
        self.linear("qkv", self.rows["x"], self.qkv, stream)
        k, v = self.qkv.addr + H * D * e, self.qkv.addr + (H + H_KV) * D * e
        col = _lib.strides((QKV, D, QKV))
        row = _lib.strides((H * D, D, H * D))
        # Queries into rows of their own, keys where they are.
        _lib.check(self.lib.anima_hip_rope_axes_dev(
            self.qkv.addr, col, self.turned.addr, row, H, k, col, k, col, H_KV, self.pos.addr, 3,
            None, self.freqs.addr, self.axis.addr, 3, P, B, 1, D, self.dtype, False, False, stream),
            "rope")
        _lib.check(self.lib.anima_hip_kv4_append_dev(
            k, v, self.dtype, col, col, *self.cache.addrs, self.starts.addr, None, B, 1, H_KV, D,
            self.S_max, stream), "append")
        _lib.check(self.lib.anima_hip_kv4_attention_dev(
            self.turned.addr, self.dtype, row, *self.cache.addrs, self.lens.addr, None,
            self.att.addr, row, B, B, 1, H, H_KV, D, self.S_max, ct.c_float(D ** -0.5), True,
            self.scratch.addr, self.need, stream), "attention")
        _lib.check(self.lib.anima_hip_fp8_pack_dev(
            self.att.addr, H * D, self.dtype, *(b.addr for b in self.rows["att"]), B, H * D, stream),
            "pack")
        self.linear("o", self.rows["att"], self.x, stream)

    def place(self, lens, pos):
        self.starts.put(np.array(lens, np.int32), 0)
        self.lens.put(np.array(lens, np.int32) + 1, 0)
        self.pos.put(np.asarray(pos, np.int32), 0)

    def raw(self, buf, cols):
        return buf.get((self.B, cols), np.float32 if self.dtype == ref.F32 else np.uint16)

    def read(self, buf, cols):
        return ref.untyped(self.raw(buf, cols), self.dtype)

    def packed(self, name, k):
        return tuple(b.get((self.B, n), np.uint8) for b, n in zip(self.rows[name], ref.sizes(k)))


def start(layer, seed):
    rng = np.random.default_rng(seed)
    for buf, s in ((layer.x, 1.0), (layer.stream_, 4.0)):
        buf.put(ref.typed(rng.standard_normal((layer.B, W)) * s, layer.dtype)[0], 0)


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
def test_steps(dtype):
    """Tokens one after another, ragged sequences at far places on three axes: every step of the
    chain against 64 bits."""
    B, S_max = 3, 90
    layer = Layer(dtype, B, S_max, 1)
    start(layer, 2)
    lens = [0, 30, 80]
    rng = np.random.default_rng(5)
    old, _ = ref.typed(rng.standard_normal((B, S_max, H_KV, D)), dtype)
    kv4.append(layer.cache, old, old[:, ::-1].copy(), dtype, [0] * B, lens)
    for i in range(3):
        pos = rng.integers(0, 100000, (B, 3))
        layer.place(lens, pos)
        x, r = layer.read(layer.x, W), layer.read(layer.stream_, W)
        layer.step()
        rows = layer.packed("x", W)
        fp8t.check_norm({"s": layer.raw(layer.stream_, W), "c": rows}, x, r, layer.norm_w, EPS, dtype)
        qkv = layer.read(layer.qkv, QKV)
        fresh = fp8t.linear_dev(rows, layer.w["qkv"][4], W, dtype)  # keys before their turn
        fp8t.check_linear(fresh, rows, layer.w["qkv"][4], W, dtype)
        keep = np.r_[0:H * D, (H + H_KV) * D:QKV]
        np.testing.assert_array_equal(qkv[:, keep], fresh[:, keep])
        q = layer.raw(layer.turned, H * D).reshape(B, 1, H, D)
        kt = layer.raw(layer.qkv, QKV)[:, H * D:(H + H_KV) * D].reshape(B, 1, H_KV, D)
        for got, src, h in ((q, fresh[:, :H * D], H), (kt, fresh[:, H * D:(H + H_KV) * D], H_KV)):
            ropet.check(got, src.reshape(B, 1, h, D), pos[:, None], FREQS, AXIS.astype(int), dtype,
                        False, False)
        keys, values = layer.cache.values()
        new = {"k": ref.untyped(kt, dtype)[:, 0], "v": qkv[:, (H + H_KV) * D:].reshape(B, H_KV, D)}
        for b in range(B):
            for t, cached in ((new["k"], keys), (new["v"], values)):
                np.testing.assert_array_equal(cached[b, :, lens[b]],
                                              mx4_ref.unpack(*mx4_ref.pack(t[b]), D))
        lens = [n + 1 for n in lens]
        qv = ref.untyped(q, dtype)
        want, mag = mx4_ref.attention(qv, keys, values, lens, None, True, D ** -0.5)
        d = (3 * D + 6) * kv4.U * D ** -0.5 * np.abs(qv).sum(-1, keepdims=True) * np.nanmax(
            np.abs(keys))
        bound = (4 * d + (S_max + 64) * kv4.U + (2.0 ** -8 if dtype == ref.BF16 else 0.0)) * mag \
            + ref.HALF[dtype] * np.abs(want) + 1e-30
        att = layer.read(layer.att, H * D)
        assert (np.abs(att.reshape(want.shape) - want) <= bound).all()
        rows = layer.packed("att", H * D)
        for got, exact in zip(rows, ref.pack(att)):
            np.testing.assert_array_equal(got, exact)
        fp8t.check_linear(layer.read(layer.x, W), rows, layer.w["o"][4], H * D, dtype)


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
def test_captured_steps(dtype):
    """Two layers' steps captured into a graph each, replayed in turn for token after token with
    eager work between: the outputs and caches of the eager run, bit for bit."""
    from devmem import CapturedCall
    B, S_max, steps = 2, 40, 4
    pos = np.random.default_rng(8).integers(0, 5000, (steps, B, 3))

    def run(captured):
        layers = [Layer(dtype, B, S_max, seed) for seed in (1, 2)]
        for layer in layers:
            start(layer, 3)
            old, _ = ref.typed(np.random.default_rng(4).standard_normal((B, 9, H_KV, D)), dtype)
            kv4.append(layer.cache, old, old, dtype, [0] * B, [0, 9])
            layer.place([0, 9], pos[0])
        calls = [CapturedCall(layer.step) if captured else None for layer in layers]
        out = []
        for i in range(steps):
            for layer, call in zip(layers, calls):
                layer.place([i, 9 + i], pos[i])
                if captured:
                    call.replay()
                    fp8.pack(np.ones((3, 200), np.float32))  # eager work between the replays
                else:
                    layer.step()
                out.append((layer.raw(layer.x, W), layer.raw(layer.stream_, W)))
        caches = [layer.cache.raw() for layer in layers]
        for call in calls:
            if call:
                call.close()
        return out, caches

    eager, again = run(False), run(True)
    for a, b in zip(eager[0], again[0]):
        for u, v in zip(a, b):
            assert np.isfinite(ref.untyped(u, dtype)).all()
            np.testing.assert_array_equal(u, v)
    for a, b in zip(eager[1], again[1]):
        for (c1, s1), (c2, s2) in zip(a, b):
            np.testing.assert_array_equal(c1, c2)
            np.testing.assert_array_equal(s1, s2)


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
def test_numpy_functions(dtype):
    rng = np.random.default_rng(6)
    wr, wv = ref.typed(rng.standard_normal((300, W)) * 0.05, dtype)
    lin = FP8Linear(wr)
    packed = fp8.pack(wr)
    for got, want in zip(packed, ref.pack(wv)):
        np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(fp8.unpack(*packed, W), ref.unpack(*packed, W))
    xr, x = ref.typed(rng.standard_normal((2, 5, W)), dtype)
    y = lin(xr)
    assert y.shape == (2, 5, 300) and y.dtype == xr.dtype
    fp8t.check_linear(ref.untyped(y, dtype).reshape(10, 300), ref.pack(x.reshape(10, W)), packed, W,
                      dtype)
    rr, r = ref.typed(rng.standard_normal((2, 5, W)) * 3, dtype)
    nw = np.float32(1 + 0.1 * rng.standard_normal(W))
    s, n = fp8.add_rmsnorm(xr, rr, nw, EPS)
    fp8t.check_norm({"s": s.reshape(10, W), "y": n.reshape(10, W)}, x.reshape(10, W),
                    r.reshape(10, W), nw, EPS, dtype)
    y, h = lin.after_norm(xr, rr, nw, EPS)
    np.testing.assert_array_equal(h, s)
    rows = fp8t.norm_dev(xr.reshape(10, W), rr.reshape(10, W), nw, EPS, dtype, "c")["c"]
    fp8t.check_linear(ref.untyped(y, dtype).reshape(10, 300), rows, packed, W, dtype)
    assert lin(xr[:0]).shape == (0, 5, 300)
    for bad in (lambda: lin(xr[..., :W - 1]), lambda: fp8.pack(xr), lambda: FP8Linear(wr[0]),
                lambda: fp8.unpack(packed[0], packed[1][:-1], W),
                lambda: lin.after_norm(xr, rr[:1]), lambda: lin.after_norm(xr, rr, nw[1:]),
                lambda: fp8.add_rmsnorm(xr, rr.astype(np.float64 if dtype == ref.BF16 else np.uint16))):
        with pytest.raises(ValueError):
            bad()


def test_numpy_rotation():
    """`rotate` over an image grid of `grid_axes`: the DiT's own table's turn (its angles are rounded
    to f32: 24 * 2^-24 at most, its frequencies by some 2^-22 of them), and back."""
    T, Hh, Wd = 2, 5, 7
    S = T * Hh * Wd
    rng = np.random.default_rng(7)
    q, k = (np.float32(rng.standard_normal((2, S, h, D))) for h in (3, 1))
    grid = rope_axes.grid_axes(Hh, Wd, T, D)
    qt, kt = rope_axes.rotate(q, k, *grid)
    table = generate_rope_freqs(Hh, Wd, T, D).astype(np.float64)
    for x, got in ((q, qt), (k, kt)):
        a, b = x[..., :D // 2].astype(float), x[..., D // 2:].astype(float)
        m = table[:, None]
        want = np.concatenate([m[..., 0, 0] * a + m[..., 0, 1] * b,
                               m[..., 1, 0] * a + m[..., 1, 1] * b], -1)
        np.testing.assert_allclose(got, want, rtol=0,
                                   atol=2 * np.abs(x).max() * (ropet.TOL + 7 * 2.0 ** -21))
    back, none = rope_axes.rotate(qt, None, *grid, inverse=True)
    assert none.shape == (2, S, 0, D)
    np.testing.assert_allclose(back, q, rtol=0, atol=4 * np.abs(q).max() * ropet.TOL)
    bits = ref.bits_of(q)
    far = np.arange(2 * S).reshape(2, S, 1) * 100000
    turned, _ = rope_axes.rotate(bits, None, far, FREQS, interleaved=True)
    ropet.check(turned, ref.values_of(bits), far, FREQS, np.zeros(P, int), ref.BF16, True, False)
    for args in ((q[0], None, *grid), (q, k[:1], *grid), (q, ref.bits_of(k), *grid),
                 (q, k, grid[0][:, :-1], *grid[1:]), (q, k, grid[0] * 0.5, *grid[1:]),
                 (q, k, grid[0].astype(np.int64) + 2 ** 31, *grid[1:]), (q, k, grid[0], grid[1], [3]),
                 (q, k, grid[0], grid[1], np.full(D // 2, 3))):
        with pytest.raises(ValueError):
            rope_axes.rotate(*args)
    with pytest.raises(_lib.AnimaHipError, match="pairs"):
        rope_axes.rotate(q, k, grid[0], np.ones(D))


def test_linear_from_a_weight_store(tmp_path):
    """Weights packed from the memory-mapped file's device copies."""
    import safetensors_file
    rng = np.random.default_rng(11)
    w = np.float32(rng.standard_normal((96, 160)) * 0.1)
    path = str(tmp_path / "w.safetensors")
    safetensors_file.write(path, {"net.a.weight": ("BF16", ref.bits_of(w)), "net.b.weight": ("F32", w)})
    with rt.Weights(path) as store:
        for name, values in (("a.weight", ref.values_of(ref.bits_of(w))), ("b.weight", w)):
            lin = FP8Linear.from_store(store, name)
            x = np.float32(rng.standard_normal((3, 160)))
            fp8t.check_linear(lin(x).astype(float), ref.pack(x.astype(float)),
                              ref.pack(values.astype(np.float64)), 160, ref.F32)


def test_threads_share_a_layer():
    """One layer under six threads, calls of different sizes: each result is the one it has alone."""
    rng = np.random.default_rng(2)
    lin = FP8Linear(np.float32(rng.standard_normal((256, 5120)) * 0.05))
    xs = [np.float32(rng.standard_normal((3 + 17 * i, 5120))) for i in range(6)]
    want = [(lin(x), *lin.after_norm(x)) for x in xs]
    for _ in range(3):
        for got, alone in zip(in_threads(6, lambda i: (lin(xs[i]), *lin.after_norm(xs[i]))), want):
            for a, b in zip(got, alone):
                np.testing.assert_array_equal(a, b)
