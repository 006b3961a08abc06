"""The 4-bit operators together, as a program uses them: a layer's projections with 4-bit weights,
the new token's keys and values into the 4-bit cache, attention over it, the output projection; and
the numpy classes over them.

Tolerances: each step is held to 64-bit numpy on the step's own inputs with the bounds of
test_gpu_mx4.py and test_gpu_kv4.py, or the whole chain to its eager run bit for bit.
"""
import ctypes as ct

import numpy as np
import pytest

import mx4_ref as ref
import test_gpu_kv4 as kv4
from anima_hip import KV4Cache, MX4Linear, _lib, mx4, rt

pytestmark = pytest.mark.gpu

W, H, H_KV, D = 512, 4, 2, 128  # model width, heads, K/V heads, head width


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


class Layer:
    """Projections and cache of one layer on the device; step() enqueues one token's work."""

    def __init__(self, dtype, B, S_max, rng):
        from devmem import DevBuf
        self.dtype, self.B, self.S_max = dtype, B, S_max
        self.lib = _lib.load()
        size = 4 if dtype == ref.F32 else 2
        self.w = {}
        for name, n, k in (("q", H * D, W), ("k", H_KV * D, W), ("v", H_KV * D, W),
                           ("o", W, H * D)):
            codes, scales = ref.pack(np.float32(rng.standard_normal((n, k)) * 0.05).astype(float))
            self.w[name] = (DevBuf.of(codes), DevBuf.of(scales), n, k, codes, scales)
        self.cache = kv4.Cache(B, H_KV, S_max, D)
        self.x = DevBuf(B * W * size)
        self.buf = {n: DevBuf(B * self.w[n][2] * size) for n in "qkvo"}
        self.att = DevBuf(B * H * D * size)
        self.starts, self.lens = kv4.ints([0] * B), kv4.ints([0] * B)
        need = max([self.lib.anima_hip_linear_mx4_scratch_bytes(B, w[2], w[3], dtype)
                    for w in self.w.values()]
                   + [self.lib.anima_hip_kv4_attention_scratch_bytes(B, 1, H, H_KV, D, S_max, dtype)])
        self.need, self.scratch = need, DevBuf(max(need, 16))

    def linear(self, name, src, dst, stream):
        codes, scales, n, k = self.w[name][:4]
        _lib.check(self.lib.anima_hip_linear_mx4_dev(
            src.addr, k, codes.addr, scales.addr, dst.addr, n, self.B, n, k, self.dtype,
            self.scratch.addr, self.need, stream), "linear")

    def step(self, stream=None):
        for n in "qkv":
            self.linear(n, self.x, self.buf[n], stream)
        one = _lib.strides((H_KV * D, D, H_KV * D))
        _lib.check(self.lib.anima_hip_kv4_append_dev(
            self.buf["k"].addr, self.buf["v"].addr, self.dtype, one, one, *self.cache.addrs,
            self.starts.addr, None, self.B, 1, H_KV, D, self.S_max, stream), "append")
        row = _lib.strides((H * D, D, H * D))
        _lib.check(self.lib.anima_hip_kv4_attention_dev(
            self.buf["q"].addr, self.dtype, row, *self.cache.addrs, self.lens.addr, None,
            self.att.addr, row, self.B, self.B, 1, H, H_KV, D, self.S_max,
            ct.c_float(D ** -0.5), True, self.scratch.addr, self.need, stream), "attention")
        self.linear("o", self.att, self.buf["o"], stream)

    def feed(self, raw, lens):
        self.x.put(raw, 0)
        self.starts.put(np.array(lens, np.int32), 0)
        self.lens.put(np.array(lens, np.int32) + 1, 0)

    def read(self, buf, cols):
        raw = buf.get((self.B, cols), np.float32 if self.dtype == ref.F32 else np.uint16)
        return ref.untyped(raw, self.dtype)


def check_product(got, a, codes, scales, K, dtype):
    w = ref.unpack(codes, scales, K)
    want, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    n = K * (3 if dtype == ref.F32 else 1) + 32
    assert (np.abs(got - want) <= n * kv4.U * mag + ref.HALF[dtype] * np.abs(want)).all()


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
def test_decoding_steps(dtype):
    """Tokens one after another, ragged sequences: every step of the chain against 64 bits."""
    rng = np.random.default_rng(1)
    B, S_max = 3, 700
    layer = Layer(dtype, B, S_max, rng)
    lens = [0, 40, 690]
    old = rng.standard_normal((B, S_max, H_KV, D))
    raw, _ = ref.typed(old, dtype)
    kv4.append(layer.cache, raw, raw[:, ::-1].copy(), dtype, [0] * B, lens)
    for _ in range(4):
        xr, x = ref.typed(rng.standard_normal((B, W)), dtype)
        layer.feed(xr, lens)
        layer.step()
        got = {n: layer.read(layer.buf[n], layer.w[n][2]) for n in "qkvo"}
        att = layer.read(layer.att, H * D)
        for n in "qkv":
            check_product(got[n], x, *layer.w[n][4:], W, dtype)
        k, v = layer.cache.values()
        for b in range(B):
            for new, cached in ((got["k"], k), (got["v"], v)):
                rows = new[b].reshape(H_KV, D)
                np.testing.assert_array_equal(cached[b, :, lens[b]], ref.unpack(*ref.pack(rows), D))
        lens = [n + 1 for n in lens]
        q = got["q"].reshape(B, 1, H, D)
        want, mag = ref.attention(q, k, v, lens, None, True, D ** -0.5)
        d = (3 * D + 6) * kv4.U * D ** -0.5 * np.abs(q).sum(-1, keepdims=True) * np.nanmax(np.abs(k))
        r = 2.0 ** -8 if dtype == ref.BF16 else 0.0
        bound = (4 * d + (S_max + 64) * kv4.U + r) * mag + ref.HALF[dtype] * np.abs(want) + 1e-30
        assert (np.abs(att.reshape(want.shape) - want) <= bound).all()
        check_product(got["o"], att, *layer.w["o"][4:], H * D, dtype)


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
def test_captured_step(dtype):
    """One step captured into a HIP graph and replayed for token after token, eager work between
    the replays: the outputs and the cache of the eager run, bit for bit."""
    from devmem import CapturedCall
    B, S_max, steps = 2, 600, 5
    xs = [ref.typed(np.random.default_rng(9 + i).standard_normal((B, W)), dtype)[0]
          for i in range(steps)]

    def run(captured):
        layer = Layer(dtype, B, S_max, np.random.default_rng(2))
        lens, out = [0, 500], []
        start, _ = ref.typed(np.random.default_rng(4).standard_normal((B, 500, H_KV, D)), dtype)
        kv4.append(layer.cache, start, start, dtype, [0] * B, lens)
        call = CapturedCall(layer.step) if captured else None
        for x in xs:
            layer.feed(x, lens)
            if captured:
                call.replay()
                kv4.append(kv4.Cache(1, 1, 4, D), start[:1, :1, :1], start[:1, :1, :1], dtype, [1])
            else:
                layer.step()
            out.append(layer.read(layer.buf["o"], W))
            lens = [n + 1 for n in lens]
        raw = layer.cache.raw()
        if captured:
            call.close()
        return out, raw

    eager, cache = run(False)
    again, cache2 = run(True)
    for a, b in zip(eager, again):
        assert np.isfinite(a).all()
        np.testing.assert_array_equal(a, b)
    for (c1, s1), (c2, s2) in zip(cache, cache2):
        np.testing.assert_array_equal(c1, c2)
        np.testing.assert_array_equal(s1, s2)


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
def test_numpy_classes(dtype):
    """MX4Linear and KV4Cache: a prompt of ragged lengths, then single tokens, then a shared
    context; the values they hold and the results against 64 bits."""
    rng = np.random.default_rng(6)
    wr, wv = ref.typed(rng.standard_normal((300, W)) * 0.05, dtype)
    lin = MX4Linear(wr)
    codes, scales = mx4.pack(wr)
    want = ref.pack(wv)
    np.testing.assert_array_equal(codes, want[0])
    np.testing.assert_array_equal(scales, want[1])
    np.testing.assert_array_equal(mx4.unpack(codes, scales, W), ref.unpack(codes, scales, W))
    xr, x = ref.typed(rng.standard_normal((2, 5, W)), dtype)
    y = lin(xr)
    assert y.shape == (2, 5, 300) and y.dtype == xr.dtype
    check_product(ref.untyped(y, dtype).reshape(10, 300), x.reshape(10, W), codes, scales, W, dtype)
    assert lin(xr[:0]).shape == (0, 5, 300)

    cache = KV4Cache(2, H_KV, D, 64)
    k0, _ = ref.typed(rng.standard_normal((2, 40, H_KV, D)), dtype)
    cache.append(k0, k0[:, ::-1], counts=[40, 17])
    cache.append(k0[:, :1], k0[:, 1:2])
    assert cache.lens.tolist() == [41, 18]
    qr, q = ref.typed(rng.standard_normal((2, 3, H, D)), dtype)
    out = ref.untyped(cache.attend(qr, counts=[3, 1]), dtype)
    k, v = (np.float64(t) for t in cache.values())
    want, mag = ref.attention(q, k, v, [41, 18], [3, 1], True, D ** -0.5)
    d = (3 * D + 6) * kv4.U * D ** -0.5 * np.abs(q).sum(-1, keepdims=True) * np.abs(k[0, :, :41]).max()
    r = 2.0 ** -8 if dtype == ref.BF16 else 0.0
    assert (np.abs(out - want) <= (4 * d + 128 * kv4.U + r) * mag
            + ref.HALF[dtype] * np.abs(want)).all()
    assert (out[1, 1:] == 0).all()
    with pytest.raises(ValueError, match="max_tokens"):
        cache.append(k0[:, :24], k0[:, :24])
    with pytest.raises(ValueError, match="counts"):
        cache.append(k0, k0, counts=[41, 0])
    with pytest.raises(ValueError, match="attend"):
        cache.attend(qr[:, :, :, :64])
    with pytest.raises(_lib.AnimaHipError, match="multiple"):
        cache.attend(np.ascontiguousarray(qr[:, :, :3]))
    shared = KV4Cache(1, H_KV, D, 64)
    shared.append(k0[:1], k0[:1])
    out = ref.untyped(shared.attend(qr, is_causal=False), dtype)
    k, v = (np.float64(t) for t in shared.values())
    want, mag = ref.attention(q, k, v, [40], None, False, D ** -0.5)
    assert (np.abs(out - want) <= (4 * d + 128 * kv4.U + r) * mag + 2 * ref.HALF[dtype]
            * np.abs(want)).all()


def test_linear_from_a_weight_store(tmp_path):
    """Weights packed from the memory-mapped file's device copies."""
    import safetensors_file
    rng = np.random.default_rng(11)
    w = np.float32(rng.standard_normal((96, 160)) * 0.1)
    path = str(tmp_path / "w.safetensors")
    safetensors_file.write(path, {"net.a.weight": ("BF16", ref.bits_of(w)), "net.b.weight": ("F32", w)})
    with rt.Weights(path) as store:
        for name, values in (("a.weight", ref.values_of(ref.bits_of(w))), ("b.weight", w)):
            lin = MX4Linear.from_store(store, name)
            codes, scales = ref.pack(values.astype(np.float64))
            x = np.float32(rng.standard_normal((3, 160)))
            check_product(lin(x).astype(float), x.astype(float), codes, scales, 160, ref.F32)
