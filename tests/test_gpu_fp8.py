"""The 8-bit rows on the GPU against 64-bit numpy: packing, the norm and the linear layer.

Packing is a function of the values and is compared byte for byte.

Norm: h is rounded to f32 once, which moves y by at most 2 * 2^-24 (itself, and through the mean);
the root is of 64 bits; y is rounded to f32 twice (times the root, times w).  So y is within
EPS = 4 * 2^-24 of the definition, relatively, before its own rounding.

Linear, C f32: |C - ref| <= n 2^-24 sum |a w| + 2^-24 |ref|, n = K + 16 additions (the products,
and the waves' or splits' partial sums).  C bf16: the adder cuts each of eight neighbouring products
off at 2^-13 of the largest one's power of two, so the other seven lose less than 7 * 2^-13 of the
largest together; that, over all eights, and 2^-8 |ref| are added.
"""
import ctypes as ct

import numpy as np
import pytest

import fp8_ref as ref
from anima_hip import _lib, rt

pytestmark = pytest.mark.gpu

TYPES = [ref.F32, ref.BF16]
EPS = 4 * 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


def rows_of(raw, ld, fill, shift=0):
    """Rows of a 2-D array ld elements apart in one flat buffer, `shift` elements in front."""
    buf = np.full((raw.shape[0], ld), fill, raw.dtype)
    buf[:, :raw.shape[1]] = raw
    return np.concatenate([np.zeros(shift, raw.dtype), buf.reshape(-1)])


def np_type(dtype):
    return np.float32 if dtype == ref.F32 else np.uint16


def pack_dev(raw, dtype, ld=None, shift=0):
    """Codes and scales through anima_hip_fp8_pack_dev; bytes past the outputs must stay."""
    from devmem import DevBuf
    rows, K = raw.shape
    ld = ld or K
    x = DevBuf.of(rows_of(raw, ld, 0x55, shift))
    n = [rows * b for b in ref.sizes(K)]
    out = [DevBuf.of(np.full(b + 64, 0xA5, np.uint8)) for b in n]
    _lib.check(_lib.load().anima_hip_fp8_pack_dev(x.addr + shift * raw.itemsize, ld, dtype,
                                                  out[0].addr, out[1].addr, rows, K, None), "pack")
    got = [o.get((b + 64,), np.uint8) for o, b in zip(out, n)]
    assert all((g[b:] == 0xA5).all() for g, b in zip(got, n))
    return [g[:b].reshape(rows, -1) for g, b in zip(got, n)]


def unpack_dev(codes, scales, K, dtype, ld=None):
    from devmem import DevBuf
    rows, ld = codes.shape[0], ld or K
    out = DevBuf.of(np.full((rows, ld), 7, np_type(dtype)))
    c, s = DevBuf.of(codes), DevBuf.of(scales)
    _lib.check(_lib.load().anima_hip_fp8_unpack_dev(c.addr, s.addr, out.addr, ld, dtype, rows, K,
                                                    None), "unpack")
    got = out.get((rows, ld), np_type(dtype))
    assert (got[:, K:] == 7).all()
    return ref.untyped(got[:, :K], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,ld,shift", [
    (1, 1, None, 0), (3, 127, None, 0), (5, 128, None, 0), (7, 129, 136, 0), (129, 68, None, 0),
    (33, 96, 104, 3), (64, 1000, 1001, 1), (257, 2048, None, 0), (1, 8192, None, 0),
    (17, 513, 520, 0), (9, 640, None, 8)])
def test_pack_and_unpack(rows, K, ld, shift, dtype):
    rng = np.random.default_rng(rows * 100 + K)
    x = rng.standard_normal((rows, K)) * np.exp2(rng.integers(-140, 126, (rows, 1)).astype(float))
    raw, val = ref.typed(np.clip(x, -3e38, 3e38), dtype)
    codes, scales = pack_dev(raw, dtype, ld, shift)
    want = ref.pack(val)
    np.testing.assert_array_equal(scales, want[1])
    np.testing.assert_array_equal(codes, want[0])
    for out_type in TYPES:
        got = unpack_dev(codes, scales, K, out_type, ld)
        np.testing.assert_array_equal(got, ref.unpack(codes, scales, K))


def test_pack_borders():
    """Ties, values next to them, zeros of both signs, the scales' ends, infinities and NaN: each
    group byte for byte, and values that pack unchanged."""
    mid = (ref.NUMBERS[1:] + ref.NUMBERS[:-1]) / 2
    rows = []
    for e in (-149, -135, -126, -117, -20, 0, 60, 110, 119):
        for part in (mid[:60], mid[60:], np.nextafter(np.float32(mid), np.float32(0))[60:],
                     np.nextafter(np.float32(mid), np.float32(999))[60:], ref.NUMBERS[:120]):
            for top in (448.0, np.nextafter(np.float32(448), np.float32(0)),
                        np.nextafter(np.float32(448), np.float32(999)), 224.0, 464.0):
                g = np.zeros(128)
                g[:len(part)] = np.minimum(part, top)
                g[::2] *= -1
                g[127] = top
                rows.append(np.float32(np.clip(g * 2.0 ** e, -3.4028234e38, 3.4028234e38)))
    rows += [np.zeros(128), -np.zeros(128), np.full(128, 3.4028235e38), np.full(128, 1e-45)]
    for bad in (np.inf, -np.inf, np.nan):
        g = np.linspace(-3, 3, 128)
        g[77] = bad
        rows.append(g)
    raw, val = ref.typed(np.stack(rows), ref.F32)
    codes, scales = pack_dev(raw, ref.F32)
    want = ref.pack(val)
    np.testing.assert_array_equal(scales, want[1])
    np.testing.assert_array_equal(codes, want[0])
    assert (scales[-3:, 0] == 255).all() and (codes[-3:] == 0).all()
    assert np.isnan(unpack_dev(codes[-3:], scales[-3:], 128, ref.BF16)).all()
    values = unpack_dev(codes[:-3], scales[:-3], 128, ref.BF16)
    np.testing.assert_array_equal(values, ref.unpack(codes[:-3], scales[:-3], 128))
    again = pack_dev(np.float32(values), ref.F32)
    np.testing.assert_array_equal(ref.unpack(*again, 128), values)


def test_unpack_every_scale_byte():
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    codes[:, 127] = codes[:, 255] = 0  # the two NaN codes, which the packer does not write
    scales = np.zeros((256, 4), np.uint8)
    scales[:, :2] = np.arange(256)[:, None]
    want = ref.unpack(codes, scales, 256)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(unpack_dev(codes, scales, 256, ref.F32), np.float32(want))


# ------------------------------------------------------------------ norm

def norm_dev(x, r, w, eps, dtype, outputs="syc", ld=None, shift=0, in_place=False):
    """{"s": sum, "y": y, "c": (codes, scales)} in raw types, those of `outputs`."""
    from devmem import DevBuf
    rows, K = x.shape
    ld = ld or K
    at = shift * x.itemsize
    xd = DevBuf.of(rows_of(x, ld, 1, shift))
    rd = None if r is None else DevBuf.of(rows_of(r, ld, 1, shift))
    wd = None if w is None else DevBuf.of(np.float32(w))
    blank = rows_of(np.full((rows, K), 7, x.dtype), ld, 7, shift)
    sd = (rd if in_place else DevBuf.of(blank)) if "s" in outputs else None
    yd = (xd if in_place else DevBuf.of(blank)) if "y" in outputs else None
    n = [rows * b for b in ref.sizes(K)]
    cd = [DevBuf.of(np.full(b + 64, 0xA5, np.uint8)) for b in n] if "c" in outputs else None

    def a(b):
        return None if b is None else b.addr + at

    _lib.check(_lib.load().anima_hip_add_rmsnorm_fp8_dev(
        a(xd), ld, a(rd), ld, wd.addr if wd else None, ct.c_float(eps), dtype, a(sd), ld, a(yd), ld,
        cd[0].addr if cd else None, cd[1].addr if cd else None, rows, K, None), "norm")
    out = {}
    for key, b in (("s", sd), ("y", yd)):
        if b is not None:
            got = b.get((shift + rows * ld,), x.dtype)[shift:].reshape(rows, ld)
            assert (got[:, K:] == (1 if in_place else 7)).all()
            out[key] = got[:, :K]
    if cd:
        got = [c.get((b + 64,), np.uint8) for c, b in zip(cd, n)]
        assert all((g[b:] == 0xA5).all() for g, b in zip(got, n))
        out["c"] = [g[:b].reshape(rows, -1) for g, b in zip(got, n)]
    return out


def check_norm(out, x, r, w, eps, dtype):
    h, y = ref.norm(x, r, w, eps)
    K = x.shape[1]
    if "s" in out:
        # An f32 sum, and its rounding.
        err = np.abs(ref.untyped(out["s"], dtype) - h)
        assert (err <= (ref.HALF[dtype] + 2.0 ** -24) * np.abs(h) + 1e-44).all()
    if "y" in out:
        err = np.abs(ref.untyped(out["y"], dtype) - y)
        tol = (EPS + (ref.HALF[ref.BF16] if dtype == ref.BF16 else 0.0)) * np.abs(y)
        assert (err <= tol + 1e-44).all()
    if "c" in out:
        codes, scales = out["c"]
        groups = codes.shape[1] // 128
        g = np.zeros((len(x), groups * 128))
        g[:, :K] = y
        top = np.abs(g).reshape(len(x), groups, 128).max(-1)
        s = scales[:, :groups].astype(int)
        assert (s >= ref.scale_bytes(top * (1 - EPS))).all()
        assert (s <= ref.scale_bytes(top * (1 + EPS))).all()
        assert (scales[:, groups:] == 0).all() and (codes[:, K:] == 0).all()
        unit = np.exp2(np.repeat(s, 128, -1)[:, :K] - 127.0)
        mag = np.abs(y) / unit
        step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(mag, 1e-30))), -6) - 3)
        err = np.abs(ref.unpack(codes, scales, K) - y) / unit
        # Half a step (of the power of two above, where the value is just below it).
        assert (err <= step * 0.5 * (1 + 1e-6) + EPS * mag).all()
    if dtype == ref.F32 and "c" in out and "y" in out:
        want = ref.pack(out["y"].astype(np.float64))
        np.testing.assert_array_equal(out["c"][0], want[0])
        np.testing.assert_array_equal(out["c"][1], want[1])


def norm_inputs(rows, K, dtype, seed):
    rng = np.random.default_rng(seed)
    size = np.exp2(rng.integers(-20, 20, (rows, 1)).astype(float))
    x = ref.typed(rng.standard_normal((rows, K)) * size, dtype)
    r = ref.typed(rng.standard_normal((rows, K)) * size * 3, dtype)
    return x, r, np.float32(1 + 0.3 * rng.standard_normal(K))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,ld,shift", [
    (1, 1, None, 0), (2, 127, None, 0), (5, 128, None, 0), (9, 500, 512, 0), (4, 512, None, 0),
    (3, 513, 520, 0), (1, 2048, None, 0), (33, 2048, None, 0), (6, 2050, 2051, 1),
    (3, 4096, None, 8), (2, 8190, None, 0), (2, 8193, None, 0), (2, 16384, None, 0),
    (1, 32768, None, 0), (2, 33001, 33008, 0)])
def test_norm(rows, K, ld, shift, dtype):
    (x, xv), (r, rv), w = norm_inputs(rows, K, dtype, rows + K)
    out = norm_dev(x, r, w, 1e-6, dtype, ld=ld, shift=shift)
    check_norm(out, xv, rv, w.astype(np.float64), 1e-6, dtype)


@pytest.mark.parametrize("outputs", ["s", "y", "c", "yc", "sc"])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_optional_arguments(outputs, dtype):
    (x, xv), (r, rv), w = norm_inputs(5, 700, dtype, 3)
    for rr, rrv in ((r, rv), (None, None)):
        for ww in (w, None):
            out = norm_dev(x, rr, ww, 1e-5, dtype, outputs)
            assert sorted(out) == sorted(outputs)
            check_norm(out, xv, rrv, None if ww is None else ww.astype(np.float64), 1e-5, dtype)


@pytest.mark.parametrize("K", [300, 2048, 16000, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_in_place(K, dtype):
    """sum into the residual's array and y into x's: the same bytes as into arrays of their own."""
    (x, _), (r, _), w = norm_inputs(3, K, dtype, K)
    want = norm_dev(x, r, w, 1e-6, dtype)
    got = norm_dev(x, r, w, 1e-6, dtype, in_place=True)
    for k in "sy":
        np.testing.assert_array_equal(got[k], want[k])
    for a, b in zip(got["c"], want["c"]):
        np.testing.assert_array_equal(a, b)


def test_norm_extremes():
    """Rows whose squares leave f32's range on either side, zero rows, infinities and NaN."""
    rng = np.random.default_rng(5)
    base = rng.standard_normal((1, 640))
    x = np.concatenate([base * 1e-30, base * 3e37, base * 1e-40, base * 0, base, base, base])
    x[4, 5], x[5, 300], x[6, 600] = np.inf, np.nan, -np.inf
    raw, val = ref.typed(x, ref.F32)
    out = norm_dev(raw, None, None, 0.0, ref.F32)
    check_norm({k: v[:3] if k != "c" else [a[:3] for a in v] for k, v in out.items()}, val[:3], None,
               None, 0.0, ref.F32)
    # Nothing over nothing: NaN, as 0 / 0.
    assert np.isnan(out["y"][3]).all() and (out["c"][1][3, :5] == 255).all()
    for row, col in ((4, 5), (6, 600)):
        y, scales = out["y"][row], out["c"][1][row]
        assert np.isnan(y[col]) and (np.delete(y, col) == 0).all()
        assert [int(s) for s in scales[:5]] == [255 if g == col // 128 else 10 for g in range(5)]
    assert np.isnan(out["y"][5]).all()
    # With eps, a zero row stays zero.
    out = norm_dev(raw[3:4], None, None, 1e-6, ref.F32)
    assert (out["y"] == 0).all() and (out["c"][0] & 127 == 0).all()


# ---------------------------------------------------------------- linear

def linear_dev(a, w, K, dtype, ldc=None, shift=0):
    """a, w: (codes, scales).  C with rows ldc apart; bytes between rows must stay."""
    from devmem import DevBuf
    lib = _lib.load()
    M, N = len(a[0]), len(w[0])
    ldc = ldc or N
    c = DevBuf.of(np.full(shift + M * ldc, 77, np_type(dtype)))
    d = [DevBuf.of(x) for x in (*a, *w)]
    nbytes = lib.anima_hip_linear_fp8_scratch_bytes(M, N, K, dtype)
    scratch = DevBuf(max(nbytes, 16))
    at = c.addr + shift * np_type(dtype)().itemsize

    def call(addr, size):
        return lib.anima_hip_linear_fp8_dev(*(x.addr for x in d), at, ldc, M, N, K, dtype, addr,
                                            size, None)
    if nbytes:
        for addr, size in ((scratch.addr, nbytes - 1), (None, nbytes), (scratch.addr + 8, nbytes)):
            assert not call(addr, size) and "scratch" in _lib.last_error()
    _lib.check(call(scratch.addr, nbytes), "linear")
    got = c.get((shift + M * ldc,), np_type(dtype))
    assert (got[:shift] == 77).all()
    got = got[shift:].reshape(M, ldc)
    assert (got[:, N:] == 77).all()
    return ref.untyped(got[:, :N], dtype)


def check_linear(got, a, w, K, dtype):
    av, wv = ref.unpack(*a, K), ref.unpack(*w, K)
    want, mag = av @ wv.T, np.abs(av) @ np.abs(wv).T
    tol = (K + 16) * 2.0 ** -24 * mag + ref.HALF[dtype] * np.abs(want)
    if dtype == ref.BF16:
        pad = [np.pad(np.abs(v), ((0, 0), (0, -K % 8))) for v in (av, wv)]
        for k in range(0, K, 8):
            p = pad[0][:, None, k:k + 8] * pad[1][None, :, k:k + 8]
            tol += 7 * 2.0 ** -13 * p.max(-1)
    err = np.abs(got - want)
    assert (err <= tol).all(), (np.unravel_index(np.argmax(err - tol), err.shape), err.max())


def linear_inputs(M, N, K, seed):
    rng = np.random.default_rng(seed)
    a, w = (np.float32(rng.standard_normal((n, K)) * np.exp(0.5 * rng.standard_normal((n, 1))) * s)
            for n, s in ((M, 1.0), (N, 0.02)))
    return ref.pack(a.astype(np.float64)), ref.pack(w.astype(np.float64))


LINEAR = [(1, 1, 1, None, 0), (1, 16, 128, None, 0), (3, 17, 129, 20, 0), (16, 48, 1000, None, 0),
          (17, 33, 512, 35, 1), (33, 100, 640, None, 0), (64, 256, 2048, None, 0),
          (130, 70, 384, 72, 2), (1, 2048, 2048, None, 0), (2, 300, 4000, None, 0),
          (40, 64, 9000, None, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,ldc,shift", LINEAR)
def test_linear(M, N, K, ldc, shift, dtype):
    a, w = linear_inputs(M, N, K, M + N + K)
    check_linear(linear_dev(a, w, K, dtype, ldc, shift), a, w, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 20, 200])
def test_linear_without_terms_is_zero(M, dtype):
    """K = 0: zeros, and no operand is read."""
    from devmem import DevBuf
    c = DevBuf.of(np.full((M, 30), 5, np_type(dtype)))
    _lib.check(_lib.load().anima_hip_linear_fp8_dev(None, None, None, None, c.addr, 30, M, 30, 0,
                                                    dtype, None, 0, None), "linear")
    assert (c.get((M, 30), np_type(dtype)) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(5, 40, 700), (70, 130, 1300), (300, 260, 640)])
def test_linear_nan_groups(M, N, K, dtype):
    """A NaN group of a row of either operand makes that row or column NaN, and no other."""
    a, w = linear_inputs(M, N, K, 9)
    clean = linear_dev(a, w, K, dtype)
    a[1][M // 2, 3], w[1][N // 3, 1] = 255, 255
    a[0][M // 2, 384:512] = 0
    w[0][N // 3, 128:256] = 0
    got = linear_dev(a, w, K, dtype)
    bad = np.zeros((M, N), bool)
    bad[M // 2], bad[:, N // 3] = True, True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_single_products(M):
    """One non-zero weight per row: no addition to round, so C is the product itself, for every
    scale byte that the packer writes."""
    rng = np.random.default_rng(M)
    K, N = 1024, 240
    a, _ = linear_inputs(M, 1, K, 4)
    w = np.zeros((N, K), np.uint8), np.full((N, 8), 10, np.uint8)
    at = rng.integers(0, K, N)
    w[0][np.arange(N), at] = rng.integers(1, 127, N) | rng.integers(0, 2, N) << 7
    w[1][np.arange(N), at // 128] = 10 + np.arange(N) % 237
    want = ref.unpack(*a, K) @ ref.unpack(*w, K).T
    with np.errstate(over="ignore"):
        f32 = np.float32(want).astype(np.float64)
        fits = (np.abs(want) >= 2.0 ** -120) & np.isfinite(f32) | (want == 0)
        np.testing.assert_array_equal(linear_dev(a, w, K, ref.F32)[fits], f32[fits])
        np.testing.assert_array_equal(linear_dev(a, w, K, ref.BF16)[fits],
                                      ref.values_of(ref.bits_of(f32))[fits])


def test_calls_without_work():
    lib = _lib.load()
    assert lib.anima_hip_fp8_pack_dev(None, 0, ref.F32, None, None, 0, 5, None)
    assert lib.anima_hip_fp8_unpack_dev(None, None, None, 0, ref.F32, 5, 0, None)
    assert lib.anima_hip_add_rmsnorm_fp8_dev(None, 0, None, 0, None, ct.c_float(0), ref.F32, 4096, 0,
                                             None, 0, None, None, 0, 5, None)
    assert lib.anima_hip_linear_fp8_dev(None, None, None, None, None, 0, 0, 5, 5, ref.F32, None, 0,
                                        None)
