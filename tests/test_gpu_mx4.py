"""The 4-bit rows on the GPU: packing and the linear layer against 64-bit numpy.

Packing is a function of the values and is compared byte for byte.  The linear layer's weights and
activations enter exactly, so only its f32 sums and the last rounding are off:

  |C - ref| <= n 2^-24 sum_k |a_k w_k| + HALF |ref|

with n the additions of one result (K per term, three terms in f32, and the waves' or the splits'
partial sums), HALF the last rounding's half step.  Products with one non-zero weight per row have
no addition to round and are compared bit for bit.
"""
import numpy as np
import pytest

import mx4_ref as ref
from anima_hip import _lib, rt

pytestmark = pytest.mark.gpu

TYPES = [ref.F32, ref.BF16]


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


def _ld(raw, ld, fill):
    """Rows of a 2-D array ld elements apart in one buffer."""
    buf = np.full((raw.shape[0], ld), fill, raw.dtype)
    buf[:, :raw.shape[1]] = raw
    return buf


def pack_dev(raw, dtype, ld=None, shift=0):
    """Codes and scales through anima_hip_mx4_pack_dev, with rows ld apart and the base `shift`
    elements past an aligned address; bytes past the outputs must stay."""
    from devmem import DevBuf
    rows, K = raw.shape
    ld, G = ld or K, -(-K // 32)
    flat = np.concatenate([np.zeros(shift, raw.dtype), _ld(raw, ld, 0x55).reshape(-1)])
    x = DevBuf.of(flat)
    codes, scales = (DevBuf.of(np.full(rows * G * w + 64, 0xA5, np.uint8)) for w in (16, 1))
    _lib.check(_lib.load().anima_hip_mx4_pack_dev(x.addr + shift * raw.itemsize, ld, dtype,
                                                  codes.addr, scales.addr, rows, K, None), "pack")
    c = codes.get((rows * G * 16 + 64,), np.uint8)
    s = scales.get((rows * G + 64,), np.uint8)
    assert (c[rows * G * 16:] == 0xA5).all() and (s[rows * G:] == 0xA5).all()
    return c[:rows * G * 16].reshape(rows, -1), s[:rows * G].reshape(rows, -1)


def unpack_dev(codes, scales, K, dtype, ld=None):
    from devmem import DevBuf
    rows, ld = codes.shape[0], ld or K
    out = DevBuf.of(np.full((rows, ld), 7, np.float32 if dtype == ref.F32 else np.uint16))
    c, s = DevBuf.of(codes), DevBuf.of(scales)
    _lib.check(_lib.load().anima_hip_mx4_unpack_dev(c.addr, s.addr, out.addr, ld, dtype, rows, K,
                                                    None), "unpack")
    got = out.get((rows, ld), np.float32 if dtype == ref.F32 else np.uint16)
    assert (got[:, K:] == 7).all()
    return ref.untyped(got[:, :K], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,ld,shift", [
    (1, 1, None, 0), (3, 31, None, 0), (5, 32, None, 0), (7, 33, 40, 0), (129, 68, None, 0),
    (33, 96, 104, 3), (64, 1000, 1001, 1), (257, 2048, None, 0), (1, 8192, None, 0)])
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
    """Ties, values next to them, zeros of both signs, saturation, the scales' ends, infinities
    and NaN: each group byte for byte."""
    edges = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], np.float32)
    around = np.concatenate([edges, np.nextafter(edges, 0), np.nextafter(edges, 9)])[:26]
    rows = []
    for e in (-148, -130, -126, -124, -20, 0, 60, 125):
        for top in (4.0, 6.0, 6.999999, 7.0, 7.0000005, 7.99):
            g = np.concatenate([around, -edges[:4], [top], [-0.0]]).astype(np.float32)
            g = np.where(np.abs(g) > top, top, g)
            with np.errstate(over="ignore"):
                rows.append(np.clip(np.float64(g) * 2.0 ** e, -3.4e38, 3.4e38))
    rows += [np.zeros(32), -np.zeros(32), np.full(32, 3.4028235e38), np.full(32, 1e-45)]
    for bad in (np.inf, -np.inf, np.nan):
        g = np.linspace(-3, 3, 32)
        g[11] = bad
        rows.append(g)
    raw, val = ref.typed(np.stack(rows), ref.F32)
    codes, scales = pack_dev(raw, ref.F32)
    want = ref.pack(val)
    np.testing.assert_array_equal(scales, want[1])
    np.testing.assert_array_equal(codes, want[0])
    assert (scales[-3:] == 255).all() and (codes[-3:] == 0).all()
    assert np.isnan(unpack_dev(codes[-3:], scales[-3:], 32, ref.BF16)).all()


def linear(raw, codes, scales, K, N, dtype, lda=None, ldc=None, shift=0):
    from devmem import DevBuf
    lib = _lib.load()
    M = raw.shape[0]
    lda, ldc = lda or max(K, 1), ldc or N
    flat = np.concatenate([np.zeros(shift, raw.dtype), _ld(raw, lda, 0x7F).reshape(-1)])
    a, c = DevBuf.of(flat), DevBuf.of(np.full((M, ldc), 77, raw.dtype))
    w, s = DevBuf.of(codes), DevBuf.of(scales)
    nbytes = lib.anima_hip_linear_mx4_scratch_bytes(M, N, K, dtype)
    scratch = DevBuf(max(nbytes, 16))
    if nbytes:
        ok = lib.anima_hip_linear_mx4_dev(a.addr, lda, w.addr, s.addr, c.addr, ldc, M, N, K, dtype,
                                          scratch.addr, nbytes - 1, None)
        assert not ok and "scratch" in _lib.last_error()
    _lib.check(lib.anima_hip_linear_mx4_dev(a.addr + shift * raw.itemsize, lda, w.addr, s.addr,
                                            c.addr, ldc, M, N, K, dtype, scratch.addr, nbytes,
                                            None), "linear_mx4")
    got = c.get((M, ldc), raw.dtype)
    assert (got[:, N:] == 77).all()
    return ref.untyped(got[:, :N], dtype)


def check_linear(M, N, K, dtype, seed, **kw):
    rng = np.random.default_rng(seed)
    raw, a = ref.typed(rng.standard_normal((M, K)), dtype)
    codes, scales = ref.pack(np.float32(rng.standard_normal((N, K)) * 0.02).astype(float))
    w = ref.unpack(codes, scales, K)
    got = linear(raw, codes, scales, K, N, dtype, **kw)
    want, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    n = K * (3 if dtype == ref.F32 else 1) + 32
    err = np.abs(got - want)
    bound = n * 2.0 ** -24 * mag + ref.HALF[dtype] * np.abs(want)
    assert (err <= bound).all(), (err / np.maximum(bound, 1e-300)).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 32, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 33), (130, 68), (257, 1024), (64, 2500)])
def test_linear(M, N, K, dtype):
    print(f"linear_mx4 M={M} N={N} K={K} dtype={dtype}", flush=True)
    check_linear(M, N, K, dtype, M * 31 + N + K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 2048, 8192), (16, 300, 8192), (24, 2048, 8192),
                                   (333, 2048, 1024), (1500, 2100, 256), (2049, 8000, 96)])
def test_linear_layer_sizes(M, N, K, dtype):
    print(f"linear_mx4 M={M} N={N} K={K} dtype={dtype}", flush=True)
    check_linear(M, N, K, dtype, M + N + K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [3, 40, 200])
def test_linear_strides(M, dtype):
    """Wider rows, rows that are not 16-byte aligned, a base that is not."""
    check_linear(M, 70, 160, dtype, 1, lda=168, ldc=75)
    check_linear(M, 70, 160, dtype, 2, lda=163, ldc=70)
    check_linear(M, 70, 160, dtype, 3, lda=168, shift=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 16, 20, 60, 150])
def test_linear_is_exact_without_additions(M, dtype):
    """W with one power of two per row: C is A's column times it, every bit of f32 A included."""
    K, N = 416, 200
    rng = np.random.default_rng(M)
    x = rng.standard_normal((M, K)) * np.exp2(rng.integers(-60, 60, (M, K)).astype(float))
    raw, a = ref.typed(x, dtype)
    cols = rng.integers(0, K, N)
    w = np.zeros((N, K))
    w[np.arange(N), cols] = np.exp2(rng.integers(-9, 9, N).astype(float)) * rng.choice([-1, 1], N)
    codes, scales = ref.pack(w)
    np.testing.assert_array_equal(ref.unpack(codes, scales, K), w)
    got = linear(raw, codes, scales, K, N, dtype)
    np.testing.assert_array_equal(got, (a @ w.T))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [2, 40, 150])
def test_linear_infinities_and_nan(M, dtype):
    """An infinite activation gives infinities where its weight is not zero and no NaN beside
    them; a NaN group of the weights makes its output column NaN and no other."""
    K, N = 64, 40
    a = np.ones((M, K))
    a[0, 5] = np.inf
    a[1, 6] = np.nan
    raw, val = ref.typed(a, dtype)
    codes, scales = ref.pack(np.full((N, K), 1.5))
    scales[7, 1] = 255
    got = linear(raw, codes, scales, K, N, dtype)
    with np.errstate(invalid="ignore"):
        want = val @ ref.unpack(codes, scales, K).T
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_without_work(dtype):
    from devmem import DevBuf
    lib = _lib.load()
    c = DevBuf.of(np.full(64, 77, np.uint32))
    for M, N in ((0, 8), (8, 0)):
        assert lib.anima_hip_linear_mx4_dev(None, 8, None, None, c.addr, 8, M, N, 8, dtype, None,
                                            0, None)
    assert (c.get((64,), np.uint32) == 77).all()
    # K = 0: an empty sum.
    assert lib.anima_hip_linear_mx4_dev(None, 0, None, None, c.addr, 4, 2, 4, 0, dtype, None, 0,
                                        None)
    words = 8 if dtype == ref.F32 else 4
    got = c.get((64,), np.uint32)
    assert (got[:words] == 0).all() and (got[words:] == 77).all()


def test_linear_repeats():
    rng = np.random.default_rng(3)
    raw, _ = ref.typed(rng.standard_normal((24, 4096)), ref.F32)
    codes, scales = ref.pack(rng.standard_normal((512, 4096)))
    first = linear(raw, codes, scales, 4096, 512, ref.F32)
    for _ in range(3):
        np.testing.assert_array_equal(linear(raw, codes, scales, 4096, 512, ref.F32), first)
