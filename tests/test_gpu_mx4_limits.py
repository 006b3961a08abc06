"""The 4-bit operators at their ends: codes past 4 GiB, default strides, the scale bytes packing
never writes, empty calls."""
import ctypes as ct

import numpy as np
import pytest

import mx4_ref as ref
import test_gpu_kv4 as kv4
import test_gpu_mx4 as mx4
from anima_hip import _lib, rt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_weights_past_4_gib(M):
    """1.1 M weight rows of 8192 (4.5 GB of codes): the first and last rows' outputs.  The rows
    between hold whatever the memory does."""
    from devmem import DevBuf
    lib, N, K, edge = _lib.load(), 1100001 if M < 300 else 600001, 8192, 40
    if M == 300:
        K = 16384
    rng = np.random.default_rng(M)
    raw, a = ref.typed(rng.standard_normal((M, K)), ref.BF16)
    codes, scales = ref.pack(rng.standard_normal((2 * edge, K)) * 0.02)
    w, s = DevBuf(N * K // 2), DevBuf(N * K // 32)
    assert w.nbytes > 1 << 32
    for at, rows in ((0, slice(0, edge)), (N - edge, slice(edge, 2 * edge))):
        w.put(codes[rows], at * K // 2)
        s.put(scales[rows], at * K // 32)
    x, c = DevBuf.of(raw), DevBuf(M * N * 2)
    n = lib.anima_hip_linear_mx4_scratch_bytes(M, N, K, ref.BF16)
    scratch = DevBuf(max(n, 16))
    _lib.check(lib.anima_hip_linear_mx4_dev(x.addr, K, w.addr, s.addr, c.addr, N, M, N, K, ref.BF16,
                                            scratch.addr, n, None), "linear")
    got = c.get((M, N), np.uint16)
    got = ref.untyped(np.concatenate([got[:, :edge], got[:, -edge:]], 1), ref.BF16)
    wv = ref.unpack(codes, scales, K)
    want, mag = a @ wv.T, np.abs(a) @ np.abs(wv).T
    assert (np.abs(got - want) <= (K + 32) * kv4.U * mag + ref.HALF[ref.BF16] * np.abs(want)).all()


@pytest.mark.parametrize("S_q", [1, 60])
def test_cache_past_4_gib(S_q):
    """1100 sequences x 2 heads x 32768 tokens (4.6 GB of K codes): the last ones, and a first."""
    Bk, H_kv, S_max, D, n = 1100, 2, 32768, 128, 70
    cache = kv4.Cache.__new__(kv4.Cache)
    from devmem import DevBuf
    cache.shape = (Bk, H_kv, S_max, D)
    rows = Bk * H_kv * S_max
    cache.bufs = [DevBuf(rows * D // 2), DevBuf(rows * D // 32), DevBuf(rows * D // 2),
                  DevBuf(rows * D // 32)]
    assert cache.bufs[0].nbytes > 1 << 32
    rng = np.random.default_rng(S_q)
    live = [0, 1098, 1099]
    lens = [n if b in live else 0 for b in range(Bk)]
    k, v = (np.zeros((Bk, n, H_kv, D), np.float32) for _ in range(2))
    for x in (k, v):
        x[live] = rng.standard_normal((len(live), n, H_kv, D))
    kv4.append(cache, k, v, ref.F32, [0] * Bk, lens)
    q = np.zeros((Bk, S_q, 4, D), np.float32)
    q[live] = rng.standard_normal((len(live), S_q, 4, D))
    got = kv4.attend(cache, q, ref.F32, lens)
    kc, vc = (ref.unpack(*ref.pack(x[live].reshape(-1, D).astype(float)), D).reshape(
        len(live), n, H_kv, D).transpose(0, 2, 1, 3) for x in (k, v))
    want, mag = ref.attention_rows(q[live].astype(float), kc, vc, [n] * 3, None, True, D ** -0.5)
    d = (3 * D + 6) * kv4.U * D ** -0.5 * np.abs(q[live]).sum(-1, keepdims=True) * np.abs(kc).max()
    assert (np.abs(got[live] - want) <= (4 * d + (n + 64) * kv4.U) * mag
            + kv4.U * np.abs(want)).all()
    assert not got[[b for b in range(Bk) if b not in live]].any()


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
@pytest.mark.parametrize("S_q", [3, 300])
def test_default_strides(S_q, dtype):
    """NULL strides: [B, H, S, D]."""
    from devmem import DevBuf
    lib = _lib.load()
    B, H, D, S = 2, 32, 64, 100
    rng = np.random.default_rng(2)
    (kr, _), (vr, _) = (ref.typed(rng.standard_normal((B, H, S, D)), dtype) for _ in range(2))
    cache = kv4.Cache(B, H, S, D)
    bufs = [DevBuf.of(kr), DevBuf.of(vr), kv4.ints([0, 0])]
    _lib.check(lib.anima_hip_kv4_append_dev(bufs[0].addr, bufs[1].addr, dtype, None, None,
                                            *cache.addrs, bufs[2].addr, None, B, S, H, D, S, None),
               "append")
    raw, q = ref.typed(rng.standard_normal((B, H, S_q, D)), dtype)
    qd, out, lens = DevBuf.of(raw), DevBuf(raw.nbytes), kv4.ints([S, S - 7])
    n = lib.anima_hip_kv4_attention_scratch_bytes(B, S_q, H, H, D, S, dtype)
    scratch = DevBuf(max(n, 16))
    _lib.check(lib.anima_hip_kv4_attention_dev(
        qd.addr, dtype, None, *cache.addrs, lens.addr, None, out.addr, None, B, B, S_q, H, H, D, S,
        ct.c_float(0.125), True, scratch.addr, n, None), "attention")
    got = ref.untyped(out.get(raw.shape, raw.dtype), dtype).transpose(0, 2, 1, 3)
    k, v = cache.values()
    q = q.transpose(0, 2, 1, 3)
    want, mag = ref.attention_rows(q, k, v, [S, S - 7], None, True, 0.125)
    d = (3 * D + 6) * kv4.U * 0.125 * np.abs(q).sum(-1, keepdims=True) * np.abs(k).max()
    r = 2.0 ** -8 if dtype == ref.BF16 else 0.0
    assert (np.abs(got - want) <= (4 * d + (S + 64) * kv4.U + r) * mag
            + ref.HALF[dtype] * np.abs(want)).all()


@pytest.mark.parametrize("M", [2, 40, 200])
def test_linear_takes_any_scale_byte(M):
    """Weights from elsewhere: scale bytes 0 and 1 (subnormal bf16 values among them), 253 and 254,
    each against one activation per column.  Weights of 2^128 and more are infinite; times the
    zeros behind the first of an f32 activation's three terms they are NaN, so such a result is
    only known not to be finite."""
    K, N = 128, 512
    codes = np.zeros((N, K // 2), np.uint8)
    scales = np.full((N, K // 32), 127, np.uint8)
    n = np.arange(N)
    code = (n % 16).astype(np.uint8)
    byte = np.array([0, 1, 2, 3, 120, 252, 253, 254], np.uint8)[n // 16 % 8]
    col = n * 7 % K
    codes[n, col // 2] = np.where(col % 2, code << 4, code)
    scales[n, col // 32] = byte
    a = np.exp2(np.random.default_rng(1).integers(-2, 3, (M, K)).astype(float)) * 3
    a *= 2.0 ** 20
    raw, val = ref.typed(a, ref.F32)
    got = mx4.linear(raw, codes, scales, K, N, ref.F32)
    wv = ref.unpack(codes, scales, K)
    one = wv[n, col]
    with np.errstate(over="ignore"):
        want = np.float64(np.float32(val[:, col] * one))
    past = np.abs(one) >= 2.0 ** 128
    assert past.any() and not np.isfinite(got[:, past]).any()
    np.testing.assert_array_equal(got[:, ~past], want[:, ~past])


def test_empty_calls():
    lib = _lib.load()
    assert lib.anima_hip_kv4_append_dev(None, None, 0, None, None, None, None, None, None, None, None,
                                        0, 5, 2, 128, 16, None)
    assert lib.anima_hip_kv4_append_dev(None, None, 0, None, None, None, None, None, None, None, None,
                                        2, 5, 2, 128, 0, None)
    assert lib.anima_hip_kv4_attention_dev(None, 0, None, None, None, None, None, None, None, None,
                                           None, 3, 3, 0, 4, 2, 128, 16, ct.c_float(1.0), True, None,
                                           0, None)
    assert lib.anima_hip_mx4_pack_dev(None, 0, 0, None, None, 0, 64, None)
    assert lib.anima_hip_mx4_unpack_dev(None, None, None, 0, 0, 5, 0, None)
    # A cache without room: every query sees no key.
    from devmem import DevBuf
    q, out, lens = DevBuf.of(np.ones((1, 2, 2, 64), np.float32)), DevBuf.of(
        np.full((1, 2, 2, 64), 7, np.float32)), kv4.ints([9])
    assert lib.anima_hip_kv4_attention_dev(q.addr, 0, None, None, None, None, None, lens.addr, None,
                                           out.addr, None, 1, 1, 2, 2, 2, 64, 0, ct.c_float(1.0),
                                           True, None, 0, None)
    assert (out.get((1, 2, 2, 64)) == 0).all()


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
@pytest.mark.parametrize("S_q", [2, 300])
@pytest.mark.parametrize("power", [20, 31, 45, 90])
def test_far_scores(power, S_q, dtype):
    """Scores of up to 6 * 2^power, some steps of 2^power / 2 apart, exact in f32: each row is the
    mean of the values of the keys of its largest score, which one in seven keys has."""
    B, H, D, S, scale = 1, 2, 128, 333, 0.1
    rng = np.random.default_rng(power)
    k, v = np.zeros((B, S, H, D)), rng.standard_normal((B, S, H, D))
    steps = np.array([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    k[..., 0] = steps[np.arange(S) % 7][None, :, None]
    q = np.zeros((B, S_q, H, D))
    q[..., 0] = 2.0 ** power * np.where(np.arange(S_q) % 2, -1, 1)[None, :, None]
    cache = kv4.Cache(B, H, S, D)
    kv4.append(cache, ref.typed(k, dtype)[0], ref.typed(v, dtype)[0], dtype, [0])
    got = kv4.attend(cache, ref.typed(q, dtype)[0], dtype, [S], causal=False, scale=scale)
    _, vc = cache.values()
    for s in range(2):
        top = np.arange(S) % 7 == (0 if s else 6)
        val = vc[:, :, top]                                   # [B, H, keys, D]
        want, mag = val.mean(2)[:, None], np.abs(val).mean(2)[:, None]
        rows = got[:, s::2]
        # Probabilities of 2^r (the top) and 0, one rounding each; f32 sums; out once.
        bound = (2 * ref.HALF[dtype] + (S + 64) * kv4.U) * mag + ref.HALF[dtype] * np.abs(want)
        assert (np.abs(rows - want) <= bound).all(), (power, s)


def test_too_large_for_one_launch():
    """Refused on the host, before any launch."""
    from devmem import DevBuf
    lib = _lib.load()
    mem = DevBuf(4096)
    at = mem.addr
    for call in (
            lambda: lib.anima_hip_mx4_pack_dev(at, 32, 0, at, at, 1 << 29, 32, None),
            lambda: lib.anima_hip_mx4_unpack_dev(at, at, at, 32, 0, 1 << 29, 32, None),
            lambda: lib.anima_hip_kv4_append_dev(at, at, 0, None, None, at, at, at, at, at, None,
                                                 1 << 20, 1 << 8, 4, 64, 1 << 20, None),
            lambda: lib.anima_hip_linear_mx4_dev(at, 4096, at, at, at, 1 << 30, 16, 1 << 30, 4096, 2,
                                                 at, 4096, None),
            lambda: lib.anima_hip_kv4_attention_dev(at, 2, None, at, at, at, at, at, None, at, None,
                                                    1 << 23, 1, 1, 32, 32, 64, 512, ct.c_float(1.0),
                                                    True, at, 4096, None)):
        assert not call() and ("too many" in _lib.last_error() or "launch" in _lib.last_error())


@pytest.mark.parametrize("K", [128, 100])
@pytest.mark.parametrize("M", [3, 40, 200])
def test_linear_nan_patterns(M, K):
    """f32 NaN of every kind (quiet, signalling, payload in the low half alone) make their row NaN;
    infinities of both signs give infinities of the weight's sign."""
    N = 64
    rng = np.random.default_rng(M)
    a = rng.standard_normal((M, K)).astype(np.float32)
    bits = a.view(np.uint32)
    bits[0, 5], bits[M // 2, K - 1], bits[M - 1, 40] = 0x7F800001, 0xFF800002, 0x7FC00000
    bits[1, 7], bits[M - 2 if M > 3 else 1, 8] = 0x7F800000, 0xFF800000
    w = rng.choice([-1.0, 1.0], (N, K)) * rng.choice([0.5, 1.0, 3.0, 6.0], (N, K))
    codes, scales = ref.pack(w)
    wv = ref.unpack(codes, scales, K)
    assert (wv != 0).all()
    got = mx4.linear(a, codes, scales, K, N, ref.F32)
    with np.errstate(invalid="ignore"):
        want = np.stack([[np.sum(a[m].astype(float) * wv[n]) for n in range(N)] for m in range(M)])
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    far = np.isinf(want)
    np.testing.assert_array_equal(got[far], want[far])
    ok = np.isfinite(want)
    mag = np.abs(np.where(np.isfinite(a), a, 0).astype(float)) @ np.abs(wv).T
    bound = (K + 32) * kv4.U * mag + kv4.U * np.abs(want)
    assert (np.abs(got[ok] - want[ok]) <= bound[ok]).all()


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
@pytest.mark.parametrize("M,N,K", [(1, 32753, 2048), (3, 70001, 500), (16, 33333, 96), (5, 65537, 1000),
                                   (1, 40000, 1), (16, 32768, 768), (4, 50007, 2560)])
def test_linear_many_weight_rows(M, N, K, dtype):
    """N of 2048 strips of 16 and more: 97 distinct weight rows over and over (97 shares no factor
    with a strip), one of them with a NaN group, which is its column's alone."""
    rng = np.random.default_rng(N)
    raw, a = ref.typed(rng.standard_normal((M, K)), dtype)
    codes, scales = ref.pack(rng.standard_normal((97, K)) * 0.05)
    scales[13, -1] = 255
    rows = np.arange(N) % 97
    for shift, ld in ((0, K), (1, K + 3)):
        got = mx4.linear(raw, codes[rows], scales[rows], K, N, dtype, lda=ld, shift=shift)
        wv = ref.unpack(codes, scales, K)
        want, mag = a @ wv.T, np.abs(a) @ np.abs(wv).T
        assert np.isnan(got[:, rows == 13]).all()
        ok = rows != 13
        err = np.abs(got - want[:, rows])[:, ok]
        bound = (K + 32) * kv4.U * mag + ref.HALF[dtype] * np.abs(want)
        assert (err <= bound[:, rows][:, ok]).all()


@pytest.mark.parametrize("dtype", [ref.F32, ref.BF16])
@pytest.mark.parametrize("M,N,K", [(700, 2047, 384), (333, 2001, 640), (130, 1001, 128),
                                   (24, 300, 1408), (60, 257, 11008), (90, 515, 896), (260, 600, 1152)])
def test_linear_odd_and_even_chunks(M, N, K, dtype):
    """K of odd and even numbers of 128 elements, whole and in splits of either."""
    mx4.check_linear(M, N, K, dtype, M + K)
