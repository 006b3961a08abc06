"""The 4-bit K/V cache on the GPU: append, and attention over it, against 64-bit numpy.

K, V and f32 queries enter the products exactly.  With u = 2^-24: a score is off by at most
d = (3 D + 4) u scale sum |q k| + 2 u |score|, its probability by a factor of exp(2 d) with the
maximum's, plus 4 u for the exponential, and an output, a mean of n values weighted by them, by

  (4 d + (n + 64) u) sum_j p_j |v_j| + r sum_j p_j |v_j| + HALF |out|

where r is the rounding of the probabilities: 2^-8 with bf16 queries (one bf16 term), none with f32
ones (three).  A probability below 2^-126 of the largest is less than f32's smallest normal number
and may be zero (exp(-200) = 1e-87 is, whatever its relative bound says): n of them make n 2^-126
max |v|, added below.  A row that sees one key is V's row bit for bit.
"""
import ctypes as ct
import math

import numpy as np
import pytest

import mx4_ref as ref
from anima_hip import _lib, rt

pytestmark = pytest.mark.gpu

TYPES = [ref.F32, ref.BF16]
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


class Cache:
    """Device arrays of a cache [Bk, H_kv, S_max, D]."""

    def __init__(self, Bk, H_kv, S_max, D, fill=0xFF):
        from devmem import DevBuf
        self.shape = (Bk, H_kv, S_max, D)
        rows = Bk * H_kv * S_max
        self.sizes = [rows * D // 2, rows * D // 32] * 2
        self.bufs = [DevBuf.of(np.full(max(n, 16), fill, np.uint8)) for n in self.sizes]

    @classmethod
    def of(cls, k, v):
        c = cls(*k.shape)
        for i, x in enumerate((k, v)):
            codes, scales = ref.pack(x.reshape(-1, k.shape[-1]))
            c.bufs[2 * i].put(codes, 0)
            c.bufs[2 * i + 1].put(scales, 0)
        return c

    @property
    def addrs(self):
        return [b.addr for b in self.bufs]

    def raw(self):
        """(codes, scales) of K and of V as [Bk, H_kv, S_max, ...]."""
        Bk, H, S, D = self.shape
        out = []
        for i in (0, 2):
            codes = self.bufs[i].get((self.sizes[i],), np.uint8).reshape(Bk, H, S, D // 2)
            scales = self.bufs[i + 1].get((self.sizes[i + 1],), np.uint8)
            out.append((codes, scales.reshape(Bk, H, S, D // 32)))
        return out

    def values(self):
        return [ref.unpack(c, s, self.shape[-1]) for c, s in self.raw()]


def ints(values):
    from devmem import DevBuf
    return DevBuf.of(np.array(values, np.int32))


def append(cache, raw_k, raw_v, dtype, starts, counts=None, strides=None, shift=0, stream=None):
    """raw: [B, S_new, H_kv, D] arrays (strides: of both, as {batch, head, token})."""
    from devmem import DevBuf
    _, H, S_max, D = cache.shape
    B, S = raw_k.shape[:2]
    st = strides or (S * H * D, D, H * D)
    pad = np.zeros(shift, raw_k.dtype)
    k, v = (DevBuf.of(np.concatenate([pad, x.reshape(-1)])) for x in (raw_k, raw_v))
    at, n = ints(starts), None if counts is None else ints(counts)
    off = shift * raw_k.itemsize
    _lib.check(_lib.load().anima_hip_kv4_append_dev(
        k.addr + off, v.addr + off, dtype, _lib.strides(st), _lib.strides(st), *cache.addrs,
        at.addr, n.addr if n else None, B, S, H, D, S_max, stream), "append")


def attend(cache, raw_q, dtype, lens, counts=None, causal=True, scale=None, pad=0, fill=77):
    """raw_q [B, S_q, H, D]; pad: elements between token rows of q and out."""
    from devmem import DevBuf
    lib = _lib.load()
    Bk, H_kv, S_max, D = cache.shape
    B, S, H, _ = raw_q.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    ld = H * D + pad
    buf = np.full((B, S, ld), fill, raw_q.dtype)
    buf[:, :, :H * D] = raw_q.reshape(B, S, H * D)
    q, out = DevBuf.of(buf), DevBuf.of(np.full((B, S, ld), fill, raw_q.dtype))
    n = lib.anima_hip_kv4_attention_scratch_bytes(B, S, H, H_kv, D, S_max, dtype)
    scratch = DevBuf(max(n, 16))
    ln, cn = ints(lens), None if counts is None else ints(counts)
    st = _lib.strides((S * ld, D, ld))

    def call(nbytes):
        return lib.anima_hip_kv4_attention_dev(
            q.addr, dtype, st, *cache.addrs, ln.addr, cn.addr if cn else None, out.addr, st, B, Bk,
            S, H, H_kv, D, S_max, ct.c_float(scale), causal, scratch.addr, nbytes, None)

    if n:
        assert not call(n - 1) and "scratch" in _lib.last_error()
    _lib.check(call(n), "kv4_attention")
    got = out.get((B, S, ld), raw_q.dtype)
    assert (got[:, :, H * D:] == fill).all()
    for b in range(B):
        m = S if counts is None else min(max(counts[b], 0), S)
        assert (got[b, m:] == fill).all(), "rows past counts were written"
        got[b, m:] = 0
    return ref.untyped(got[:, :, :H * D].reshape(raw_q.shape), dtype)


def check(cache, q_raw, q, dtype, lens, counts=None, causal=True, scale=None, **kw):
    D = q.shape[-1]
    sc = 1 / math.sqrt(D) if scale is None else scale
    k, v = cache.values()
    got = attend(cache, q_raw, dtype, lens, counts, causal, scale, **kw)
    want, mag = ref.attention(q, k, v, lens, counts, causal, sc)
    # The score's own bound, per row: sum |q k| <= |q|_1 max |k|.
    l1 = np.abs(q).sum(-1, keepdims=True) * (np.nanmax(np.abs(k)) if k.size else 0.0)
    d = (3 * D + 6) * U * abs(sc) * l1
    n = max(list(lens) + [0])
    r = 2.0 ** -8 if dtype == ref.BF16 else 0.0
    bound = (4 * d + (n + 64) * U + r) * mag + ref.HALF[dtype] * np.abs(want)
    bound = bound + n * 2.0 ** -126 * (np.nanmax(np.abs(v)) if v.size else 0.0)
    err = np.abs(got - want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = np.isnan(want) | (err <= bound)
    assert ok.all(), np.nanmax(err / np.maximum(bound, 1e-300))
    return got


def make(seed, Bk, H_kv, S_max, D):
    rng = np.random.default_rng(seed)
    k, v = (np.float32(rng.standard_normal((Bk, H_kv, S_max, D))).astype(float) for _ in range(2))
    return Cache.of(k, v), rng


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,H_kv,starts,counts", [
    (1, 1, 1, [0], None), (3, 1, 4, [5, 0, 19], None), (2, 7, 3, [3, 13], [7, 4]),
    (3, 5, 2, [-2, 17, 2 ** 31 - 3], [5, 5, 5]), (2, 4, 2, [0, 4], [0, -3]),
    (2, 20, 2, [0, 0], [99, 20])])
def test_append(B, S, H_kv, starts, counts, D, dtype):
    """Rows land where they belong; rows past the counts or outside the cache are left out and
    every other byte stays."""
    S_max = 20
    rng = np.random.default_rng(S * 10 + B)
    cache = Cache(B, H_kv, S_max, D, fill=0x5A)
    (kr, k), (vr, v) = (ref.typed(rng.standard_normal((B, S, H_kv, D)), dtype) for _ in range(2))
    append(cache, kr, vr, dtype, starts, counts)
    for x, (codes, scales) in zip((k, v), cache.raw()):
        want_c, want_s = np.full_like(codes, 0x5A), np.full_like(scales, 0x5A)
        for b in range(B):
            for s in range(min(S, S if counts is None else counts[b])):
                at = starts[b] + s
                if 0 <= at < S_max:
                    want_c[b, :, at], want_s[b, :, at] = ref.pack(x[b, s])
        np.testing.assert_array_equal(scales, want_s)
        np.testing.assert_array_equal(codes, want_c)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_strides(dtype):
    """[B, H, S, D] rows, and a base that is not 16-byte aligned."""
    B, S, H, D = 2, 6, 3, 64
    rng = np.random.default_rng(8)
    (kr, k), (vr, v) = (ref.typed(rng.standard_normal((B, H, S, D)), dtype) for _ in range(2))
    for shift in (0, 1):
        cache = Cache(B, H, S, D)
        append(cache, kr.reshape(B, S, H, D), vr.reshape(B, S, H, D), dtype, [0, 0],
               strides=(H * S * D, S * D, D), shift=shift)
        for x, (codes, scales) in zip((k, v), cache.raw()):
            want = ref.pack(x.reshape(-1, D))
            np.testing.assert_array_equal(codes.reshape(want[0].shape), want[0])
            np.testing.assert_array_equal(scales.reshape(want[1].shape), want[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv", [(4, 4), (8, 2), (24, 1)])
@pytest.mark.parametrize("S", [1, 2, 15, 31, 32, 33, 64, 130, 517])
def test_one_query(S, H, H_kv, D, dtype):
    print(f"kv4 S={S} H={H}/{H_kv} D={D} dtype={dtype}", flush=True)
    cache, rng = make(S, 2, H_kv, S + 3, D)
    raw, q = ref.typed(rng.standard_normal((2, 1, H, D)) * 2, dtype)
    check(cache, raw, q, dtype, [S, max(1, S // 2)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S_q,S,H,H_kv", [
    (2, 2, 4, 4), (3, 70, 4, 2), (9, 40, 6, 1), (17, 17, 2, 2), (40, 200, 4, 2), (130, 131, 2, 1),
    (70, 5, 2, 2)])
def test_many_queries(S_q, S, H, H_kv, causal, D, dtype):
    """S_q > S under a causal mask leaves the first rows without a key: zeros."""
    print(f"kv4 S_q={S_q} S={S} H={H}/{H_kv} D={D} causal={causal} dtype={dtype}", flush=True)
    cache, rng = make(S_q + S, 2, H_kv, S + 1, D)
    raw, q = ref.typed(rng.standard_normal((2, S_q, H, D)) * 2, dtype)
    got = check(cache, raw, q, dtype, [S, S - 1], causal=causal)
    if causal and S_q > S:
        assert (got[0, :S_q - S] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S_q", [1, 6, 90])
def test_ragged_batches(S_q, causal, dtype):
    """Lengths of zero, one, negative and past S_max; counts of zero, fewer and more than S_q."""
    lens = [0, 1, 300, 77, -5, 1000, 150]
    counts = [S_q, S_q, S_q - 1, 0, S_q, S_q + 9, 1]
    cache, rng = make(5, len(lens), 2, 300, 64)
    raw, q = ref.typed(rng.standard_normal((len(lens), S_q, 4, 64)), dtype)
    check(cache, raw, q, dtype, lens, counts, causal, pad=3)
    check(cache, raw, q, dtype, lens, None, causal, pad=8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S_q", [1, 100])
def test_shared_cache(S_q, dtype):
    """One sequence for every batch entry."""
    cache, rng = make(6, 1, 2, 90, 128)
    raw, q = ref.typed(rng.standard_normal((3, S_q, 2, 128)), dtype)
    check(cache, raw, q, dtype, [88], causal=False)
    check(cache, raw, q, dtype, [88], [S_q, 1, S_q], causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S_q", [1, 40, 150])
def test_one_key_is_its_value(S_q, D, dtype):
    """A softmax over one key: V's row, bit for bit."""
    cache, rng = make(7, 1, 2, 64, D)
    raw, _ = ref.typed(rng.standard_normal((1, S_q, 4, D)) * 30, dtype)
    got = attend(cache, raw, dtype, [1], causal=False)
    v = cache.values()[1][0, :, 0]
    np.testing.assert_array_equal(got, np.broadcast_to(np.repeat(v, 2, 0), got.shape))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S_q", [1, 33, 140])
def test_scores_far_apart(S_q, dtype):
    """Scores of several hundred, a scale of zero, a negative scale."""
    cache, rng = make(9, 1, 2, 200, 64)
    raw, q = ref.typed(rng.standard_normal((1, S_q, 2, 64)) * 40, dtype)
    for scale in (1.0, 0.0, -0.3):
        check(cache, raw, q, dtype, [190], causal=False, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S_q", [1, 5, 40, 130])
def test_nan_stays_with_the_rows_that_see_it(S_q, D, dtype):
    """Bytes past the length are never used (0xFF: NaN scales), a NaN group of V reaches its
    dimensions of the rows that see the key, a NaN group of K makes those rows NaN."""
    S = 150
    cache, rng = make(10, 2, 2, S + 20, D)
    k, v = cache.values()
    for x, buf_c, buf_s in ((k, 0, 1), (v, 2, 3)):
        codes, scales = ref.pack(x.reshape(-1, D))
        codes = codes.reshape(2, 2, S + 20, -1)
        scales = scales.reshape(2, 2, S + 20, -1)
        codes[:, :, S:], scales[:, :, S:] = 0xFF, 0xFF
        if buf_s == 3:
            scales[0, 0, S - 3, 1] = 255   # seen by the last three queries
            scales[0, 1, 2, 0] = 255       # seen by all
        else:
            scales[1, 1, S - 2, 0] = 255
        cache.bufs[buf_c].put(codes, 0)
        cache.bufs[buf_s].put(scales, 0)
    raw, q = ref.typed(rng.standard_normal((2, S_q, 4, D)), dtype)
    with np.errstate(invalid="ignore"):
        got = check(cache, raw, q, dtype, [S, S])
    assert np.isnan(got[0, -1, 0]).sum() == 32 and np.isnan(got[1, -1, 2:]).all()
    if S_q > 3:
        assert not np.isnan(got[0, :S_q - 3, :2]).any()
        assert not np.isnan(got[1, :S_q - 2]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinite_queries(dtype):
    """A query's NaN is its own row's; an infinite query gives NaN (inf - inf) in its own row."""
    cache, rng = make(11, 1, 1, 100, 64)
    x = rng.standard_normal((1, 40, 1, 64))
    x[0, 3, 0, 9] = np.nan
    x[0, 7, 0, 1] = np.inf
    raw, _ = ref.typed(x, dtype)
    got = attend(cache, raw, dtype, [100], causal=False)
    bad = np.isnan(got).any(-1)[0, :, 0]
    assert bad[3] and bad[7] and bad.sum() == 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S_q", [1, 70])
def test_long_cache(S_q, dtype):
    """Keys shared out over workgroups and joined; and the same call twice, bit for bit."""
    cache, rng = make(12, 1, 1, 9000, 128)
    raw, q = ref.typed(rng.standard_normal((1, S_q, 2, 128)) * 3, dtype)
    got = check(cache, raw, q, dtype, [8999])
    np.testing.assert_array_equal(attend(cache, raw, dtype, [8999]), got)
    check(cache, raw, q, dtype, [40])  # most shares are empty
