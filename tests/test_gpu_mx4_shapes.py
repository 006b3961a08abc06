"""Every shape of the 4-bit linear layer's staged tiles and of the tile attention kernel, at sizes
that reach it (tests/test_mx4_plan.py holds them to their shapes on the CPU), with the bounds of
test_gpu_mx4.py and test_gpu_kv4.py."""
import numpy as np
import pytest

import mx4_ref as ref
import test_gpu_kv4 as kv4
import test_gpu_mx4 as mx4
from anima_hip import rt

pytestmark = pytest.mark.gpu

F, B = ref.F32, ref.BF16

# (dtype, M, N, K, plan): ragged M and N wherever the size allows it.
LINEAR = [(B, 4600, 8190, 128, "staged 0 1"), (B, 4000, 6199, 128, "staged 1 1"),
          (B, 1500, 2100, 256, "staged 2 1"), (B, 700, 2047, 256, "staged 3 1"),
          (B, 333, 2001, 1024, "staged 4 1"), (B, 130, 1001, 384, "staged 5 1"),
          (B, 33, 300, 4096, "staged 5 8"), (B, 90, 2001, 8192, "staged 3 8"),
          (F, 2040, 8190, 128, "staged 0 1"), (F, 3000, 2001, 128, "staged 1 1"),
          (F, 900, 2047, 256, "staged 2 1"), (F, 100, 1001, 384, "staged 3 1"),
          (F, 333, 2001, 8192, "staged 1 8"), (F, 33, 300, 2048, "staged 3 8"),
          # K padded to 128 in copies, and the plain tiles.
          (B, 333, 2001, 1501, "pad"), (F, 333, 1001, 1000, "pad"), (B, 40, 4000, 700, "pad"),
          (B, 100, 300, 1000, "tiles"), (F, 30, 1001, 333, "tiles")]

# (dtype, B, S_q, H, H_kv, D, S, causal, plan)
ATTEND = [(B, 1, 300, 64, 64, 128, 70, False, "tile 1"), (B, 1, 300, 64, 64, 64, 70, True, "tile 1"),
          (F, 1, 500, 64, 64, 128, 70, True, "tile 1"), (F, 1, 300, 64, 64, 64, 70, False, "tile 1"),
          (B, 2, 520, 32, 32, 128, 200, True, "tile 1"), (F, 2, 520, 32, 16, 64, 200, True, "tile 1"),
          (B, 1, 250, 16, 1, 128, 9000, False, "tile 8"), (B, 1, 700, 8, 1, 64, 9000, False, "tile 8"),
          (F, 1, 500, 8, 1, 64, 8000, False, "tile 16"), (B, 1, 600, 4, 1, 128, 20000, True, "tile 16"),
          (B, 1, 64, 8, 1, 128, 20000, True, "token 16"), (F, 1, 300, 6, 1, 64, 3000, True, "token")]


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("dtype,M,N,K,plan", LINEAR)
def test_linear_shapes(dtype, M, N, K, plan):
    print(f"linear_mx4 M={M} N={N} K={K} dtype={dtype} {plan}", flush=True)
    mx4.check_linear(M, N, K, dtype, M + N + K)


@pytest.mark.parametrize("dtype,M,N,K,plan", [c for c in LINEAR if c[1] * c[2] * c[3] < 2e9])
def test_linear_shapes_are_exact_without_additions(dtype, M, N, K, plan):
    """W with one power of two per row: every bit of A's terms, at every row and column."""
    rng = np.random.default_rng(K)
    x = rng.standard_normal((M, K)) * np.exp2(rng.integers(-60, 60, (M, K)).astype(float))
    raw, a = ref.typed(x, dtype)
    cols = rng.integers(0, K, N)
    w = np.zeros((N, K))
    w[np.arange(N), cols] = np.exp2(rng.integers(-9, 9, N).astype(float)) * rng.choice([-1, 1], N)
    codes, scales = ref.pack(w)
    got = mx4.linear(raw, codes, scales, K, N, dtype)
    np.testing.assert_array_equal(got, a[:, cols] * w[np.arange(N), cols])


@pytest.mark.parametrize("dtype,M,N,K", [(B, 1500, 2100, 256), (F, 1030, 2047, 256),
                                         (B, 333, 2001, 1501), (F, 100, 1001, 384)])
def test_linear_shapes_infinities_and_nan(dtype, M, N, K):
    a = np.ones((M, K))
    a[0, 5], a[M - 1, K - 1], a[M // 2, 40] = np.inf, np.nan, -np.inf
    raw, val = ref.typed(a, dtype)
    codes, scales = ref.pack(np.full((N, K), 1.5))
    scales[7, 1] = 255
    scales[N - 1, -1] = 255
    got = mx4.linear(raw, codes, scales, K, N, dtype)
    with np.errstate(invalid="ignore"):
        # Sums of 1.5, exact in f32, rounded once to the output's type (2251.5 is not a bf16 number).
        want = ref.typed(val @ ref.unpack(codes, scales, K).T, dtype)[1]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    np.testing.assert_array_equal(got[ok], want[ok])


@pytest.mark.parametrize("dtype,M,N,K,lda,shift", [(B, 700, 2047, 256, 264, 8), (F, 100, 1001, 384, 388, 4),
                                                   (B, 700, 300, 256, 257, 0), (F, 100, 1001, 384, 384, 1),
                                                   (B, 333, 2001, 1501, 1503, 1)])
def test_linear_shapes_strides(dtype, M, N, K, lda, shift):
    mx4.check_linear(M, N, K, dtype, 5, lda=lda, shift=shift, ldc=N + 3)


def check_rows(cache, raw, q, dtype, lens, counts, causal, scale=None, pad=0):
    D = q.shape[-1]
    sc = D ** -0.5 if scale is None else scale
    k, v = cache.values()
    got = kv4.attend(cache, raw, dtype, lens, counts, causal, scale, pad)
    want, mag = ref.attention_rows(q, k, v, lens, counts, causal, sc)
    d = (3 * D + 6) * kv4.U * abs(sc) * np.abs(q).sum(-1, keepdims=True) * np.nanmax(np.abs(k))
    n = min(max(lens), k.shape[2])
    r = 2.0 ** -8 if dtype == B else 0.0
    bound = ((4 * d + (n + 64) * kv4.U + r) * mag + ref.HALF[dtype] * np.abs(want)
             + n * 2.0 ** -126 * np.nanmax(np.abs(v)))
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    err = np.abs(got - want)
    assert (np.isnan(want) | (err <= bound)).all(), np.nanmax(err / bound)
    return got


@pytest.mark.parametrize("dtype,Bn,S_q,H,H_kv,D,S,causal,plan", ATTEND)
def test_attention_shapes(dtype, Bn, S_q, H, H_kv, D, S, causal, plan):
    print(f"kv4 B={Bn} S_q={S_q} H={H}/{H_kv} D={D} S={S} causal={causal} {plan}", flush=True)
    cache, rng = kv4.make(S, Bn, H_kv, S, D)
    raw, q = ref.typed(rng.standard_normal((Bn, S_q, H, D)) * 2, dtype)
    got = check_rows(cache, raw, q, dtype, [S] * Bn, None, causal)
    np.testing.assert_array_equal(kv4.attend(cache, raw, dtype, [S] * Bn, None, causal), got)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_ragged_masked_and_nan(D, dtype):
    """The tile kernel with lengths of 0, 1, below S_q, above S_max; counts of 0 and between; bytes
    past the lengths 0xFF; NaN groups of V that some rows may not see; rows of odd strides."""
    Bn, S_q, H, S = 5, 300, 32, 140
    cache, rng = kv4.make(3, Bn, H, S, D)
    k, v = cache.values()
    lens = [0, 1, 77, 1000, 140]
    for x, at in ((k, 0), (v, 2)):
        codes, scales = ref.pack(x.reshape(-1, D))
        codes = codes.reshape(Bn, H, S, -1)
        scales = scales.reshape(Bn, H, S, -1)
        for b, n in enumerate(lens):
            codes[b, :, n:], scales[b, :, n:] = 0xFF, 0xFF
        if at == 2:
            scales[2, 3, 70, 0] = 255   # seen by the last seven queries
            scales[4, 5, 2, 1] = 255
        else:
            scales[3, 7, 139, 0] = 255  # seen by the last query
        cache.bufs[at].put(codes, 0)
        cache.bufs[at + 1].put(scales, 0)
    raw, q = ref.typed(rng.standard_normal((Bn, S_q, H, D)), dtype)
    with np.errstate(invalid="ignore"):
        for counts, causal, pad in ((None, True, 0), ([300, 0, 200, 300, 17], True, 3),
                                    (None, False, 8)):
            check_rows(cache, raw, q, dtype, lens, counts, causal, pad=pad)


@pytest.mark.parametrize("dtype", [B, F])
def test_tiles_scales(dtype):
    """Scores of several hundred, a scale of zero, a negative one, an infinite and a NaN query."""
    cache, rng = kv4.make(4, 1, 64, 130, 64)
    raw, q = ref.typed(rng.standard_normal((1, 300, 64, 64)) * 40, dtype)
    for scale in (1.0, 0.0, -0.3):
        check_rows(cache, raw, q, dtype, [129], None, True, scale)
    x = rng.standard_normal((1, 300, 64, 64))
    x[0, 30, 3, 9], x[0, 171, 5, 1] = np.nan, np.inf
    raw, _ = ref.typed(x, dtype)
    got = kv4.attend(cache, raw, dtype, [130], causal=False)
    bad = np.isnan(got).any(-1)
    assert bad[0, 30, 3] and bad[0, 171, 5] and bad.sum() == 2


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_one_key_is_its_value(D, dtype):
    cache, rng = kv4.make(8, 1, 64, 64, D)
    raw, _ = ref.typed(rng.standard_normal((1, 300, 64, D)) * 30, dtype)
    got = kv4.attend(cache, raw, dtype, [1], causal=False)
    np.testing.assert_array_equal(got, np.broadcast_to(cache.values()[1][0, :, 0], got.shape))
