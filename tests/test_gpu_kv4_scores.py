"""Attention over a 4-bit cache where scores are infinite, or large and close to each other, and where
a value is NaN behind a weight of zero: each kernel, with its keys in one workgroup and shared out
over several, so that every place that joins partial results is met."""
import numpy as np
import pytest

import mx4_ref as ref
import test_gpu_kv4 as kv4
from anima_hip import rt

pytestmark = pytest.mark.gpu

F, B = ref.F32, ref.BF16
U = kv4.U

# (dtype, B, S_q, H, H_kv, D, S, kernel, row blocks, splits), one cached sequence for all entries.
SHAPES = [(t, 1, 3, 16, 4, D, 300, "token", 1, 1) for t in (F, B) for D in (64, 128)]
SHAPES += [(t, 1, 3, 16, 4, D, 3000, "token", 1, 16) for t in (F, B) for D in (64, 128)]
SHAPES += [(F, 72, 5, 32, 8, 64, 300, "token", 2, 1), (B, 72, 5, 32, 8, 128, 300, "token", 2, 1),
           (F, 40, 5, 8, 2, 64, 3000, "token", 2, 8), (B, 40, 5, 8, 2, 64, 3000, "token", 2, 8),
           (B, 40, 5, 8, 2, 128, 3000, "token", 2, 4),
           (F, 1, 300, 64, 64, 64, 140, "tile", 1, 1), (F, 1, 500, 64, 64, 128, 70, "tile", 1, 1),
           (B, 1, 300, 64, 64, 64, 300, "tile", 1, 1), (B, 1, 300, 64, 64, 128, 300, "tile", 1, 1),
           (F, 1, 500, 8, 1, 64, 9000, "tile", 1, 16), (B, 1, 250, 16, 1, 64, 5000, "tile", 1, 8),
           (B, 1, 250, 16, 1, 128, 5000, "tile", 1, 8)]
EACH = pytest.mark.parametrize("dtype,Bn,S_q,H,H_kv,D,S,kernel,blocks,splits", SHAPES)


def some(x):
    """The first, a middle and the last batch entry."""
    return x[sorted({0, len(x) // 2, len(x) - 1})]


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@EACH
@pytest.mark.parametrize("scale", [0.1, -0.3])
def test_infinite_scores_weigh_nothing(dtype, Bn, S_q, H, H_kv, D, S, kernel, blocks, splits, scale):
    """Scores of -2^140, -inf in f32, on the first 32, 64, 128 or half of the keys, on every second
    one, and on all: the attention over the others, and zeros where there is no other.

    The bound is test_gpu_kv4.py's on the keys that are left, whose dimension 0 is zero."""
    print(f"{kernel} {blocks} {splits} D={D} dtype={dtype} scale={scale}", flush=True)
    rng = np.random.default_rng(S + D)
    base, v = (np.float32(rng.standard_normal((1, H_kv, S, D))).astype(float) for _ in range(2))
    base[..., 0] = 0
    q = rng.standard_normal((Bn, S_q, H, D))
    q[..., 0] = -2.0 ** 70 * np.sign(scale)
    raw, q = ref.typed(q, dtype)
    key = np.arange(S)
    for out in (key < 32, key < 64, key < 128, key < S // 2, key % 2 == 0, key >= 0):
        k = base.copy()
        k[..., out, 0] = 2.0 ** 70
        cache = kv4.Cache.of(k, v)
        got = kv4.attend(cache, raw, dtype, [S], None, False, scale)
        if out.all():
            assert (got == 0).all()
            continue
        kc, vc = cache.values()
        kc, vc, qq = kc[:, :, ~out], vc[:, :, ~out], q.copy()
        qq[..., 0] = 0
        got, qq = some(got), some(qq)
        want, mag = ref.attention_rows(qq, kc, vc, [kc.shape[2]], None, False, scale)
        d = (3 * D + 6) * U * abs(scale) * np.abs(qq).sum(-1, keepdims=True) * np.abs(kc).max()
        r = 2.0 ** -8 if dtype == B else 0.0
        bound = ((4 * d + (S + 64) * U + r) * mag + ref.HALF[dtype] * np.abs(want)
                 + S * 2.0 ** -126 * np.abs(vc).max())
        assert (np.abs(got - want) <= bound).all(), out.sum()


@EACH
@pytest.mark.parametrize("far", [300.0, np.inf])
def test_nan_value_behind_a_weight_of_zero(dtype, Bn, S_q, H, H_kv, D, S, kernel, blocks, splits, far):
    """One key has a score `far` above all others, whose weights are zero in f32 beside it (far
    scores of -inf: -2^140).  A NaN group of V among the others reaches its 32 dimensions wherever
    its key lies; the rest of the row is the far key's value, bit for bit."""
    print(f"{kernel} {blocks} {splits} D={D} dtype={dtype} far={far}", flush=True)
    rng = np.random.default_rng(S)
    top, size = S // 2, 2.0 ** 70 if far == np.inf else 16.0
    k, v = np.zeros((1, H_kv, S, D)), rng.standard_normal((1, H_kv, S, D))
    k[..., 0] = size
    k[:, :, top, 0] = 0
    q = np.zeros((Bn, S_q, H, D))
    q[..., 0] = -size if far == np.inf else -far
    raw, q = ref.typed(q, dtype)
    cache = kv4.Cache.of(k, v)
    codes, scales = cache.raw()[1]
    value = np.repeat(cache.values()[1][0, :, top], H // H_kv, 0)
    at = sorted(n for n in {0, 5, 31, 33, 64, 100, S // 3, top - 1, top + 1, S - 33, S - 2, S - 1}
                if n < S)
    for nan in at:
        bad = scales.copy()
        bad[0, nan % H_kv, nan, 1] = 255
        cache.bufs[3].put(bad, 0)
        got = kv4.attend(cache, raw, dtype, [S], None, False, 1 / 16)
        want = np.broadcast_to(value, got.shape).copy()
        group = H // H_kv
        want[:, :, nan % H_kv * group:(nan % H_kv + 1) * group, 32:64] = np.nan
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=str(nan))
        ok = ~np.isnan(want)
        np.testing.assert_array_equal(got[ok], want[ok])


# Scores that are exact in f32, their distances a few steps of f32 apart: a weight is off by the
# rounding of its exponent's two products, each at most 64 in log2 units, and of the exponential.
WEIGHT = 4 * 64 * U
LOG2E = 1.4426950408889634


def check_exact_scores(cache, q, raw, dtype, scale):
    k, v = cache.values()
    S = k.shape[2]
    got = some(kv4.attend(cache, raw, dtype, [S], None, False, scale))
    want, mag = ref.attention_rows(some(q), k, v, [S], None, False, scale)
    r = 2.0 ** -8 if dtype == B else 0.0
    bound = ((2 * WEIGHT + (S + 64) * U + r) * mag + ref.HALF[dtype] * np.abs(want)
             + S * 2.0 ** -126)
    err = np.abs(got - want)
    assert (err <= bound).all(), (err / bound).max()


@EACH
@pytest.mark.parametrize("power", [10, 21, 24, 27, 40])
def test_large_scores_keep_their_distances(dtype, Bn, S_q, H, H_kv, D, S, kernel, blocks, splits,
                                           power):
    """Scores of q0 + 0 to 6 steps, q0 between 2^power and 2^(power + 1) and a step f32's there (at
    least 1): one number of steps to a run of 32 keys, of which waves take their turns, and less
    of them in every third part of the keys, which splits share out.  At a scale of 2 / step a
    step is 2.9 in log2 units.  V is 1 where the score is high and -1 or 1 where it is low,
    so that a weight's error is the result's."""
    print(f"{kernel} {blocks} {splits} D={D} dtype={dtype} 2^{power}", flush=True)
    step = max(1.0, 2.0 ** (power - 23))
    rng = np.random.default_rng(power)
    runs = np.array([0, 1.0, 2, 3, 4, 6])[rng.integers(0, 6, S // 32 + 1)]
    k, v = np.zeros((1, H_kv, S, D)), np.ones((1, H_kv, S, D))
    k[..., 0] = 1
    for h in range(H_kv):
        steps = np.roll(runs, h)[np.arange(S) // 32]
        part = np.arange(S) * 16 // S
        k[0, h, :, 32] = np.where((part + h) % 3 == 0, np.minimum(steps, 2), steps)
        v[0, h, :, ::2] = np.where(k[0, h, :, 32] >= 3, 1, -1)[:, None]
        v[0, h, :, 1::2] = np.where(np.arange(S) // 32 % 2, 1, -1)[:, None]
    cache = kv4.Cache.of(k, v)
    for c0 in (1.0, 1.375, 1.625, -1.125):
        q = np.zeros((Bn, S_q, H, D))
        q[..., 0] = c0 * 2.0 ** power * (1 + np.arange(S_q)[None, :, None] % 4 / 64)
        q[..., 32] = step
        raw, q = ref.typed(q, dtype)
        for scale in (2 / step, 1 / step, 0.25 / step):
            check_exact_scores(cache, q, raw, dtype, scale)


@EACH
@pytest.mark.parametrize("high", [1, 30])
def test_rising_scores_keep_their_distances(dtype, Bn, S_q, H, H_kv, D, S, kernel, blocks, splits,
                                            high):
    """Scores of about 2^25 of which the last key's is some 10 higher in log2 units, where a running
    maximum moves (in the last case past 2^24 of them); every second row's scores rise by 2^(24 +
    high) in the half behind.  Keys before weigh what they should beside those behind, whatever
    the rows beside them do."""
    print(f"{kernel} {blocks} {splits} D={D} dtype={dtype} high={high}", flush=True)
    k, v = np.zeros((1, H_kv, S, D)), np.ones((1, H_kv, S, D))
    key = np.arange(S)
    k[..., 0] = 1
    k[..., 32] = np.where(key == S - 1, 6, 0)
    k[..., 33] = np.where(key >= S // 2, 1, 0)
    v[..., ::2] = np.where(key >= S // 2, 1, -1)[None, None, :, None]
    v[..., 1::2] = np.where(key == S - 1, 1, -1)[None, None, :, None]
    cache = kv4.Cache.of(k, v)
    for c0, rise, scale in ((1.0, 4, 0.275), (1.5, 8, 0.1375), (-1.25, 8, 0.1375), (1.75, 8, 0.15),
                            (1.109375, 4, 0.26), (1.25, 4, (2 ** 24 - 4) / (LOG2E * 1.25 * 2 ** 25))):
        q = np.zeros((Bn, S_q, H, D))
        q[..., 0] = c0 * 2.0 ** 25
        q[:, ::2, :, 32] = rise
        q[:, 1::2, :, 33] = 2.0 ** (24 + high)
        raw, q = ref.typed(q, dtype)
        check_exact_scores(cache, q, raw, dtype, scale)


@EACH
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -126, -2.0 ** -126])
def test_distances_past_the_range(dtype, Bn, S_q, H, H_kv, D, S, kernel, blocks, splits, scale):
    """Scores of 1.5 * 2^127 and its negative, whose distance f32 does not hold: under a scale of zero
    all keys weigh the same, and under a small one the lower ones e^-6 of the one higher key."""
    print(f"{kernel} {blocks} {splits} D={D} scale={scale}", flush=True)
    k, v = np.zeros((1, H_kv, S, D)), np.ones((1, H_kv, S, D))
    key = np.arange(S)
    high = key // 32 % 3 == 1 if scale == 0 else key == S // 2
    k[..., 0] = np.where(high, 1.5, -1.5) * 2.0 ** 63
    v[..., ::2] = np.where(key // 32 % 2, 1, -1)[None, None, :, None]
    cache = kv4.Cache.of(k, v)
    q = np.zeros((Bn, S_q, H, D))
    q[..., 0] = 2.0 ** 64 * (1 if scale >= 0 else -1)
    raw, q = ref.typed(q, dtype)
    check_exact_scores(cache, q, raw, dtype, scale)
