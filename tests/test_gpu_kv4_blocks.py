"""Attention over a 4-bit cache with 17 to 32 query rows per K/V head in many sequences: the token
kernel with two blocks of rows."""
import numpy as np
import pytest

import mx4_ref as ref
import test_gpu_kv4 as kv4
import test_gpu_mx4_shapes as shapes
from anima_hip import rt

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.BF16]
# B, S_q, H, H_kv, S_max: 20 and 21 rows (a second block of 4 and 5), 32 in four splits.
CASES = [(72, 5, 32, 8, 300), (72, 7, 24, 8, 333), (16, 8, 32, 8, 5000)]


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S_q,H,H_kv,S", CASES)
def test_ragged_masked_and_nan(B, S_q, H, H_kv, S, D, causal, dtype):
    """Lengths of 0, 1, below S_q, up to S_max and past it; counts of 0 and between; bytes past
    the lengths 0xFF; NaN groups of V and of K near the ends, which some rows may not see."""
    rng = np.random.default_rng(B + S_q)
    cache = kv4.Cache(B, H_kv, S, D)
    lens = [[0, 1, S_q - 1, S + 9, S, S // 3, 64, S - 31][b % 8] for b in range(B)]
    counts = [[S_q, 1, S_q, S_q, S_q + 3, S_q - 2, S_q, 0][b % 8] for b in range(B)]
    kv = []
    for at in (0, 2):
        codes = rng.integers(0, 256, (B, H_kv, S, D // 2), np.uint8)
        scales = rng.integers(124, 128, (B, H_kv, S, D // 32), np.uint8)
        for b in range(B):
            n = min(lens[b], S)
            codes[b, :, n:] = 0xFF
            scales[b, :, n:] = 0xFF
            if b % 8 in (3, 5):
                scales[b, 1, n - 1 if at else n - 2, 1] = 0xFF
        cache.bufs[at].put(codes, 0)
        cache.bufs[at + 1].put(scales, 0)
        x = ref.unpack(codes, scales, D)
        for b in range(B):
            x[b, :, min(lens[b], S):] = 0  # not used
        kv.append(x)
    k, v = kv
    raw, q = ref.typed(rng.standard_normal((B, S_q, H, D)) * 0.5, dtype)
    got = kv4.attend(cache, raw, dtype, lens, counts, causal, None, 1)
    want, mag = ref.attention_rows(q, k, v, lens, counts, causal, D ** -0.5)
    d = (3 * D + 6) * kv4.U * D ** -0.5 * np.abs(q).sum(-1, keepdims=True) * np.nanmax(np.abs(k))
    r = 2.0 ** -8 if dtype == ref.BF16 else 0.0
    bound = ((4 * d + (S + 64) * kv4.U + r) * mag + ref.HALF[dtype] * np.abs(want)
             + S * 2.0 ** -126 * np.nanmax(np.abs(v)))
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(want).any() and not np.isnan(want).all()
    assert (np.isnan(want) | (np.abs(got - want) <= bound)).all()
    np.testing.assert_array_equal(kv4.attend(cache, raw, dtype, lens, counts, causal, None, 1), got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 40.0])
def test_scales(scale, dtype):
    B, S_q, H, H_kv, S = CASES[1]
    cache, rng = kv4.make(5, B, H_kv, S, 64)
    raw, q = ref.typed(rng.standard_normal((B, S_q, H, 64)), dtype)
    shapes.check_rows(cache, raw, q, dtype, [S] * B, None, True, scale)
