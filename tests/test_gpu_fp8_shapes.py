"""The linear layer on 8-bit rows on the GPU: sizes that reach each of its kernels' shapes, whole
and with K shared out, against 64-bit numpy.

tests/test_fp8_plan.py holds on the CPU that each case reaches the shape beside it.  The whole
output is held to the error of the format's products with the sum of magnitudes for the largest of
eight; rows at tile borders to the bound of tests/test_gpu_fp8.py."""
import numpy as np
import pytest

import fp8_ref as ref
import test_gpu_fp8 as gpu
from anima_hip import rt
from fp8_ref import BF16, F32

pytestmark = pytest.mark.gpu

# dtype, M, N, K, plan.
SHAPES = [
    (BF16, 1, 17, 33, "few 1"), (BF16, 5, 31, 139, "few 2"), (BF16, 21, 50, 460, "few 4"),
    (BF16, 18, 70, 1046, "few 8"), (BF16, 1812, 6667, 410, "tile 0 1"),
    (BF16, 2567, 3082, 32, "tile 1 1"), (BF16, 7207, 513, 9956, "tile 1 2"),
    (BF16, 980, 4219, 971, "tile 2 1"), (BF16, 341, 5470, 6429, "tile 2 3"),
    (BF16, 3745, 1128, 33, "tile 3 1"), (BF16, 5839, 349, 7621, "tile 3 3"),
    (BF16, 639, 3393, 32, "tile 4 1"), (BF16, 2861, 17, 6271, "tile 4 10"),
    (BF16, 514, 7090, 39, "tile 5 1"), (BF16, 2, 5680, 6798, "tile 5 11"),
    (BF16, 167, 5446, 35, "tile 6 1"), (BF16, 757, 18, 4403, "few 8"),
    (BF16, 762, 18, 5710, "tile 6 15"),
    (BF16, 4722, 69, 1219, "tile 7 1"), (BF16, 120, 1411, 3757, "tile 7 3"),
    (BF16, 994, 494, 32, "few 1"),
    (BF16, 83, 6162, 35, "tile 8 1"), (BF16, 1, 16, 5319, "tile 8 14"),
    (BF16, 36, 6702, 136, "tile 9 1"), (BF16, 1, 19, 7167, "tile 9 14"),
    (F32, 1, 17, 33, "few 1"), (F32, 5, 31, 139, "few 2"), (F32, 21, 50, 460, "few 4"),
    (F32, 18, 70, 1012, "few 8"), (F32, 1826, 6603, 514, "tile 0 1"),
    (F32, 4128, 1921, 32, "tile 1 1"), (F32, 2904, 1468, 130, "tile 2 1"),
    (F32, 387, 4928, 7451, "tile 2 3"), (F32, 1510, 2753, 33, "tile 3 1"),
    (F32, 3308, 72, 9805, "tile 3 8"), (F32, 5889, 352, 32, "tile 4 1"),
    (F32, 1572, 67, 5693, "tile 4 8"), (F32, 309, 3491, 672, "tile 5 1"),
    (F32, 2074, 69, 7131, "tile 5 7"), (F32, 3294, 274, 32, "tile 6 1"),
    (F32, 2784, 17, 3286, "tile 6 9"), (F32, 4298, 74, 908, "tile 7 1"),
    (F32, 2784, 18, 6101, "tile 7 4"), (F32, 2515, 268, 32, "tile 8 1"),
    (F32, 1, 17, 7518, "tile 8 15"), (F32, 34, 8103, 157, "tile 9 1"),
    (F32, 1, 16, 6367, "tile 9 13"),
]


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("dtype,M,N,K,plan", SHAPES)
def test_shape(dtype, M, N, K, plan):
    a, w = gpu.linear_inputs(M, N, K, M + N + K)
    odd = plan.endswith(" 1") and M % 2  # rows and a start that no wide store fits
    got = gpu.linear_dev(a, w, K, dtype, N + 3 if odd else None, 1 if odd else 0)
    av, wv = ref.unpack(*a, K), ref.unpack(*w, K)
    want, mag = av @ wv.T, np.abs(av) @ np.abs(wv).T
    tol = (K + 16) * 2.0 ** -24 * mag + ref.HALF[dtype] * np.abs(want)
    if dtype == BF16:
        tol += 7 * 2.0 ** -13 * mag
    assert (np.abs(got - want) <= tol).all()
    rows = np.unique(np.array([0, 31, 32, 63, 64, 191, 192, 255, 256, M - 1]).clip(0, M - 1))
    cols = np.unique(np.array([0, 31, 32, 63, 64, 127, 128, 255, 256, N - 1]).clip(0, N - 1))
    gpu.check_linear(got[rows][:, cols], tuple(x[rows] for x in a), tuple(x[cols] for x in w), K,
                     dtype)


@pytest.mark.parametrize("dtype,M,N,K", [(BF16, 1907, 1894, 2324), (F32, 1907, 1894, 2324),
                                         (BF16, 24, 2048, 8192), (F32, 24, 2048, 8192),
                                         (BF16, 3, 700, 900), (F32, 3, 700, 900)])
def test_same_bits_every_time(dtype, M, N, K):
    """No sum's order depends on the run."""
    a, w = gpu.linear_inputs(M, N, K, 3)
    first = gpu.linear_dev(a, w, K, dtype)
    for _ in range(3):
        np.testing.assert_array_equal(gpu.linear_dev(a, w, K, dtype), first)


@pytest.mark.parametrize("dtype,plan", [(BF16, "tile 6 15"), (F32, "tile 8 13")])
def test_nan_groups_in_split_k(dtype, plan):
    """A NaN group in one part of K reaches its row or column through the sum of the parts."""
    M, N, K = (762, 18, 5710) if dtype == BF16 else (1, 19, 6491)
    a, w = gpu.linear_inputs(M, N, K, 9)
    clean = gpu.linear_dev(a, w, K, dtype)
    w[1][N // 3, 30] = 255
    w[0][N // 3, 30 * 128:31 * 128] = 0
    got = gpu.linear_dev(a, w, K, dtype)
    assert np.isnan(got[:, N // 3]).all()
    keep = np.arange(N) != N // 3
    np.testing.assert_array_equal(got[:, keep], clean[:, keep])
