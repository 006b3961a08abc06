"""Where the 8-bit operators round, on the GPU against 64-bit numpy: the norm's results below f32's
normal numbers, and products whose large terms cancel."""
import numpy as np
import pytest

import fp8_ref as ref
import test_gpu_fp8 as gpu
from anima_hip import rt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("rows,K", [(5, 256), (5, 500), (3, 2047), (3, 4000), (2, 8192), (300, 4000),
                                    (270, 8192), (2, 16000), (2, 32768), (2, 70001)])
def test_norm_results_below_f32s_normal_numbers(rows, K, dtype):
    """Every y lies next to a tie of bf16's (and at one element of the 8-bit rows') smallest numbers, off
    it by less than the last place that f32 has there, and is rounded once all the same.

    h is 1 but for one element 2^-20 smaller, so that 1 / sqrt(mean(h^2)) is 1 + 2^-20 / K, 2^-28 to 2^-36
    above 1 and off by some 2^-52; y is that times the weight, which is half a step of the type."""
    x, r = np.ones((rows, K)), np.zeros((rows, K))
    r[:, 3] = -2.0 ** -20
    (x, xv), (r, rv) = ref.typed(x, dtype), ref.typed(r, dtype)
    w = np.ones(K)
    w[:128] = (2 * np.arange(128) + 1) * 2.0 ** -134  # between bf16's multiples of 2^-133
    w[128:256] = 2.0 ** -127  # half of the 8-bit rows' smallest number
    w[128:256:2] *= -1
    out = gpu.norm_dev(x, r, np.float32(w), 0.0, dtype)
    _, y = ref.norm(xv, rv, w, 0.0)
    assert (np.abs(y[:, 4:256]) > np.abs(w[4:256])).all()
    for got, want in zip(out["c"], ref.pack(y)):
        np.testing.assert_array_equal(got, want)
    assert (out["c"][0][:, 128:256] & 127 == 1).all()  # the smallest number, not zero
    # Multiples of the smallest number of either type, ties to even (there are none).
    unit = 2.0 ** (-149 if dtype == ref.F32 else -133)
    np.testing.assert_array_equal(ref.untyped(out["y"], dtype)[:, :256],
                                  np.rint(y[:, :256] / unit) * unit)


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("M,N,K", [(3, 20, 1024), (40, 200, 4096), (300, 260, 2048),
                                   (600, 512, 1024)])
def test_products_whose_large_terms_cancel(M, N, K, dtype):
    """Two elements of each row 2^13 times the others, their products equal but for the sign, and in
    different eights: C in f32 keeps the sum of the small ones to f32's steps of the large ones; C in
    bf16 may lose 7 * 2^-13 of the largest product of each eight, no more."""
    rng = np.random.default_rng(M)
    a, w = rng.standard_normal((M, K)), rng.standard_normal((N, K))
    big = 2.0 ** 13
    a[:, 5], a[:, K - 3] = big, big
    w[:, 5], w[:, K - 3] = 1.5, -1.5
    a, w = (ref.pack(np.float32(x).astype(np.float64)) for x in (a, w))
    gpu.check_linear(gpu.linear_dev(a, w, K, dtype), a, w, K, dtype)
