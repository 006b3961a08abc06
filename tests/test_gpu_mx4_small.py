"""The 4-bit linear layer on f32 activations next to zero: exact from 2^-110 on, and below it as many
bits as three bf16 terms hold, cut off below 2^-133."""
import numpy as np
import pytest

import mx4_ref as ref
import test_gpu_mx4 as mx4
from anima_hip import rt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("M,N,K", [(2, 64, 128), (40, 300, 256), (200, 130, 100), (1, 32800, 96)])
@pytest.mark.parametrize("power", [-100, -109, -110, -120, -128, -140])
def test_small_activations(power, M, N, K):
    """One weight of 2^90 to 2^97 per row, so that no result is small: each is exact, or from an activation
    cut off to a multiple of 2^-133 and no further."""
    rng = np.random.default_rng(-power)
    a = np.float32((1 + rng.random((M, K))) * 2.0 ** power * rng.choice([-1, 1], (M, K)))
    cols, n = rng.integers(0, K, N), np.arange(N)
    w = np.zeros((N, K))
    w[n, cols] = 2.0 ** rng.integers(90, 98, N)
    codes, scales = ref.pack(w)
    got = mx4.linear(a, codes, scales, K, N, ref.F32)
    x = a.astype(float)
    if power < -110:
        x = np.trunc(x * 2.0 ** 133) * 2.0 ** -133
    np.testing.assert_array_equal(got, x[:, cols] * w[n, cols])
