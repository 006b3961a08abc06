"""MX4Linear and KV4Cache as a program uses them: sequences taken back, calls from several threads."""
import numpy as np
import pytest

import mx4_ref as ref
from anima_hip import KV4Cache, MX4Linear, mx4, rt
from test_mx4_classes_cpu import in_threads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("kind", [np.int32, np.int64, list])
def test_sequences_taken_back(kind):
    """Tokens appended, taken back and appended anew give what the last ones alone give, bit for bit."""
    rng = np.random.default_rng(1)
    k, v = (np.float32(rng.standard_normal((3, 60, 2, 64))) for _ in range(2))
    q = np.float32(rng.standard_normal((3, 2, 4, 64)))
    once, again = KV4Cache(3, 2, 64, 80), KV4Cache(3, 2, 64, 80)
    once.append(k[:, :40], v[:, :40], counts=[40, 7, 21])
    again.append(k[:, :50], v[:, :50], counts=[50, 9, 50])
    # Sequence 2 goes back to 15 tokens and takes 6 others, its own 15th to 20th.
    again.lens = [40, 7, 15] if kind is list else np.array([40, 7, 15], kind)
    again.append(k[:, 15:21], v[:, 15:21], counts=[0, 0, 6])
    assert list(again.lens) == [40, 7, 21]
    np.testing.assert_array_equal(again.attend(q), once.attend(q))


def test_threads_share_objects():
    """One layer and one cache under six threads: each call's result is the one it has alone."""
    rng = np.random.default_rng(2)
    lin = MX4Linear(np.float32(rng.standard_normal((256, 512)) * 0.05))
    xs = [np.float32(rng.standard_normal((3 + 17 * i, 512))) for i in range(6)]
    cache = KV4Cache(1, 2, 64, 300)
    kv = np.float32(rng.standard_normal((1, 300, 2, 64)))
    cache.append(kv, kv[:, ::-1])
    qs = [np.float32(rng.standard_normal((1 + i, 1 + 30 * i, 4, 64))) for i in range(6)]
    want = [(lin(x), cache.attend(q)) for x, q in zip(xs, qs)]
    for _ in range(3):
        got = in_threads(6, lambda i: (lin(xs[i]), cache.attend(qs[i])))
        for (y, o), (wy, wo) in zip(got, want):
            np.testing.assert_array_equal(y, wy)
            np.testing.assert_array_equal(o, wo)
    codes, scales = mx4.pack(kv.reshape(-1, 64))
    np.testing.assert_array_equal(cache.values()[0][0].transpose(1, 0, 2).reshape(-1, 64),
                                  ref.unpack(codes, scales, 64))
