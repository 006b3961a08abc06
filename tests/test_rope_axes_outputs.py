"""The rotation's outputs whose rows share elements are refused, before any device work: threads would
write different results to one place.  Rows that only lie between one another's are taken."""
import itertools

import numpy as np
import pytest

import fp8_ref as ref
from anima_hip import _lib

P = 4096  # a 16-byte aligned address that is never read


def taken(B, H, S, D, strides, which="q"):
    """Whether outputs of these strides pass: the call's input is the output's array at other
    strides, which is refused next, so that none gets as far as the device."""
    moved = (strides[0], strides[1] + 1, strides[2])
    q, k = ((moved, strides), (None, None)) if which == "q" else ((None, None), (moved, strides))
    heads = (H, 2) if which == "q" else (2, H)
    assert H > 1
    assert not _lib.load().anima_hip_rope_axes_dev(
        P, _lib.strides(q[0]), P, _lib.strides(q[1]), heads[0], 64 * P, _lib.strides(k[0]), 64 * P,
        _lib.strides(k[1]), heads[1], P, 0, None, P, None, 1, 1, B, S, D, ref.F32, False, False, None)
    error = _lib.last_error()
    assert ("rows of an output overlap" in error) != ("must have its input's strides" in error), error
    return "overlap" not in error


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("B,H,S,strides", [
    (2, 4, 5, (1280, 64, 64)),     # head 1 of token 0 is head 0 of token 1
    (2, 4, 5, (320, 320, 64)),     # batch entries are heads
    (2, 4, 5, (64, 640, 64)),
    (1, 4, 5, (0, 128, 192)),      # 3 heads on is 2 tokens on
    (3, 2, 5, (300, 4096, 64)),    # a sequence ends inside the next
    (2, 4, 5, (1280, -64, 64)),
    (2, 4, 5, (1280, 320, -63)),
    (2, 2, 2, (127, 64, 4096)),    # by one element
])
def test_shared_rows(which, B, H, S, strides):
    assert not taken(B, H, S, 64, strides, which)


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("B,H,S,strides", [
    (2, 4, 5, (1280, 320, 64)), (2, 4, 5, (1280, 64, 256)), (2, 4, 5, (64, 640, 128)),
    (2, 4, 5, (-1280, 64, -256)), (2, 4, 5, (3840, 192, 768)),
    (1, 2, 3, (0, 192, 128)),      # 0, 128, 256 and 192, 320, 448
    (3, 2, 1, (128, 64, 0)), (1, 2, 1, (0, 64, 0)),
    (2, 2, 2, (2 ** 62, 2 ** 61, 64)),
    (2000, 2048, 4001, (64 * 2048, 64, 2 ** 40)),
])
def test_rows_apart(which, B, H, S, strides):
    assert taken(B, H, S, 64, strides, which)


def test_interleaved_axes_past_any_memory():
    """Refused at once: nothing goes through 2^31 steps on the host."""
    assert not taken(2 ** 30, 2, 2 ** 30, 64, (2 ** 40, 2 ** 36 + 64, 128))
    assert taken(2, 2, 2 ** 20, 64, (2 ** 40, 2 ** 26 + 64, 128))


def test_against_every_row():
    rng = np.random.default_rng(0)
    seen = [0, 0]
    for _ in range(4000):
        B, H, S = (int(n) for n in rng.integers(1, 6, 3))
        H += H == 1
        D = int(rng.integers(2, 5))
        strides = [int(x) * (1 if rng.random() < 0.8 else -1) for x in rng.integers(D, 12 * D, 3)]
        starts = sorted(b * strides[0] + h * strides[1] + s * strides[2]
                        for b, h, s in itertools.product(range(B), range(H), range(S)))
        apart = all(y - x >= D for x, y in zip(starts, starts[1:]))
        assert taken(B, H, S, D, strides) == apart, (B, H, S, D, strides)
        seen[apart] += 1
    assert min(seen) > 400
