"""The rows that one call of the 8-bit operators takes, as include/anima_hip.h counts them: narrow rows up
to the last one, and refusals from the next on, before anything is read or written."""
import ctypes as ct

import numpy as np
import pytest

import fp8_ref as ref
import test_gpu_fp8 as gpu
from anima_hip import _lib, rt

pytestmark = pytest.mark.gpu

GROUPS = 2 ** 28 - 16
NORM_ROWS = {1: 67108860, 512: 67108860, 513: 16777215, 8192: 16777215, 8193: 4194303}
EDGE = 64


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


def norm(addr, rows, K, codes, scales, y=None):
    return _lib.load().anima_hip_add_rmsnorm_fp8_dev(
        addr, K, None, 0, None, ct.c_float(1e-6), ref.BF16, None, 0, y, K, codes, scales, rows, K,
        None)


@pytest.mark.parametrize("K", [1, 128, 129, 1000])
def test_packing_refusals(K):
    from devmem import DevBuf
    lib, memory = _lib.load(), DevBuf(4096)
    at = memory.addr
    rows = GROUPS // -(-K // 128) + 1
    for dtype in gpu.TYPES:
        assert not lib.anima_hip_fp8_pack_dev(at, K, dtype, at, at, rows, K, None)
        assert "too many elements" in _lib.last_error()
        assert not lib.anima_hip_fp8_unpack_dev(at, at, at, K, dtype, rows, K, None)
        assert "too many elements" in _lib.last_error()


@pytest.mark.parametrize("K", sorted(NORM_ROWS))
def test_norm_refusals(K):
    from devmem import DevBuf
    memory = DevBuf(4096)
    at = memory.addr
    assert not norm(at, NORM_ROWS[K] + 1, K, at, at)
    assert "too many rows" in _lib.last_error()


def edges(rows):
    """First and last rows' values, bf16 bits, of single elements, and where they go."""
    raw, val = ref.typed(np.random.default_rng(1).standard_normal((2 * EDGE, 1)), ref.BF16)
    return raw, val, ((0, slice(0, EDGE)), (rows - EDGE, slice(EDGE, None)))


def read(buf, at, shape, dtype):
    from devmem import hip
    assert hip().hipDeviceSynchronize() == 0
    out = np.empty(shape, dtype)
    assert hip().hipMemcpy(out.ctypes.data, buf.addr + at, out.nbytes, 2) == 0
    return out


def test_single_elements_packed_up_to_the_last_row():
    """2^28 - 16 rows of one element: 34 GB of codes."""
    from devmem import DevBuf
    lib, rows = _lib.load(), GROUPS
    x, codes, scales = DevBuf(rows * 2), DevBuf(rows * 128), DevBuf(rows * 4)
    raw, val, places = edges(rows)
    for at, part in places:
        x.put(raw[part], at * 2)
    _lib.check(lib.anima_hip_fp8_pack_dev(x.addr, 1, ref.BF16, codes.addr, scales.addr, rows, 1,
                                          None), "pack")
    want = ref.pack(val)
    for at, part in places:
        np.testing.assert_array_equal(read(codes, at * 128, (EDGE, 128), np.uint8), want[0][part])
        np.testing.assert_array_equal(read(scales, at * 4, (EDGE, 4), np.uint8), want[1][part])
    _lib.check(lib.anima_hip_fp8_unpack_dev(codes.addr, scales.addr, x.addr, 1, ref.BF16, rows, 1,
                                            None), "unpack")
    for at, part in places:
        got = ref.untyped(read(x, at * 2, (EDGE, 1), np.uint16), ref.BF16)
        np.testing.assert_array_equal(got, ref.unpack(*(p[part] for p in want), 1))


def test_single_elements_normed_up_to_the_last_row():
    from devmem import DevBuf
    rows = NORM_ROWS[1]
    x, codes, scales, y = DevBuf(rows * 2), DevBuf(rows * 128), DevBuf(rows * 4), DevBuf(rows * 2)
    raw, val, places = edges(rows)
    for at, part in places:
        x.put(raw[part], at * 2)
    _lib.check(norm(x.addr, rows, 1, codes.addr, scales.addr, y.addr), "norm")
    _, want = ref.norm(val, None, None, float(np.float32(1e-6)))
    packed = ref.pack(want)
    for at, part in places:
        np.testing.assert_array_equal(read(codes, at * 128, (EDGE, 128), np.uint8), packed[0][part])
        np.testing.assert_array_equal(read(scales, at * 4, (EDGE, 4), np.uint8), packed[1][part])
        got = ref.untyped(read(y, at * 2, (EDGE, 1), np.uint16), ref.BF16)
        assert (np.abs(got - want[part]) <= ref.HALF[ref.BF16] * np.abs(want[part])).all()
