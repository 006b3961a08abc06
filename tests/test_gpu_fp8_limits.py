"""The 8-bit operators and the rotation at their ends: memory past 4 GiB, long sums, many short
sequences, vectors at odd places, streams of their own."""
import ctypes as ct

import numpy as np
import pytest

import fp8_ref as ref
import test_gpu_fp8 as gpu
import test_gpu_rope_axes as ropet
from anima_hip import _lib, rt
from test_mx4_classes_cpu import in_threads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    rt.init()


@pytest.mark.parametrize("M,N,K", [(1, 40000001, 128), (3, 1100001, 4096), (300, 550001, 8192)])
def test_linear_weights_past_4_gib(M, N, K):
    """The first and last weight rows' outputs; the rows between hold whatever the memory does."""
    from devmem import DevBuf
    lib, edge = _lib.load(), 40
    rng = np.random.default_rng(M)
    a = ref.pack(rng.standard_normal((M, K)))
    wc, ws = ref.pack(rng.standard_normal((2 * edge, K)) * 0.02)
    nc, ns = ref.sizes(K)
    w, s = DevBuf(N * nc), DevBuf(N * ns)
    assert w.nbytes > 1 << 32
    for at, rows in ((0, slice(0, edge)), (N - edge, slice(edge, 2 * edge))):
        w.put(wc[rows], at * nc)
        s.put(ws[rows], at * ns)
    d, c = [DevBuf.of(x) for x in a], DevBuf(M * N * 2)
    n = lib.anima_hip_linear_fp8_scratch_bytes(M, N, K, ref.BF16)
    scratch = DevBuf(max(n, 16))
    _lib.check(lib.anima_hip_linear_fp8_dev(d[0].addr, d[1].addr, w.addr, s.addr, c.addr, N, M, N, K,
                                            ref.BF16, scratch.addr, n, None), "linear")
    got = c.get((M, N), np.uint16)
    got = ref.untyped(np.concatenate([got[:, :edge], got[:, -edge:]], 1), ref.BF16)
    gpu.check_linear(got, a, (wc, ws), K, ref.BF16)


@pytest.mark.parametrize("M", [2, 300])
@pytest.mark.parametrize("dtype", gpu.TYPES)
def test_linear_rows_past_4_gib_apart(M, dtype):
    """C's rows 2^25 elements apart: 300 of them span 20 or 40 GB."""
    from devmem import DevBuf
    lib, N, K, ldc = _lib.load(), 70, 384, 1 << 25
    a, w = gpu.linear_inputs(M, N, K, 5)
    size = 4 if dtype == ref.F32 else 2
    d = [DevBuf.of(x) for x in (*a, *w)]
    c = DevBuf(((M - 1) * ldc + N) * size)
    n = lib.anima_hip_linear_fp8_scratch_bytes(M, N, K, dtype)
    scratch = DevBuf(max(n, 16))
    _lib.check(lib.anima_hip_linear_fp8_dev(*(x.addr for x in d), c.addr, ldc, M, N, K, dtype,
                                            scratch.addr, n, None), "linear")
    from devmem import hip
    assert hip().hipDeviceSynchronize() == 0
    got = np.empty((M, N), gpu.np_type(dtype))
    for i in range(M):
        assert hip().hipMemcpy(got[i].ctypes.data, c.addr + i * ldc * size, N * size, 2) == 0
    gpu.check_linear(ref.untyped(got, dtype), a, w, K, dtype)


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("M,N,K", [(2, 3, 300001), (70, 40, 100000), (1, 2, 4194305)])
def test_linear_long_sums(M, N, K, dtype):
    """The last is past what the tiles take."""
    a, w = gpu.linear_inputs(M, N, K, 1)
    gpu.check_linear(gpu.linear_dev(a, w, K, dtype), a, w, K, dtype)


@pytest.mark.parametrize("dtype", gpu.TYPES)
def test_pack_past_4_gib(dtype):
    """Rows 2^20 elements apart, the last of them past 4 GiB, packed, normed and read back."""
    from devmem import DevBuf, hip
    rows, K, ld = 2300, 300, 1 << 20
    size = 4 if dtype == ref.F32 else 2
    raw, x = ref.typed(np.random.default_rng(3).standard_normal((rows, K)), dtype)
    buf = DevBuf(((rows - 1) * ld + K) * size)
    assert buf.nbytes > 1 << 32
    for i in range(rows):
        buf.put(raw[i], i * ld * size)
    lib = _lib.load()
    c, s = (DevBuf(rows * b) for b in ref.sizes(K))
    _lib.check(lib.anima_hip_fp8_pack_dev(buf.addr, ld, dtype, c.addr, s.addr, rows, K, None), "pack")
    got = c.get((rows, 384), np.uint8), s.get((rows, 4), np.uint8)
    for g, want in zip(got, ref.pack(x)):
        np.testing.assert_array_equal(g, want)
    # The norm in place, then the rows' values over them.
    _lib.check(lib.anima_hip_add_rmsnorm_fp8_dev(
        buf.addr, ld, None, 0, None, ct.c_float(1e-6), dtype, None, 0, buf.addr, ld, c.addr, s.addr,
        rows, K, None), "norm")
    packed = c.get((rows, 384), np.uint8), s.get((rows, 4), np.uint8)
    out = np.empty((2, K), gpu.np_type(dtype))
    for j, i in enumerate((0, rows - 1)):
        assert hip().hipMemcpy(out[j].ctypes.data, buf.addr + i * ld * size, K * size, 2) == 0
    gpu.check_norm({"y": out, "c": [p[[0, -1]] for p in packed]}, x[[0, -1]], None, None, 1e-6, dtype)
    _lib.check(lib.anima_hip_fp8_unpack_dev(c.addr, s.addr, buf.addr, ld, dtype, rows, K, None),
               "unpack")
    assert hip().hipDeviceSynchronize() == 0
    assert hip().hipMemcpy(out[1].ctypes.data, buf.addr + (rows - 1) * ld * size, K * size, 2) == 0
    np.testing.assert_array_equal(ref.untyped(out[1], dtype), ref.unpack(*packed, K)[-1])


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("rows,K", [(900, 500), (300, 2047), (150, 4000), (80, 8192), (300, 4000),
                                    (270, 8192), (40, 16000), (20, 32768), (9, 70001)])
def test_norm_rows_are_those_of_the_64_bit_result(rows, K, dtype):
    """Every code and scale, by each of the norm's kernels: y is off by some 2^-50 of itself before
    its only rounding."""
    (x, xv), (r, rv), w = gpu.norm_inputs(rows, K, dtype, K)
    out = gpu.norm_dev(x, r, w, 1e-6, dtype)
    _, y = ref.norm(xv, rv, w.astype(np.float64), float(np.float32(1e-6)))
    for got, want in zip(out["c"], ref.pack(y)):
        np.testing.assert_array_equal(got, want)
    err = np.abs(ref.untyped(out["y"], dtype) - y)
    assert (err <= ref.HALF[dtype] * np.abs(y) * (1 + 2.0 ** -20) + 1e-44).all()


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("B,S,H,D,P", [(2, 5000, (8, 8), 64, 32), (9000, 3, (4, 1), 64, 24),
                                       (1, 70000, (1, 0), 78, 39), (40000, 1, (3, 1), 40, 17)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_workgroups_of_many_tokens(B, S, H, D, P, interleaved, dtype):
    """Large enough that a workgroup takes two rounds of tokens, of several sequences where these
    are short; a count for each."""
    raw, val, pos, freqs, axis = ropet.inputs(B, S, H, D, 3, P, dtype, 4)
    counts = np.random.default_rng(9).integers(0, S + 1, B)
    got = ropet.rope(*raw, pos, freqs, axis, dtype, interleaved, counts=counts)
    for g, x in zip(got, val):
        if x.shape[2]:
            ropet.check(g, x, pos, freqs, axis, dtype, interleaved, False, counts)


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_vectors_at_odd_places(interleaved, dtype):
    """Rows that whole vectors fit but that begin anywhere, and in place."""
    raw, val, pos, freqs, axis = ropet.inputs(2, 37, (3, 2), 64, 3, 24, dtype, 4)
    for in_place in (False, True):
        got = ropet.rope(*raw, pos, freqs, axis, dtype, interleaved, layout=("bsh", 3, 1),
                         in_place=in_place)
        for g, x in zip(got, val):
            ropet.check(g, x, pos, freqs, axis, dtype, interleaved, False)


@pytest.mark.parametrize("dtype", gpu.TYPES)
def test_rope_rows_past_4_gib(dtype):
    from devmem import DevBuf, hip
    B, S, H, D, P, step = 3, 2, 2, 24, 12, 1 << 30
    raw, val, pos, freqs, axis = ropet.inputs(B, S, (H, 0), D, 1, P, dtype, 4)
    size = 4 if dtype == ref.F32 else 2
    buf = DevBuf(((B - 1) * step + S * H * D) * size)
    for b in range(B):
        buf.put(raw[0][b], b * step * size)
    st = _lib.strides((step, D, H * D))
    pd, fd, ad = (DevBuf.of(x) for x in (pos.astype(np.int32), freqs, axis.astype(np.uint8)))
    _lib.check(_lib.load().anima_hip_rope_axes_dev(
        buf.addr, st, buf.addr, st, H, None, None, None, None, 0, pd.addr, S, None, fd.addr, ad.addr,
        1, P, B, S, D, dtype, False, False, None), "rope")
    assert hip().hipDeviceSynchronize() == 0
    got = np.empty((B, S, H, D), gpu.np_type(dtype))
    for b in range(B):
        assert hip().hipMemcpy(got[b].ctypes.data, buf.addr + b * step * size, S * H * D * size, 2) == 0
    ropet.check(got, val[0], pos, freqs, axis, dtype, False, False)


def test_streams_of_their_own():
    """Products on eight streams at once from as many threads, each with scratch of its own."""
    from devmem import DevBuf, hip
    lib, h = _lib.load(), hip()
    sizes = [(24, 512, 8192), (300, 260, 640), (5, 700, 1100), (130, 70, 9000)] * 2
    cases = []
    for i, (M, N, K) in enumerate(sizes):
        a, w = gpu.linear_inputs(M, N, K, i)
        dtype = gpu.TYPES[i % 2]
        st = ct.c_void_p()
        assert h.hipStreamCreate(ct.byref(st)) == 0
        n = lib.anima_hip_linear_fp8_scratch_bytes(M, N, K, dtype)
        cases.append((M, N, K, dtype, a, w, [DevBuf.of(x) for x in (*a, *w)], DevBuf(M * N * 4),
                      DevBuf(max(n, 16)), n, st))
    want = [gpu.linear_dev(c[4], c[5], c[2], c[3]) for c in cases]

    def run(i):
        M, N, K, dtype, _, _, d, c, scratch, n, st = cases[i]
        for _ in range(20):
            _lib.check(lib.anima_hip_linear_fp8_dev(*(x.addr for x in d), c.addr, N, M, N, K, dtype,
                                                    scratch.addr, n, st), "linear")
    assert in_threads(8, run) == [None] * 8
    for c, w in zip(cases, want):
        got = c[7].get((c[0], c[1]), gpu.np_type(c[3]))
        np.testing.assert_array_equal(ref.untyped(got, c[3]), w)
        h.hipStreamDestroy(c[10])
