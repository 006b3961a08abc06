"""MX4Linear and KV4Cache without a GPU: what they hand to the library, over device arrays held in host
memory and a library that notes its calls."""
import ctypes as ct
import threading
import time

import numpy as np
import pytest

from anima_hip import _lib, mx4


class HostArray:
    """A dit.DeviceArray in host memory."""

    def __init__(self, nbytes):
        self.nbytes = int(nbytes)
        self.mem = ct.create_string_buffer(max(self.nbytes, 1))
        self.ptr = ct.addressof(self.mem)

    @classmethod
    def of(cls, a):
        d = cls(np.asarray(a).nbytes)
        d.upload(a)
        return d

    def upload(self, a):
        a = np.ascontiguousarray(a)
        assert a.nbytes <= self.nbytes
        ct.memmove(self.ptr, a.ctypes.data, a.nbytes)

    def download(self, shape, dtype=np.float32):
        out = np.empty(shape, dtype)
        assert out.nbytes <= self.nbytes
        ct.memmove(out.ctypes.data, self.ptr, out.nbytes)
        return out

    def close(self):
        self.ptr = None


class Library:
    """Every entry succeeds; the int32 arrays that cache entries get are noted."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        return lambda *args: True

    @staticmethod
    def ints(addr, n):
        return list((ct.c_int32 * n).from_address(addr))

    def anima_hip_kv4_attention_scratch_bytes(self, *args):
        return 0

    def anima_hip_kv4_append_dev(self, *args):
        self.seen.append(("append", self.ints(args[9], args[11])))
        return True

    def anima_hip_kv4_attention_dev(self, *args):
        self.seen.append(("attend", self.ints(args[7], args[12])))
        return True


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    monkeypatch.setattr(mx4, "DeviceArray", HostArray)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    return lib


def step(cache, S=1):
    x = np.zeros((cache.batch, S, cache.heads, cache.head_dim), np.float32)
    cache.append(x, x)
    cache.attend(x)


@pytest.mark.parametrize("kind", [np.int32, np.int64, np.uint8, list])
def test_lens_may_be_set(lib, kind):
    """A cache taken back to fewer tokens: lens of any integer type."""
    cache = mx4.KV4Cache(3, 2, 64, 50)
    step(cache, 9)
    cache.lens = [4, 0, 9] if kind is list else np.array([4, 0, 9], kind)
    step(cache)
    assert lib.seen[2:] == [("append", [4, 0, 9]), ("attend", [5, 1, 10])]
    assert list(cache.lens) == [5, 1, 10]
    cache.lens = np.array([[8, 1], [2, 1], [5, 1]])[:, 0]
    step(cache)
    assert lib.seen[4:] == [("append", [8, 2, 5]), ("attend", [9, 3, 6])]


@pytest.mark.parametrize("lens", [[1, 2], [1, 2, 3, 4], 3, [-1, 0, 0], [0, 51, 0], [1.0, 2.0, 3.0],
                                  [2 ** 32, 0, 0]])
def test_lens_out_of_place_are_refused(lib, lens):
    """Too few (the library reads one of each sequence), too many, past the cache, no integers."""
    cache = mx4.KV4Cache(3, 2, 64, 50)
    x = np.zeros((3, 1, 2, 64), np.float32)
    cache.lens = np.array(lens)
    for call in (lambda: cache.append(x, x), lambda: cache.attend(x)):
        with pytest.raises(ValueError, match="lens"):
            call()
    assert not lib.seen


@pytest.mark.parametrize("args,word", [((1, 2, 80, 8), "head_dim"), ((1, 2, 256, 8), "head_dim"),
                                       ((1, 2, 0, 8), "head_dim"), ((0, 2, 64, 8), "positive"),
                                       ((1, 2, 64, 2 ** 30 + 1), "2\\^30")])
def test_caches_that_no_call_would_take(lib, args, word):
    """Refused when they are made, before memory is taken for them."""
    with pytest.raises(ValueError, match=word):
        mx4.KV4Cache(*args)


def in_threads(n, work):
    """work(i) in n threads at once; what each returned, or raised."""
    got, gate = [None] * n, threading.Barrier(n)

    def run(i):
        gate.wait()
        try:
            got[i] = work(i)
        except Exception as e:
            got[i] = e

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return got


def test_linear_from_several_threads(lib, monkeypatch):
    """A layer's device arrays are one call's at a time: each thread gets its own result, and no
    array is closed while a call holds it.  The library copies x to the output, slowly."""
    def slow_copy(x, ldx, codes, scales, out, *args):
        assert x and out
        time.sleep(0.02)
        ct.memmove(out, x, args[1] * ldx * 4)
        return True

    lib.anima_hip_linear_mx4_scratch_bytes = lambda *args: 0
    lib.anima_hip_linear_mx4_dev = slow_copy
    lin = mx4.MX4Linear(np.zeros((32, 32), np.float32))
    xs = [np.full((i + 1, 32), i, np.float32) for i in range(6)]
    for x, got in zip(xs, in_threads(len(xs), lambda i: lin(xs[i]))):
        np.testing.assert_array_equal(got, x)


def test_cache_from_several_threads(lib, monkeypatch):
    """Appends from several threads each get places of their own; an attention sees the lens that
    go with it."""
    def slow(note):
        def call(*args):
            time.sleep(0.01)
            return note(*args)
        return call

    lib.anima_hip_kv4_append_dev = slow(lib.anima_hip_kv4_append_dev)
    cache = mx4.KV4Cache(2, 1, 64, 50)
    x = np.zeros((2, 3, 1, 64), np.float32)

    def work(i):
        cache.append(x, x)
        cache.attend(x)

    assert in_threads(5, work) == [None] * 5
    assert cache.lens.tolist() == [15, 15]
    starts = [n for what, n in lib.seen if what == "append"]
    assert sorted(starts) == [[3 * i, 3 * i] for i in range(5)]
