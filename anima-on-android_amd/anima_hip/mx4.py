"""Linear weights and key/value caches in 4 bits, on numpy buffers.

MX4 rows are the OCP microscaling format with e2m1 elements and one scale byte
per 32 of them (include/anima_hip.h): 4.25 bits per value.  `MX4Linear` keeps a
layer's weights so and multiplies float32 or bf16 activations by them; `KV4Cache`
keeps keys and values so and attends over them.  Arrays are float32, or uint16
holding bf16 bit patterns; results have the type of the activations.  An object may be
called from several threads; its calls take turns.
"""
from __future__ import annotations

import ctypes as ct
import functools
import math
import threading

import numpy as np

from . import _lib
from .dit import DTYPE_CODES, DeviceArray


def _typed(a):
    """(contiguous array, dtype code): float32, or uint16 as bf16 bit patterns."""
    a = np.asarray(a)
    if a.dtype == np.uint16:
        return np.ascontiguousarray(a), DTYPE_CODES["BF16"]
    return np.ascontiguousarray(a, dtype=np.float32), DTYPE_CODES["F32"]


def _sizes(rows, K):
    groups = -(-K // 32)
    return rows * groups * 16, rows * groups


class _Buffers:
    """Grow-only device buffers by role, one call's at a time (`lock`)."""

    def __init__(self):
        self._bufs = {}
        self.lock = threading.RLock()

    def get(self, role, nbytes):
        b = self._bufs.get(role)
        if b is None or b.nbytes < nbytes:
            if b is not None:
                del self._bufs[role]  # first: the allocation below may fail
                b.close()
            b = self._bufs[role] = DeviceArray(max(int(nbytes), 16))
        return b

    def upload(self, role, a):
        b = self.get(role, a.nbytes)
        b.upload(a)
        return b

    def close(self):
        for b in self._bufs.values():
            b.close()
        self._bufs = {}


def _one_at_a_time(method):
    """The foreign calls release the interpreter's lock: without the object's own another thread
    could refill or close a device array that a call is about to read."""
    @functools.wraps(method)
    def call(self, *args, **kwargs):
        with self._bufs.lock:
            return method(self, *args, **kwargs)
    return call


def pack(x):
    """(codes, scales) of the rows of x [rows, K]: uint8 [rows, ceil(K/32)*16] and
    [rows, ceil(K/32)] (anima_hip_mx4_pack_dev)."""
    x, dtype = _typed(x)
    if x.ndim != 2:
        raise ValueError(f"pack expects [rows, K], got {x.shape}")
    rows, K = x.shape
    nc, ns = _sizes(rows, K)
    bufs = _Buffers()
    try:
        xd, codes, scales = bufs.upload("x", x), bufs.get("codes", nc), bufs.get("scales", ns)
        _lib.check(_lib.load().anima_hip_mx4_pack_dev(xd.ptr, K, dtype, codes.ptr, scales.ptr, rows,
                                                      K, None), "anima_hip_mx4_pack_dev")
        groups = -(-K // 32)
        return (codes.download((rows, groups * 16), np.uint8),
                scales.download((rows, groups), np.uint8))
    finally:
        bufs.close()


def unpack(codes, scales, K):
    """The float32 values [rows, K] of MX4 rows (anima_hip_mx4_unpack_dev)."""
    codes = np.ascontiguousarray(codes, dtype=np.uint8)
    scales = np.ascontiguousarray(scales, dtype=np.uint8)
    rows = codes.shape[0]
    if (codes.size, scales.size) != _sizes(rows, K):
        raise ValueError(f"unpack: codes {codes.shape} and scales {scales.shape} are not rows of {K}")
    bufs = _Buffers()
    try:
        cd, sd = bufs.upload("codes", codes), bufs.upload("scales", scales)
        out = bufs.get("out", rows * K * 4)
        _lib.check(_lib.load().anima_hip_mx4_unpack_dev(cd.ptr, sd.ptr, out.ptr, K, 0, rows, K,
                                                        None), "anima_hip_mx4_unpack_dev")
        return out.download((rows, K))
    finally:
        bufs.close()


class MX4Linear:
    """A linear layer y = x W^T whose weights [out, in] stay on the GPU in 4 bits.

    weight: float32 [N, K], or uint16 bf16 bit patterns; it is packed on the GPU.
    ``MX4Linear.from_store`` packs a matrix of an ``rt.Weights`` store in place."""

    def __init__(self, weight):
        w, dtype = _typed(weight)
        if w.ndim != 2:
            raise ValueError(f"MX4Linear expects a [out, in] matrix, got {w.shape}")
        d = DeviceArray.of(w)
        try:
            self._pack(d.ptr, dtype, *w.shape)
        finally:
            d.close()

    @classmethod
    def from_store(cls, weights, name):
        dt, shape = weights.info(name)
        if dt not in ("F32", "BF16") or len(shape) != 2:
            raise ValueError(f"{name} is {dt} {shape}, expected a F32 or BF16 matrix")
        self = cls.__new__(cls)
        self._pack(weights.device(name), DTYPE_CODES[dt], *shape)
        return self

    def _pack(self, ptr, dtype, N, K):
        self.shape = (int(N), int(K))
        self._lib = _lib.load()
        nc, ns = _sizes(N, K)
        self._bufs = _Buffers()
        self._codes, self._scales = self._bufs.get("codes", nc), self._bufs.get("scales", ns)
        _lib.check(self._lib.anima_hip_mx4_pack_dev(ptr, K, dtype, self._codes.ptr,
                                                    self._scales.ptr, N, K, None),
                   "anima_hip_mx4_pack_dev")
        _lib.check(self._lib.anima_hip_synchronize(), "anima_hip_synchronize")

    @_one_at_a_time
    def __call__(self, x):
        """x [..., K] -> [..., N], float32 or bf16 bits like x."""
        x, dtype = _typed(x)
        N, K = self.shape
        if x.ndim < 1 or x.shape[-1] != K:
            raise ValueError(f"MX4Linear of {self.shape}: x is {x.shape}")
        M = x.size // K if K else int(np.prod(x.shape[:-1]))
        out = self._bufs.get("out", M * N * x.itemsize)
        xd = self._bufs.upload("x", x)
        n = self._lib.anima_hip_linear_mx4_scratch_bytes(M, N, K, dtype)
        scratch = self._bufs.get("scratch", n)
        _lib.check(self._lib.anima_hip_linear_mx4_dev(
            xd.ptr, K, self._codes.ptr, self._scales.ptr, out.ptr, N, M, N, K, dtype, scratch.ptr, n,
            None), "anima_hip_linear_mx4_dev")
        return out.download(x.shape[:-1] + (N,), x.dtype)

    def close(self):
        if getattr(self, "_bufs", None) is not None:
            with self._bufs.lock:
                self._bufs.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KV4Cache:
    """Keys and values of `batch` sequences of up to `max_tokens` tokens, `heads` K/V heads of
    `head_dim` (64 or 128), on the GPU in 4 bits.  ``lens`` holds each sequence's tokens; set to
    fewer, it takes sequences back to their first ones."""

    def __init__(self, batch, heads, head_dim, max_tokens):
        if min(batch, heads, max_tokens) < 1:
            raise ValueError("batch, heads and max_tokens must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if max_tokens > 1 << 30:
            raise ValueError(f"max_tokens must be at most 2^30, got {max_tokens}")
        self._lib = _lib.load()
        self.batch, self.heads = int(batch), int(heads)
        self.head_dim, self.max_tokens = int(head_dim), int(max_tokens)
        self.lens = np.zeros(self.batch, np.int32)
        nc, ns = _sizes(self.batch * self.heads * self.max_tokens, self.head_dim)
        self._bufs = _Buffers()
        self._cache = [self._bufs.get(n, b) for n, b in (("kc", nc), ("ks", ns), ("vc", nc),
                                                         ("vs", ns))]

    def _held(self):
        """lens as the library reads it: int32, one of each sequence."""
        n = np.asarray(self.lens)
        if n.shape != (self.batch,) or n.dtype.kind not in "iu" or (n < 0).any() or \
                (n > self.max_tokens).any():
            raise ValueError(f"lens must be {self.batch} whole numbers between 0 and max_tokens = "
                             f"{self.max_tokens}")
        return n.astype(np.int32)

    def _counts(self, counts, S):
        c = np.full(self.batch, S, np.int32) if counts is None else np.asarray(counts, np.int32)
        if c.shape != (self.batch,) or (c < 0).any() or (c > S).any():
            raise ValueError(f"counts must be {self.batch} numbers between 0 and {S}")
        return np.ascontiguousarray(c)

    @_one_at_a_time
    def append(self, k, v, counts=None):
        """Tokens k, v [batch, S, heads, head_dim] behind each sequence's last; counts: how many
        of the S each sequence takes (all, when None)."""
        (k, dtype), (v, dv) = _typed(k), _typed(v)
        want = (self.batch, k.shape[1] if k.ndim == 4 else -1, self.heads, self.head_dim)
        if k.shape != want or v.shape != want or dtype != dv:
            raise ValueError(f"append: k {k.shape}, v {v.shape} for a cache of {want}")
        S = k.shape[1]
        c, lens = self._counts(counts, S), self._held()
        if (lens.astype(np.int64) + c > self.max_tokens).any():
            raise ValueError(f"append: more than max_tokens = {self.max_tokens} tokens")
        kd, vd = self._bufs.upload("k", k), self._bufs.upload("v", v)
        at, cd = self._bufs.upload("starts", lens), self._bufs.upload("counts", c)
        st = _lib.strides((S * self.heads * self.head_dim, self.head_dim,
                           self.heads * self.head_dim))
        _lib.check(self._lib.anima_hip_kv4_append_dev(
            kd.ptr, vd.ptr, dtype, st, st, *(b.ptr for b in self._cache), at.ptr, cd.ptr, self.batch,
            S, self.heads, self.head_dim, self.max_tokens, None), "anima_hip_kv4_append_dev")
        self.lens = lens + c

    @_one_at_a_time
    def attend(self, q, counts=None, is_causal=True, scale=None):
        """softmax(scale q K^T) V of q [B, S, H, head_dim], H a multiple of the cache's heads and B
        the cache's batch, or any with a cache of one sequence.  Causal: the S queries (counts[b]
        of them, when given) are the last tokens of their sequence.  Rows past counts are zeros."""
        q, dtype = _typed(q)
        if q.ndim != 4 or q.shape[3] != self.head_dim or self.batch not in (1, q.shape[0]):
            raise ValueError(f"attend: q {q.shape} for a cache of batch {self.batch}, head_dim "
                             f"{self.head_dim}")
        B, S, H, D = q.shape
        c = None
        if counts is not None:
            c = np.ascontiguousarray(counts, dtype=np.int32)
            if c.shape != (B,):
                raise ValueError(f"counts must be {B} numbers")
        scale = 1.0 / math.sqrt(D) if scale is None else scale
        qd, ld = self._bufs.upload("q", q), self._bufs.upload("lens", self._held())
        cd = None if c is None else self._bufs.upload("qcounts", c)
        od = self._bufs.upload("o", np.zeros_like(q)) if c is not None else \
            self._bufs.get("o", q.nbytes)
        n = self._lib.anima_hip_kv4_attention_scratch_bytes(B, S, H, self.heads, D, self.max_tokens,
                                                            dtype)
        scratch = self._bufs.get("scratch", n)
        st = _lib.strides((S * H * D, D, H * D))
        _lib.check(self._lib.anima_hip_kv4_attention_dev(
            qd.ptr, dtype, st, *(b.ptr for b in self._cache), ld.ptr, cd.ptr if cd else None, od.ptr,
            st, B, self.batch, S, H, self.heads, D, self.max_tokens, ct.c_float(scale),
            bool(is_causal), scratch.ptr, n, None), "anima_hip_kv4_attention_dev")
        return od.download(q.shape, q.dtype)

    @_one_at_a_time
    def values(self):
        """(keys, values) as float32 [batch, heads, max_tokens, head_dim]; tokens past lens hold
        whatever the memory does."""
        rows = self.batch * self.heads * self.max_tokens
        shape = (self.batch, self.heads, self.max_tokens, self.head_dim)
        out = self._bufs.get("values", rows * self.head_dim * 4)
        res = []
        for codes, scales in (self._cache[:2], self._cache[2:]):
            _lib.check(self._lib.anima_hip_mx4_unpack_dev(codes.ptr, scales.ptr, out.ptr,
                                                          self.head_dim, 0, rows, self.head_dim,
                                                          None), "anima_hip_mx4_unpack_dev")
            res.append(out.download(shape))
        return tuple(res)

    def close(self):
        if getattr(self, "_bufs", None) is not None:
            with self._bufs.lock:
                self._bufs.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


__all__ = ["KV4Cache", "MX4Linear", "pack", "unpack"]
