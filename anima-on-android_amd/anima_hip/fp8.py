"""Linear layers whose weights and activations are 8-bit floating point, on numpy buffers.

FP8 rows are e4m3 elements with one power-of-two scale per 128 of them
(include/anima_hip.h): 8.06 bits per value.  `FP8Linear` keeps a layer's weights so and
packs the activations it is called with, alone or as the result of the norm before the
layer.  Arrays are float32, or uint16 holding bf16 bit patterns; results have the type of
the activations.  An object may be called from several threads; its calls take turns.
"""
from __future__ import annotations

import ctypes as ct

import numpy as np

from . import _lib
from .dit import DTYPE_CODES, DeviceArray
from .mx4 import _Buffers, _one_at_a_time, _typed


def _sizes(rows, K):
    """(bytes of the rows' codes, of their scales)."""
    return rows * (-(-K // 128) * 128), rows * (-(-K // 512) * 4)


def pack(x):
    """(codes, scales) of the rows of x [rows, K]: uint8 [rows, ceil(K/128)*128] and
    [rows, ceil(K/512)*4] (anima_hip_fp8_pack_dev)."""
    x, dtype = _typed(x)
    if x.ndim != 2:
        raise ValueError(f"pack expects [rows, K], got {x.shape}")
    rows, K = x.shape
    nc, ns = _sizes(1, K)
    bufs = _Buffers()
    try:
        xd = bufs.upload("x", x)
        codes, scales = bufs.get("codes", rows * nc), bufs.get("scales", rows * ns)
        _lib.check(_lib.load().anima_hip_fp8_pack_dev(xd.ptr, K, dtype, codes.ptr, scales.ptr, rows,
                                                      K, None), "anima_hip_fp8_pack_dev")
        return codes.download((rows, nc), np.uint8), scales.download((rows, ns), np.uint8)
    finally:
        bufs.close()


def unpack(codes, scales, K):
    """The float32 values [rows, K] of FP8 rows (anima_hip_fp8_unpack_dev)."""
    codes = np.ascontiguousarray(codes, dtype=np.uint8)
    scales = np.ascontiguousarray(scales, dtype=np.uint8)
    rows = codes.shape[0]
    if (codes.size, scales.size) != _sizes(rows, K):
        raise ValueError(f"unpack: codes {codes.shape} and scales {scales.shape} are not rows of {K}")
    bufs = _Buffers()
    try:
        cd, sd = bufs.upload("codes", codes), bufs.upload("scales", scales)
        out = bufs.get("out", rows * K * 4)
        _lib.check(_lib.load().anima_hip_fp8_unpack_dev(cd.ptr, sd.ptr, out.ptr, K, 0, rows, K,
                                                        None), "anima_hip_fp8_unpack_dev")
        return out.download((rows, K))
    finally:
        bufs.close()


def _norm_inputs(bufs, x, dtype, residual, w):
    """Device pointers of residual and w, or None."""
    K, pr, pw = x.shape[-1], None, None
    if residual is not None:
        r, dr = _typed(residual)
        if r.shape != x.shape or dr != dtype:
            raise ValueError(f"residual {r.shape} {r.dtype} for x {x.shape} {x.dtype}")
        pr = bufs.upload("residual", r).ptr
    if w is not None:
        w = np.ascontiguousarray(w, dtype=np.float32)
        if w.shape != (K,):
            raise ValueError(f"norm weights {w.shape} for rows of {K}")
        pw = bufs.upload("norm", w).ptr
    return pr, pw


def add_rmsnorm(x, residual=None, w=None, eps=1e-6):
    """(x + residual, its root-mean-square norm times w), each of x's type and shape [..., K]
    (anima_hip_add_rmsnorm_fp8_dev without its 8-bit result)."""
    x, dtype = _typed(x)
    K = x.shape[-1]
    bufs = _Buffers()
    try:
        xd = bufs.upload("x", x)
        pr, pw = _norm_inputs(bufs, x, dtype, residual, w)
        s, y = bufs.get("sum", x.nbytes), bufs.get("y", x.nbytes)
        _lib.check(_lib.load().anima_hip_add_rmsnorm_fp8_dev(
            xd.ptr, K, pr, K, pw, ct.c_float(eps), dtype, s.ptr, K, y.ptr, K, None, None,
            x.size // K if K else 0, K, None), "anima_hip_add_rmsnorm_fp8_dev")
        return s.download(x.shape, x.dtype), y.download(x.shape, x.dtype)
    finally:
        bufs.close()


class FP8Linear:
    """A linear layer y = x W^T in 8-bit floating point; its weights [out, in] stay on the GPU.

    weight: float32 [N, K], or uint16 bf16 bit patterns; it is packed on the GPU.
    ``FP8Linear.from_store`` packs a matrix of an ``rt.Weights`` store in place."""

    def __init__(self, weight):
        w, dtype = _typed(weight)
        if w.ndim != 2:
            raise ValueError(f"FP8Linear expects a [out, in] matrix, got {w.shape}")
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
        _lib.check(self._lib.anima_hip_fp8_pack_dev(ptr, K, dtype, self._codes.ptr,
                                                    self._scales.ptr, N, K, None),
                   "anima_hip_fp8_pack_dev")
        _lib.check(self._lib.anima_hip_synchronize(), "anima_hip_synchronize")

    def _rows(self, x):
        """(x, dtype, rows, their codes and scales on the device, to be filled)."""
        x, dtype = _typed(x)
        N, K = self.shape
        if x.shape[-1] != K:
            raise ValueError(f"FP8Linear of {self.shape}: x is {x.shape}")
        M = x.size // K if K else int(np.prod(x.shape[:-1]))
        nc, ns = _sizes(M, K)
        return x, dtype, M, self._bufs.get("x_codes", nc), self._bufs.get("x_scales", ns)

    def _product(self, x, dtype, M, codes, scales):
        N, K = self.shape
        out = self._bufs.get("out", M * N * x.itemsize)
        n = self._lib.anima_hip_linear_fp8_scratch_bytes(M, N, K, dtype)
        scratch = self._bufs.get("scratch", n)
        _lib.check(self._lib.anima_hip_linear_fp8_dev(
            codes.ptr, scales.ptr, self._codes.ptr, self._scales.ptr, out.ptr, N, M, N, K, dtype,
            scratch.ptr, n, None), "anima_hip_linear_fp8_dev")
        return out.download(x.shape[:-1] + (N,), x.dtype)

    @_one_at_a_time
    def __call__(self, x):
        """x [..., K] -> [..., N], float32 or bf16 bits like x; x is packed first."""
        x, dtype, M, codes, scales = self._rows(x)
        xd, K = self._bufs.upload("x", x), self.shape[1]
        _lib.check(self._lib.anima_hip_fp8_pack_dev(xd.ptr, K, dtype, codes.ptr, scales.ptr, M, K,
                                                    None), "anima_hip_fp8_pack_dev")
        return self._product(x, dtype, M, codes, scales)

    @_one_at_a_time
    def after_norm(self, x, residual=None, w=None, eps=1e-6):
        """(y, h): h = x + residual and y the layer's product with h's root-mean-square norm times
        w, which goes into 8 bits without another rounding."""
        x, dtype, M, codes, scales = self._rows(x)
        xd, K = self._bufs.upload("x", x), self.shape[1]
        pr, pw = _norm_inputs(self._bufs, x, dtype, residual, w)
        h = self._bufs.get("sum", x.nbytes)
        _lib.check(self._lib.anima_hip_add_rmsnorm_fp8_dev(
            xd.ptr, K, pr, K, pw, ct.c_float(eps), dtype, h.ptr, K, None, K, codes.ptr, scales.ptr,
            M, K, None), "anima_hip_add_rmsnorm_fp8_dev")
        return self._product(x, dtype, M, codes, scales), h.download(x.shape, x.dtype)

    def close(self):
        if getattr(self, "_bufs", None) is not None:
            with self._bufs.lock:
                self._bufs.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


__all__ = ["FP8Linear", "add_rmsnorm", "pack", "unpack"]
