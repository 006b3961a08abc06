"""Rotary positions on several axes, on numpy buffers.

`rotate` turns queries and keys by their tokens' positions (anima_hip_rope_axes_dev): text on one
axis, images and video on three, with no table of angles and positions of any size.  `grid_axes`
holds the DiT's own grid (src/position_embedding.py:100-163) in its terms.
"""
from __future__ import annotations

import numpy as np

from . import _lib
from .mx4 import _Buffers, _typed
from .rope import _split


def grid_axes(H: int, W: int, T: int = 1, head_dim: int = 128):
    """(positions [1, T*H*W, 3], freqs [head_dim/2], pair_axis [head_dim/2]) of a T x H x W token
    grid for `rotate`: the angles of `rope.generate_rope_freqs` in 64 bits, without its table."""
    dim_t, dim_h, spatial_base = _split(head_dim)
    freqs = [base ** -(np.arange(0, dim, 2) / dim)
             for base, dim in ((1e4, dim_t), (spatial_base, dim_h), (spatial_base, dim_h))]
    positions = np.stack(np.meshgrid(np.arange(T), np.arange(H), np.arange(W), indexing="ij"), -1)
    return (positions.reshape(1, -1, 3).astype(np.int32), np.concatenate(freqs),
            np.repeat(np.arange(3, dtype=np.uint8), [len(f) for f in freqs]))


def rotate(q, k, positions, freqs, pair_axis=None, interleaved=False, inverse=False):
    """Queries q [B, S, H_q, D] and keys k [B, S, H_k, D] (or None) turned by their tokens'
    positions, int [B or 1, S, axes]: pair p of each row by positions[..., pair_axis[p]] * freqs[p],
    or back (anima_hip_rope_axes_dev).  float32, or uint16 bf16 bit patterns; pairs past
    len(freqs) stay.  Returns (q, k) turned."""
    q, dtype = _typed(q)
    if q.ndim != 4:
        raise ValueError(f"rotate expects q [B, S, heads, D], got {q.shape}")
    B, S, H_q, D = q.shape
    k, dk = _typed(q[:, :, :0] if k is None else k)
    if k.ndim != 4 or k.shape[:2] != (B, S) or k.shape[3] != D or dk != dtype:
        raise ValueError(f"rotate: k {k.shape} {k.dtype} for q {q.shape} {q.dtype}")
    at = np.asarray(positions)
    if at.ndim != 3 or at.shape[0] not in (1, B) or at.shape[1] != S or at.dtype.kind not in "iu":
        raise ValueError(f"positions must be whole numbers [{B} or 1, {S}, axes], got {at.dtype} "
                         f"{at.shape}")
    if at.size and (at.min() < -2**31 or at.max() >= 2**31):
        raise ValueError("positions must fit 32 bits")
    at = np.ascontiguousarray(at, dtype=np.int32)
    axes = at.shape[2]
    freqs = np.ascontiguousarray(freqs, dtype=np.float64)
    if freqs.ndim != 1:
        raise ValueError(f"freqs must be one number a pair, got {freqs.shape}")
    axis = None
    if pair_axis is not None:
        axis = np.asarray(pair_axis)
        if axis.dtype.kind not in "iub" and axis.size:
            raise ValueError(f"pair_axis must be whole numbers, got {axis.dtype}")
        if axis.shape != freqs.shape or (axis.size and (axis.min() < 0 or axis.max() >= axes)):
            raise ValueError(f"pair_axis must be {len(freqs)} axes below {axes}")
        axis = np.ascontiguousarray(axis, dtype=np.uint8)
    bufs = _Buffers()
    try:
        qd, kd, pd, fd = (bufs.upload(n, a) for n, a in (("q", q), ("k", k), ("at", at),
                                                         ("freqs", freqs)))
        ad = None if axis is None else bufs.upload("axis", axis).ptr
        st = [_lib.strides((S * H * D, D, H * D)) for H in (H_q, k.shape[2])]
        _lib.check(_lib.load().anima_hip_rope_axes_dev(
            qd.ptr, st[0], qd.ptr, st[0], H_q, kd.ptr, st[1], kd.ptr, st[1], k.shape[2], pd.ptr,
            0 if at.shape[0] == 1 else S * axes, None, fd.ptr, ad, axes, len(freqs), B, S, D, dtype,
            bool(interleaved), bool(inverse), None), "anima_hip_rope_axes_dev")
        return qd.download(q.shape, q.dtype), kd.download(k.shape, k.dtype)
    finally:
        bufs.close()


__all__ = ["grid_axes", "rotate"]
