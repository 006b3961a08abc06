"""The 8-bit row format, its norm and linear layer, and the rotation by several axes, in numpy, 64
bits."""
import numpy as np

from mx4_ref import BF16, F32, HALF, bits_of, typed, untyped, values_of  # noqa: F401

# The magnitudes of codes 0 .. 126.
NUMBERS = np.array([c * 2.0 ** -9 if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 10)
                    for c in range(127)])


def sizes(K):
    """(bytes of a row's codes, of its scales)."""
    return -(-K // 128) * 128, -(-K // 512) * 4


def scale_bytes(top):
    """Scale byte of groups whose largest magnitudes are `top` (finite)."""
    byte = np.searchsorted(448.0 * np.exp2(np.arange(256.0) - 127), top)  # 448 * 2^(byte - 127) >= top
    return np.clip(byte, 10, 246)


def encode(mag):
    """Codes of magnitudes in units of their scale: to nearest, ties to even, saturating."""
    hi = np.minimum(np.searchsorted(NUMBERS, mag), 126)
    lo = np.maximum(hi - 1, 0)
    below, above = mag - NUMBERS[lo], NUMBERS[hi] - mag
    return np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def pack(x):
    """(codes, scales) of the rows of x (float64 holding float32 values)."""
    rows, K = x.shape
    nc, ns = sizes(K)
    g = np.zeros((rows, nc))
    g[:, :K] = x
    g = g.reshape(rows, -1, 128)
    top = np.abs(g).max(-1)
    finite = np.isfinite(top)
    byte = np.where(finite, scale_bytes(np.where(finite, top, 0.0)), 255)
    g = np.where(finite[..., None], g, 0.0)
    code = encode(np.abs(g) / np.exp2(np.where(finite, byte, 127) - 127.0)[..., None])
    code = code + 128 * (np.signbit(g) & finite[..., None])
    scales = np.zeros((rows, ns), np.uint8)
    scales[:, :nc // 128] = byte
    return code.reshape(rows, nc).astype(np.uint8), scales


def unpack(codes, scales, K):
    c = codes.astype(np.int64)
    v = np.append(NUMBERS, np.nan)[c & 127] * np.where(c & 128, -1.0, 1.0)
    s = scales[:, :codes.shape[1] // 128].astype(np.float64)
    s = np.where(s == 255, np.nan, np.exp2(s - 127.0))
    return (v * np.repeat(s, 128, -1))[:, :K]


def norm(x, r, w, eps):
    """(h, y) in float64."""
    h = x if r is None else x + r
    with np.errstate(invalid="ignore", divide="ignore"):
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return h, y if w is None else y * w


def rotate(x, positions, freqs, axis, interleaved, inverse):
    """x [B, S, H, D], positions [B, S, axes]; freqs and axis [pairs]."""
    P = len(freqs)
    axis = np.minimum(axis, positions.shape[-1] - 1)
    t = positions[..., axis].astype(np.longdouble) * freqs.astype(np.longdouble)
    c, s = (f(t).astype(np.float64)[:, :, None] for f in (np.cos, np.sin))
    s = -s if inverse else s
    y = x.astype(np.float64).copy()
    at = np.arange(P)
    i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + P)
    a, b = x[..., i].astype(np.float64), x[..., j].astype(np.float64)
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y
