"""The 4-bit row format, its linear layer and its attention in numpy, 64 bits."""
import numpy as np

F32, BF16 = 0, 2  # dtype codes of include/anima_hip.h
STEPS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# Half a step of a rounding, relative to the value.
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


def bits_of(x):
    """bf16 bit patterns of float32 values (round to nearest even)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def values_of(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def typed(x, dtype):
    """(array to upload, its values in float64)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == F32:
        return x, x.astype(np.float64)
    b = bits_of(x)
    return b, values_of(b).astype(np.float64)


def untyped(raw, dtype):
    return (raw if dtype == F32 else values_of(raw)).astype(np.float64)


def pack(x):
    """(codes, scales) of the rows of x (float64 holding float32 values)."""
    rows, K = x.shape
    G = -(-K // 32)
    g = np.zeros((rows, G * 32))
    g[:, :K] = x
    g = g.reshape(rows, G, 32)
    top = np.abs(g).max(-1)
    finite = np.isfinite(top)
    e = np.full(top.shape, -200.0)
    pos = finite & (top > 0)
    e[pos] = np.floor(np.log2(top[pos]))  # corrected below where log2 rounded across an integer
    e[pos] += (np.exp2(e[pos] + 1) <= top[pos]).astype(float) - (np.exp2(e[pos]) > top[pos])
    e[pos] += top[pos] > 1.75 * np.exp2(e[pos])
    byte = np.where(finite, np.clip(e - 2 + 127, 2, 252), 255).astype(np.int64)
    unit = np.exp2(np.where(finite, byte, 127) - 127.0)[..., None]
    mag = np.abs(np.where(finite[..., None], g, 0.0)) / unit
    code = np.zeros(g.shape, np.int64)
    for i in range(1, 8):
        edge = (STEPS[i - 1] + STEPS[i]) / 2
        code += (mag > edge) | ((mag == edge) & (i % 2 == 0))
    code += 8 * (np.signbit(g) & finite[..., None])
    code = code.reshape(rows, G * 16, 2)
    return (code[..., 0] + 16 * code[..., 1]).astype(np.uint8), byte.astype(np.uint8)


def unpack(codes, scales, K):
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = STEPS[nib & 7] * np.where(nib & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return (v * np.repeat(s, 32, -1))[..., :K]


def attention(q, k, v, lens, counts, causal, scale):
    """q [B,S,H,D], k/v [Bk,H_kv,S_max,D], all float64: (out, bound on |out|'s summands): rows
    past counts and rows that see no key are zeros.  The second result is sum_j p_j |v_j|."""
    B, S, H, D = q.shape
    Bk, H_kv = k.shape[:2]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        bk = 0 if Bk == 1 else b
        n = min(max(lens[bk], 0), k.shape[2])
        nq = S if counts is None else min(max(counts[b], 0), S)
        for s in range(nq):
            m = min(max(n - nq + s + 1, 0), n) if causal else n
            if m == 0:
                continue
            for h in range(H):
                hk = h // (H // H_kv)
                w = k[bk, hk, :m] @ q[b, s, h] * scale
                w = np.exp(w - w.max())
                w /= w.sum()
                # A key's NaN group reaches the rows that see the key, and no other.
                out[b, s, h] = w @ v[bk, hk, :m]
                mag[b, s, h] = w @ np.abs(v[bk, hk, :m])
    return out, mag


def attention_rows(q, k, v, lens, counts, causal, scale):
    """attention() with all queries of a head at once, for many of them."""
    B, S, H, D = q.shape
    Bk, H_kv = k.shape[:2]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        bk = 0 if Bk == 1 else b
        n = min(max(lens[bk], 0), k.shape[2])
        nq = S if counts is None else min(max(counts[b], 0), S)
        if n == 0 or nq == 0:
            continue
        limit = np.clip(n - nq + np.arange(nq) + 1, 0, n) if causal else np.full(nq, n)
        seen = np.arange(n) < limit[:, None]
        for h in range(H):
            hk = h // (H // H_kv)
            kk, vv = k[bk, hk, :n], v[bk, hk, :n]
            w = np.where(seen, q[b, :nq, h] @ kk.T * scale, -np.inf)
            top = np.where(limit[:, None] > 0, w.max(-1, keepdims=True), 0.0)
            w = np.where(seen, np.exp(w - top), 0.0)
            w /= np.maximum(w.sum(-1, keepdims=True), 1e-300)
            bad = np.isnan(vv)
            vv = np.where(bad, 0.0, vv)
            # A NaN value reaches the rows that see its key, whatever their weight for it.
            nan = (seen.astype(float) @ bad.astype(float)) > 0
            out[b, :nq, h] = np.where(nan, np.nan, w @ vv)
            mag[b, :nq, h] = w @ np.abs(vv)
    return out, mag
