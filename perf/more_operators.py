"""The 8-bit operators and the rotation by several axes: what a program that runs its layers'
products in 8-bit floating point has the library do between two attentions, in the library's calls
and in a plain form.

8-bit rows ("FP8"): every 128 consecutive elements of a row share one scale byte s, standing for
2^(s - 127) (255: the group is NaN); an element is an e4m3 number (OCP: no infinity, largest 448).
A row of K elements has ceil(K / 128) * 128 bytes of codes, zero past K, and ceil(K / 512) * 4
scale bytes, zero past its groups.

Packing: the scale is the smallest power of two by which the largest magnitude a of a group is at
most 448 (2^E <= a < 2^(E+1): byte E - 8 + 127, one more where a > 1.75 * 2^E), kept within bytes
10 .. 246, so that every value is zero or a normal bf16 number; elements round to nearest, ties to
even, and saturate at 448.  A group with an infinity or a NaN gets 255.

Kinds:

  pack    rows of f32 or bf16 into FP8 and back
  norm    x + residual, its root-mean-square norm, the result in FP8 (and in the rows' own type)
  linear  C = A W^T with A and W in FP8, C f32 or bf16
  rope    queries and keys rotated by their tokens' positions on one to four axes, or back
"""
import ctypes as ct
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"f32": 0, "bf16": 2}  # the library's dtype codes
EPS = 1e-6
# (N, K) of the linear layers of the Anima 2B DiT: projections, fused q/k/v, MLP, the context's K/V
# and the AdaLN pair.
LAYERS = [(2048, 2048), (6144, 2048), (8192, 2048), (2048, 8192), (2048, 1024), (256, 2048),
          (6144, 256)]


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A projection's weights packed once at load, from the checkpoint's bf16.
        {"name": "pack_proj_bf16", "kind": "pack", "dtype": "bf16", "rows": 2048, "K": 2048},
        # f32 activations of a width that is no multiple of 128, packed before a product.
        {"name": "pack_ragged_f32", "kind": "pack", "dtype": "f32", "rows": 20011, "K": 1000},
        # The norm before one token's projections: latency.
        {"name": "norm_token_bf16", "kind": "norm", "dtype": "bf16", "rows": 1, "K": 2048,
         "y": False},
        # The norm of a 1024 x 1024 image's tokens, CFG pair.
        {"name": "norm_image_bf16", "kind": "norm", "dtype": "bf16", "rows": 8192, "K": 2048,
         "y": False},
        # A text chunk in f32 of an odd width; the normed rows are kept in f32 too.
        {"name": "norm_chunk_f32", "kind": "norm", "dtype": "f32", "rows": 1001, "K": 5000,
         "y": True},
        # One token through a projection: latency, one pass over 4 MiB of codes.
        {"name": "linear_token_bf16", "kind": "linear", "dtype": "bf16", "M": 1, "N": 2048,
         "K": 2048},
        # A small batch of tokens through the MLP's second layer.
        {"name": "linear_batch_bf16", "kind": "linear", "dtype": "bf16", "M": 24, "N": 2048,
         "K": 8192},
        # A text context of odd length and odd width, f32 out.
        {"name": "linear_context_f32", "kind": "linear", "dtype": "f32", "M": 333, "N": 2048,
         "K": 1000},
        # The MLP's first layer at 768 x 768 pixels, CFG pair: the largest product.
        {"name": "linear_fc1_768px_bf16", "kind": "linear", "dtype": "bf16", "M": 4608, "N": 8192,
         "K": 2048},
        # The next token of 8 running sequences at far positions, grouped heads, one axis.
        {"name": "rope_token_bf16", "kind": "rope", "dtype": "bf16", "B": 8, "S": 1, "H_q": 16,
         "H_k": 4, "D": 128, "pairs": 64, "axes": 1, "interleaved": False, "inverse": False},
        # A 1024 x 1024 image's tokens (time, height, width), CFG pair, f32.
        {"name": "rope_image_f32", "kind": "rope", "dtype": "f32", "B": 2, "S": 4096, "H_q": 16,
         "H_k": 16, "D": 128, "pairs": 64, "axes": 3, "interleaved": False, "inverse": False},
        # A long video, part of each head rotated in neighbouring pairs, rotated back (the
        # gradient's direction).
        {"name": "rope_video_back_bf16", "kind": "rope", "dtype": "bf16", "B": 1, "S": 30003,
         "H_q": 12, "H_k": 2, "D": 64, "pairs": 24, "axes": 3, "interleaved": True,
         "inverse": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pack", "norm", "norm", "linear", "linear", "linear", "rope", "rope"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "pack":
        K = rng.choice([68, 256, 1000, 1024, 2048, 8192, _log_int(rng, 1, 8192)])
        return {"kind": kind, "dtype": dtype, "rows": _log_int(rng, 1, (1 << 24) // K), "K": K}
    if kind == "norm":
        K = rng.choice([256, 1024, 2048, 8192, _log_int(rng, 1, 16384)])
        most = max(2, (1 << 23) // K)
        return {"kind": kind, "dtype": dtype, "K": K, "y": rng.random() < 0.3,
                "rows": _log_int(rng, 1, min(most, 32768))}
    if kind == "linear":
        N, K = rng.choice(LAYERS)
        if rng.random() < 0.3:
            N, K = _log_int(rng, 1, 8192), _log_int(rng, 1, 2048)
        return {"kind": kind, "dtype": dtype, "N": N, "K": K,
                "M": _log_int(rng, 1, 4608 if dtype == "bf16" else 2048)}
    D = rng.choice([64, 128, 128, 2 * rng.randint(20, 128)])
    H_q, H_k = rng.choice([(16, 16), (16, 4), (16, 8), (8, 1), (12, 2), (20, 1), (5, 0)])
    B = rng.choice([1, 2, 3, 8])
    most = max(2, (1 << 24) // (B * (H_q + H_k) * D))
    return {"kind": kind, "dtype": dtype, "B": B, "S": _log_int(rng, 1, most), "H_q": H_q,
            "H_k": H_k, "D": D, "pairs": D // 2 if rng.random() < 0.6 else rng.randint(1, D // 2),
            "axes": rng.choice([1, 3, 3, 2, 4]), "interleaved": rng.random() < 0.4,
            "inverse": rng.random() < 0.3}


def _groups(K):
    return -(-K // 128)


def _scale_bytes(K):
    return -(-K // 512) * 4


# ---------------------------------------------------------------- the inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 41)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV) * std


def _rows(g, n, K, std):
    """Rows of different size, as weights and activations are."""
    return _randn(g, n, K, std=std) * torch.exp(0.5 * _randn(g, n, 1))


def _frequencies(case):
    """Angles per position of each pair, and each pair's axis: the pairs are shared out over the
    axes in blocks, each with frequencies of its own from 1 down."""
    P, A = case["pairs"], case["axes"]
    axis = [p * A // P for p in range(P)]
    size = [axis.count(a) for a in range(A)]
    freq = [1e4 ** (-(p - axis.index(axis[p])) / size[axis[p]]) for p in range(P)]
    return (torch.tensor(freq, dtype=torch.float64, device=DEV),
            torch.tensor(axis, dtype=torch.uint8, device=DEV))


def _inputs(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "pack":
        return {"x": _rows(g, case["rows"], case["K"], 0.02).to(dt)}
    if kind == "norm":
        n, K = case["rows"], case["K"]
        # The stream between layers has a few channels far larger than the rest.
        r = _rows(g, n, K, 4.0) * torch.exp(2.0 * _randn(g, K).clamp(min=1.0) - 2.0)
        return {"x": _rows(g, n, K, 1.0).to(dt), "r": r.to(dt), "w": 1.0 + _randn(g, K, std=0.2)}
    if kind == "linear":
        K = case["K"]
        x = dict(zip(("ac", "as"), plain_pack(_rows(g, case["M"], K, 1.0))))
        x.update(zip(("wc", "ws"), plain_pack(_rows(g, case["N"], K, 0.02))))
        return x
    B, S, A = case["B"], case["S"], case["axes"]
    x = {n: _randn(g, B, S, case["H_" + n], case["D"]).to(dt) for n in "qk"}
    # Sequences at different places: text far along on one axis, else cells of a grid in order.
    start = torch.randint(0, 1 << 20, (B, 1, 1), generator=g, device=DEV)
    at = torch.arange(S, device=DEV)[None, :, None].expand(B, S, A)
    if A == 1:
        at = at + start
    else:
        edge = max(1, math.isqrt(S))
        size = torch.tensor([edge ** a for a in reversed(range(A))], device=DEV)
        at = at // size % torch.tensor([1 << 30] + [edge] * (A - 1), device=DEV) + start % 100
    x["positions"] = at.to(torch.int32).contiguous()
    x["freqs"], x["axis"] = _frequencies(case)
    return x


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case, lib=None)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if own:
        pkg = os.path.join(os.getcwd(), "anima-on-android_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from anima_hip import _lib
        s["lib"], s["check"], s["strides"] = _lib.load(), _lib.check, _lib.strides
    if kind in ("pack", "norm"):
        n, K = case["rows"], case["K"]
        s["codes"] = torch.zeros(n, _groups(K) * 128, dtype=torch.uint8, device=DEV)
        s["scales"] = torch.zeros(n, _scale_bytes(K), dtype=torch.uint8, device=DEV)
        # Values of 8-bit rows are bf16 numbers.
        s["out"] = torch.zeros(n, K, dtype=dt if kind == "pack" else torch.bfloat16, device=DEV)
    if kind == "norm":
        s["sum"] = torch.zeros_like(s["x"])
        s["y"] = torch.zeros_like(s["x"]) if case["y"] else None
    if kind == "linear":
        s["out"] = torch.zeros(case["M"], case["N"], dtype=dt, device=DEV)
        s["nbytes"] = 0
        if own:
            s["nbytes"] = s["lib"].anima_hip_linear_fp8_scratch_bytes(case["M"], case["N"],
                                                                      case["K"], CODES[case["dtype"]])
        s["scratch"] = torch.empty(max(s["nbytes"], 16), dtype=torch.uint8, device=DEV)
    if kind == "rope":
        s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c, lib, check = s["case"], s["lib"], s["check"]
    kind, dtype = c["kind"], CODES[c["dtype"]]
    stream = ct.c_void_p(torch.cuda.current_stream().cuda_stream)

    def p(n):
        return s[n].data_ptr()

    if kind == "pack":
        n, K = c["rows"], c["K"]
        check(lib.anima_hip_fp8_pack_dev(p("x"), K, dtype, p("codes"), p("scales"), n, K, stream),
              "fp8_pack_dev")
        check(lib.anima_hip_fp8_unpack_dev(p("codes"), p("scales"), p("out"), K, dtype, n, K,
                                           stream), "fp8_unpack_dev")
        return s["out"]
    if kind == "norm":
        n, K = c["rows"], c["K"]
        check(lib.anima_hip_add_rmsnorm_fp8_dev(
            p("x"), K, p("r"), K, p("w"), EPS, dtype, p("sum"), K, p("y") if c["y"] else None, K,
            p("codes"), p("scales"), n, K, stream), "add_rmsnorm_fp8_dev")
        check(lib.anima_hip_fp8_unpack_dev(p("codes"), p("scales"), p("out"), K, CODES["bf16"], n,
                                           K, stream), "fp8_unpack_dev")
        return {"sum": s["sum"], "values": s["out"], "y": s["y"]}
    if kind == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        check(lib.anima_hip_linear_fp8_dev(
            p("ac"), p("as"), p("wc"), p("ws"), p("out"), N, M, N, K, dtype, p("scratch"),
            s["nbytes"], stream), "linear_fp8_dev")
        return s["out"]
    B, S, D, A = c["B"], c["S"], c["D"], c["axes"]

    def rows(H):  # [B, S, H, D] as {batch, head, token}
        return s["strides"]((S * H * D, D, H * D))

    q, k = rows(c["H_q"]), rows(c["H_k"])
    check(lib.anima_hip_rope_axes_dev(
        p("q"), q, p("q_out"), q, c["H_q"], p("k"), k, p("k_out"), k, c["H_k"], p("positions"),
        S * A, None, p("freqs"), p("axis"), A, c["pairs"], B, S, D, dtype, c["interleaved"],
        c["inverse"], stream), "rope_axes_dev")
    return s["q_out"], s["k_out"]


def _power(byte):
    """2^(byte - 127) in f32, bytes 1 .. 254 (torch's own powers of two are not exact)."""
    return (byte.int() << 23).view(torch.float32)


def plain_pack(x):
    """FP8 codes and scale bytes of the rows of x, by the exponents of their values."""
    rows, K = x.shape
    groups = _groups(K)
    x = torch.nn.functional.pad(x.float(), (0, groups * 128 - K)).reshape(rows, groups, 128)
    a = x.abs().amax(-1)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1)
    byte = torch.where(a > 0, e + 118 + (m > 0.875).int(), 10).clamp(10, 246)
    finite = torch.isfinite(a)
    byte = torch.where(finite, byte, 255)
    y = torch.where(finite[..., None], x * _power(254 - byte.clamp(max=246))[..., None], 0.0)
    # The last place of an e4m3 number is 2^-3 of its power of two, 2^-9 at least.
    _, e = torch.frexp(y)
    e = (e - 1).clamp(min=-6)
    steps = torch.round(y.abs() * _power(130 - e)).int()  # ties to even
    up = steps >> 4  # rounded up to the next power of two
    steps, e = torch.where(up > 0, 8, steps), e + up
    code = torch.where(steps >= 8, (e + 7) * 8 + steps - 8, steps).clamp(max=126)
    code = code + 128 * torch.signbit(y).int()
    scales = torch.nn.functional.pad(byte, (0, _scale_bytes(K) - groups))
    return code.reshape(rows, -1).to(torch.uint8), scales.to(torch.uint8)


def plain_unpack(codes, scales, K):
    """f32 values [rows, K] of FP8 rows."""
    c = codes.int()
    e, f = c >> 3 & 15, (c & 7).float()
    v = torch.where(e > 0, (8.0 + f) * _power(e + 117), f * 2.0 ** -9)
    v = torch.where(c > 127, -v, v).unflatten(-1, (-1, 128))
    s = scales[:, :v.shape[1]]
    s = torch.where(s == 255, float("nan"), _power(s))
    return (v * s[..., None]).flatten(-2)[:, :K]


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "pack":
        return plain_unpack(*plain_pack(s["x"]), c["K"]).to(s["x"].dtype)
    if kind == "norm":
        h = s["x"].float() + s["r"].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"]
        return {"sum": h.to(s["x"].dtype), "y": y.to(s["x"].dtype) if c["y"] else None,
                "values": plain_unpack(*plain_pack(y), c["K"]).to(torch.bfloat16)}
    if kind == "linear":
        a, w = plain_unpack(s["ac"], s["as"], c["K"]), plain_unpack(s["wc"], s["ws"], c["K"])
        return (a @ w.t()).to(s["out"].dtype)
    # Angles in 64 bits: 32 hold none at far positions.
    angle = s["positions"].double()[..., s["axis"].long()] * s["freqs"]
    cos, sin = (f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    return tuple(_plain_rotate(s[n].float(), cos, -sin if c["inverse"] else sin, c).to(s[n].dtype)
                 for n in "qk")


def _plain_rotate(x, cos, sin, c):
    P = c["pairs"]
    r, rest = x[..., :2 * P], x[..., 2 * P:]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else (r[..., :P], r[..., P:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([r, rest], -1)


# ------------------------------------------------------------------- the work

def _fp8_bytes(rows, K):
    return float(rows) * (K + _groups(K))


def work(case):
    kind, size = case["kind"], 4.0 if case["dtype"] == "f32" else 2.0
    if kind == "pack":  # packed, and read back
        n = float(case["rows"]) * case["K"]
        return {"bytes": 2 * size * n + _fp8_bytes(case["rows"], case["K"]), "flops": 4.0 * n}
    if kind == "norm":  # the values in bf16 read back
        n = float(case["rows"]) * case["K"]
        return {"bytes": (size * (4 if case["y"] else 3) + 2) * n +
                _fp8_bytes(case["rows"], case["K"]) + 4.0 * case["K"], "flops": 9.0 * n}
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": size * M * N + _fp8_bytes(M, K) + _fp8_bytes(N, K),
                "flops": 2.0 * M * N * K}
    tokens, heads = float(case["B"]) * case["S"], case["H_q"] + case["H_k"]
    return {"bytes": 2 * size * tokens * heads * case["D"] + 4.0 * tokens * case["axes"],
            "flops": tokens * case["pairs"] * (6.0 * heads + 2)}


# ------------------------------------------------- the definition, in 64 bits

def _exact_rounded(x):
    """x as FP8 holds it: each group over its scale to the nearest e4m3 number, the even code on
    ties."""
    rows, K = x.shape
    pad = -K % 128
    g = torch.cat([x.double(), x.new_zeros(rows, pad).double()], 1).view(rows, -1, 128)
    top = g.abs().max(-1, keepdim=True).values
    power = torch.tensor([2.0 ** (k - 127) for k in range(256)], dtype=torch.float64, device=DEV)
    # The first power of two by which `top` is at most 448.
    unit = power[torch.searchsorted(448.0 * power, top).clamp(10, 246)]
    number = torch.tensor([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10)
                           for c in range(127)], dtype=torch.float64, device=DEV)
    mag = g.abs() / unit
    hi = torch.searchsorted(number, mag).clamp(max=126)  # number[hi - 1] < mag <= number[hi]
    lo = (hi - 1).clamp(min=0)
    below, above = mag - number[lo], number[hi] - mag
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (torch.sign(g) * number[code] * unit).view(rows, -1)[:, :K]


def _exact_values(codes, scales, K):
    c = codes.long()
    mag = torch.where(c % 128 < 8, c % 8 * 2.0 ** -9,
                      (8 + c % 8).double() * torch.exp2((c % 128 // 8 - 10).double()))
    s = torch.exp2(scales.double() - 127).repeat_interleave(128, -1)[:, :codes.shape[1]]
    return (torch.where(c >= 128, -mag, mag) * s)[:, :K]


def exact(case, seed):
    kind = case["kind"]
    x = _inputs(case, seed)
    if kind == "pack":
        return _exact_rounded(x["x"])
    if kind == "norm":
        h = x["x"].double() + x["r"].double()
        y = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / case["K"] + EPS) * x["w"].double()
        return {"sum": h, "values": _exact_rounded(y), "y": y if case["y"] else None}
    if kind == "linear":
        a = _exact_values(x["ac"], x["as"], case["K"])
        out = torch.empty(case["M"], case["N"], dtype=torch.float64, device=DEV)
        for n in range(0, case["N"], 1024):
            w = _exact_values(x["wc"][n:n + 1024], x["ws"][n:n + 1024], case["K"])
            out[:, n:n + 1024] = a @ w.t()
        return out
    P, out = case["pairs"], []
    theta = torch.stack([x["positions"][..., int(a)].double() * f
                         for a, f in zip(x["axis"].tolist(), x["freqs"])], -1)
    turn = torch.polar(torch.ones_like(theta), -theta if case["inverse"] else theta)[:, :, None]
    for n in "qk":
        y = x[n].double()
        at = torch.arange(P, device=DEV)
        first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + P)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return tuple(out)
