"""The 4-bit operators: what a program that keeps linear weights and key/value caches in 4 bits has
the library do, in the library's calls and in a plain form.

4-bit rows ("MX4", the OCP microscaling format with e2m1 elements): every 32 consecutive elements
of a row share one scale byte s (e8m0: 2^(s - 127), 255 for NaN); an element is a 4-bit code, sign
in bit 3, magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6 in bits 0 to 2.  Byte i of a row's codes holds
element 2i in its low half and 2i + 1 in its high half; a row of K elements has ceil(K / 32) * 16
bytes of codes (zero past K) and ceil(K / 32) scale bytes.

Packing: with a the largest magnitude of a group, 2^E <= a < 2^(E+1), the scale byte is
E - 2 + 127, one more where a > 1.75 * 2^E, kept within 2 .. 252; elements round to the nearest
magnitude (ties to the even code) and saturate at 6.  A group with an infinity or a NaN gets 255.

Kinds:

  pack    rows of f32 or bf16 into MX4 and back to f32 values
  linear  C = A W^T with MX4 weights W, A and C f32 or bf16
  append  new K/V rows of each sequence into an MX4 cache (read back as values)
  attend  attention over an MX4 cache: one query per sequence or many, grouped heads, causal or not
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
# (N, K) of the linear layers of the Anima 2B DiT: projections, fused q/k/v, MLP, the context's K/V
# and the AdaLN pair.
LAYERS = [(2048, 2048), (6144, 2048), (8192, 2048), (2048, 8192), (2048, 1024), (256, 2048),
          (6144, 256)]


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A projection's weights packed once at load, from the checkpoint's bf16.
        {"name": "pack_proj_bf16", "kind": "pack", "dtype": "bf16", "rows": 2048, "K": 2048},
        # A ragged f32 matrix (the patch embedding's 68 columns, rows of a large table).
        {"name": "pack_ragged_f32", "kind": "pack", "dtype": "f32", "rows": 30001, "K": 68},
        # One token through a projection: latency, one pass over 2 MiB of codes.
        {"name": "linear_token_bf16", "kind": "linear", "dtype": "bf16", "M": 1, "N": 2048,
         "K": 2048},
        # A small batch of tokens through the MLP's second layer.
        {"name": "linear_batch_bf16", "kind": "linear", "dtype": "bf16", "M": 24, "N": 2048,
         "K": 8192},
        # A text context of odd length through the K projection, f32.
        {"name": "linear_context_f32", "kind": "linear", "dtype": "f32", "M": 333, "N": 2048,
         "K": 1024},
        # The MLP's first layer at 768 x 768 pixels, CFG pair: the largest product.
        {"name": "linear_fc1_768px_bf16", "kind": "linear", "dtype": "bf16", "M": 4608, "N": 8192,
         "K": 2048},
        # One new token for each of 8 running sequences.
        {"name": "append_token_bf16", "kind": "append", "dtype": "bf16", "B": 8, "S_new": 1,
         "H_kv": 4, "D": 128, "S_max": 96},
        # Two contexts of up to 512 tokens written at once, ragged, f32 projections.
        {"name": "append_context_f32", "kind": "append", "dtype": "f32", "B": 2, "S_new": 512,
         "H_kv": 16, "D": 128, "S_max": 512},
        # One query over a short cache: launches and latency.
        {"name": "attend_token_short_f32", "kind": "attend", "dtype": "f32", "B": 1, "S_q": 1,
         "H": 16, "H_kv": 16, "D": 128, "S": 200, "causal": True, "shared": False},
        # One query for each of 16 long, ragged sequences, four query heads per K/V head.
        {"name": "attend_token_long_bf16", "kind": "attend", "dtype": "bf16", "B": 16, "S_q": 1,
         "H": 16, "H_kv": 4, "D": 128, "S": 16384, "causal": True, "shared": False},
        # A chunk of a long prompt over what is cached of it, six query heads per K/V head, f32.
        {"name": "attend_chunk_f32", "kind": "attend", "dtype": "f32", "B": 1, "S_q": 300,
         "H": 12, "H_kv": 2, "D": 64, "S": 5001, "causal": True, "shared": False},
        # Cross-attention of a 1024 x 1024 image, CFG pair, over one shared 512-token context.
        {"name": "attend_cross_1024px_bf16", "kind": "attend", "dtype": "bf16", "B": 2,
         "S_q": 4096, "H": 16, "H_kv": 16, "D": 128, "S": 512, "causal": False, "shared": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pack", "linear", "linear", "linear", "append", "attend", "attend",
                       "attend"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "pack":
        K = rng.choice([68, 256, 1000, 1024, 2048, 8192, _log_int(rng, 1, 8192)])
        return {"kind": kind, "dtype": dtype, "rows": _log_int(rng, 1, (1 << 24) // K), "K": K}
    if kind == "linear":
        N, K = rng.choice(LAYERS)
        if rng.random() < 0.3:
            N, K = _log_int(rng, 1, 8192), _log_int(rng, 1, 2048)
        return {"kind": kind, "dtype": dtype, "N": N, "K": K,
                "M": _log_int(rng, 1, 4096 if dtype == "bf16" else 1024)}
    D = rng.choice([64, 128, 128])
    H, H_kv = rng.choice([(16, 16), (16, 4), (16, 8), (8, 1), (12, 2), (24, 1)])
    B = rng.choice([1, 2, 3, 8])
    if kind == "append":
        S_new = rng.choice([1, 1, rng.randint(2, 9), _log_int(rng, 10, 512)])
        return {"kind": kind, "dtype": dtype, "B": B, "S_new": S_new, "H_kv": H_kv, "D": D,
                "S_max": S_new + rng.randint(0, 64)}
    S_q = rng.choice([1, 1, 1, rng.randint(2, 17), _log_int(rng, 18, 2048)])
    most = min(16384, 2 ** 23 // (S_q * B), 2 ** 18 // B)
    S, causal = _log_int(rng, 1, max(2, most)), rng.random() < 0.6
    return {"kind": kind, "dtype": dtype, "B": B, "S_q": S_q, "H": H, "H_kv": H_kv, "D": D,
            "S": max(S, S_q) if causal else S, "causal": causal, "shared": rng.random() < 0.2}


def _lens(case):
    """Cached tokens of each sequence, the queries' own among them where the mask is causal: S, and
    less from one to the next."""
    n = 1 if case["shared"] else case["B"]
    least = case["S_q"] if case["causal"] else 1
    return [max(least, case["S"] - b * case["S"] * 3 // (4 * n)) for b in range(n)]


def _counts(case):
    """New rows of each sequence of an append: S_new, and less from one to the next."""
    B, S = case["B"], case["S_new"]
    return [S - b * S // (4 * B) for b in range(B)]


# ---------------------------------------------------------------- the inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 23)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV) * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _packed_randn(g, lead, rows, K, std):
    """MX4 rows of normal values, [lead, rows, ...]: piece by piece, the f32 values are large."""
    parts = [plain_pack(_randn(g, rows, K, std=std)) for _ in range(lead)]
    return [torch.stack(t).contiguous() for t in zip(*parts)]


def _inputs(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "pack":
        # Rows of different size, as the layers' weights are.
        x = _randn(g, case["rows"], case["K"], std=0.02)
        x = x * torch.exp(0.5 * _randn(g, case["rows"], 1))
        return {"x": x.to(dt)}
    if kind == "linear":
        w = plain_pack(_randn(g, case["N"], case["K"], std=0.02))
        return {"a": _randn(g, case["M"], case["K"]).to(dt), "codes": w[0], "scales": w[1]}
    B, H_kv, D = case["B"], case["H_kv"], case["D"]
    if kind == "append":
        S, S_max = case["S_new"], case["S_max"]
        x = {n: _randn(g, B, S, H_kv, D).to(dt) for n in "kv"}
        for n in "kv":
            x[n + "c"], x[n + "s"] = _packed_randn(g, B, H_kv * S_max, D, 1.0)
        room = [S_max - n for n in _counts(case)]
        x["starts"] = _ints([r - b % (r + 1) for b, r in enumerate(room)])
        x["counts"] = _ints(_counts(case))
        return x
    lens = _lens(case)
    S_max = case["S"] + 7
    x = {"q": _randn(g, B, case["S_q"], case["H"], D).to(dt), "lens": _ints(lens)}
    for n in "kv":
        x[n + "c"], x[n + "s"] = _packed_randn(g, len(lens), H_kv * S_max, D, 1.0)
    return x


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case, lib=None)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if own:
        pkg = os.path.join(os.getcwd(), "anima-on-android_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from anima_hip import _lib
        s["lib"], s["check"] = _lib.load(), _lib.check
        s["strides"] = _lib.strides
    nbytes = 0
    if kind == "pack":
        n, groups = case["rows"], -(-case["K"] // 32)
        s["codes"] = torch.zeros(n, groups * 16, dtype=torch.uint8, device=DEV)
        s["scales"] = torch.zeros(n, groups, dtype=torch.uint8, device=DEV)
        s["out"] = torch.zeros(n, case["K"], device=DEV)
    elif kind == "linear":
        s["out"] = torch.zeros(case["M"], case["N"], dtype=dt, device=DEV)
        if own:
            nbytes = s["lib"].anima_hip_linear_mx4_scratch_bytes(
                case["M"], case["N"], case["K"], CODES[case["dtype"]])
    elif kind == "append":
        shape = (case["B"], case["H_kv"], case["S_max"], case["D"])
        s["k_out"], s["v_out"] = (torch.zeros(shape, device=DEV) for _ in range(2))
    else:
        s["out"] = torch.zeros_like(s["q"])
        if own:
            nbytes = s["lib"].anima_hip_kv4_attention_scratch_bytes(
                case["B"], case["S_q"], case["H"], case["H_kv"], case["D"], case["S"] + 7,
                CODES[case["dtype"]])
    s["nbytes"] = nbytes
    s["scratch"] = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=DEV)
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
        check(lib.anima_hip_mx4_pack_dev(p("x"), K, dtype, p("codes"), p("scales"), n, K, stream),
              "mx4_pack_dev")
        check(lib.anima_hip_mx4_unpack_dev(p("codes"), p("scales"), p("out"), K, 0, n, K, stream),
              "mx4_unpack_dev")
        return s["out"]
    if kind == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        check(lib.anima_hip_linear_mx4_dev(
            p("a"), K, p("codes"), p("scales"), p("out"), N, M, N, K, dtype, p("scratch"),
            s["nbytes"], stream), "linear_mx4_dev")
        return s["out"]
    if kind == "append":
        B, H_kv, D, S_new, S_max = c["B"], c["H_kv"], c["D"], c["S_new"], c["S_max"]
        rows = s["strides"]((S_new * H_kv * D, D, H_kv * D))  # [B, S, H, D] as {batch, head, token}
        check(lib.anima_hip_kv4_append_dev(
            p("k"), p("v"), dtype, rows, rows, p("kc"), p("ks"), p("vc"), p("vs"), p("starts"),
            p("counts"), B, S_new, H_kv, D, S_max, stream), "kv4_append_dev")
        for n in "kv":
            check(lib.anima_hip_mx4_unpack_dev(p(n + "c"), p(n + "s"), p(n + "_out"), D, 0,
                                               B * H_kv * S_max, D, stream), "mx4_unpack_dev")
        return s["k_out"], s["v_out"]
    B, H, H_kv, D, S_q = c["B"], c["H"], c["H_kv"], c["D"], c["S_q"]
    rows = s["strides"]((S_q * H * D, D, H * D))
    check(lib.anima_hip_kv4_attention_dev(
        p("q"), dtype, rows, p("kc"), p("ks"), p("vc"), p("vs"), p("lens"), None, p("out"), rows,
        B, 1 if c["shared"] else B, S_q, H, H_kv, D, c["S"] + 7, ct.c_float(1.0 / math.sqrt(D)),
        c["causal"], p("scratch"), s["nbytes"], stream), "kv4_attention_dev")
    return s["out"]


def _power(byte):
    """2^(byte - 127) in f32, bytes 1 .. 254 (torch's own powers of two are not exact)."""
    return (byte.int() << 23).view(torch.float32)


def plain_pack(x):
    """MX4 codes and scale bytes of the rows of x, by comparisons."""
    rows, K = x.shape
    x = x.float()
    if K % 32:
        x = torch.nn.functional.pad(x, (0, 32 - K % 32))
    x = x.reshape(rows, -1, 32)
    a = x.abs().amax(-1)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1)
    byte = (e + 124 + (m > 0.875).int()).clamp(2, 252)
    finite = torch.isfinite(a)
    byte = torch.where(finite, byte, 255)
    y = x * _power(254 - byte.clamp(max=252))[..., None]
    y = torch.where(finite[..., None], y, 0.0)
    code = torch.signbit(y).to(torch.uint8) * 8
    y = y.abs()
    for edge, tie_up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False),
                         (3.5, True), (5.0, False)):
        code += (y >= edge) if tie_up else (y > edge)
    code = code.reshape(rows, -1, 2)
    return code[..., 0] | (code[..., 1] << 4), byte.to(torch.uint8)


def plain_unpack(codes, scales, K):
    """f32 values [..., K] of MX4 rows."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    s = torch.where(scales == 255, float("nan"), _power(scales))
    v = table[both].unflatten(-1, (-1, 32)) * s[..., None]
    return v.flatten(-2)[..., :K]


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "pack":
        return plain_unpack(*plain_pack(s["x"]), c["K"])
    if kind == "linear":
        w = plain_unpack(s["codes"], s["scales"], c["K"])
        return (s["a"].float() @ w.t()).to(s["a"].dtype)
    if kind == "append":
        out = []
        counts, starts = _counts(c), s["starts"].tolist()
        for n in "kv":
            rows = s[n].transpose(1, 2)  # [B, H_kv, S_new, D]
            codes, scales = plain_pack(rows.reshape(-1, c["D"]))
            lead = (c["B"], c["H_kv"], c["S_new"], -1)
            codes, scales = codes.reshape(lead), scales.reshape(lead)
            cc = s[n + "c"].reshape(c["B"], c["H_kv"], c["S_max"], -1)
            cs = s[n + "s"].reshape(c["B"], c["H_kv"], c["S_max"], -1)
            for b, (at, m) in enumerate(zip(starts, counts)):
                cc[b, :, at:at + m] = codes[b, :, :m]
                cs[b, :, at:at + m] = scales[b, :, :m]
            out.append(plain_unpack(cc, cs, c["D"]))
        return tuple(out)
    B, H, H_kv, D, S_q = c["B"], c["H"], c["H_kv"], c["D"], c["S_q"]
    lens, S_max = _lens(c), c["S"] + 7
    out = torch.zeros_like(s["q"])
    for b in range(B):
        bk = 0 if c["shared"] else b
        n = lens[bk]
        k, v = (plain_unpack(s[x + "c"][bk].reshape(H_kv, S_max, -1)[:, :n],
                             s[x + "s"][bk].reshape(H_kv, S_max, -1)[:, :n], D) for x in "kv")
        q = s["q"][b].float().reshape(S_q, H_kv, H // H_kv, D).permute(1, 2, 0, 3)
        q = q.reshape(H_kv, -1, D).contiguous()
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D)
        if c["causal"]:
            at = torch.arange(n - S_q, n, device=DEV).repeat(H // H_kv)
            score = score.masked_fill(torch.arange(n, device=DEV) > at[:, None], float("-inf"))
        score = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul(score, v) / score.sum(-1, keepdim=True)
        o = o.reshape(H_kv, H // H_kv, S_q, D).permute(2, 0, 1, 3)
        out[b] = o.reshape(S_q, H, D).to(out.dtype)
    return out


# ------------------------------------------------------------------- the work

def _mx4_bytes(rows, K):
    return rows * -(-K // 32) * 17.0


def work(case):
    kind, size = case["kind"], 4.0 if case["dtype"] == "f32" else 2.0
    if kind == "pack":
        n = float(case["rows"]) * case["K"]
        return {"bytes": n * size + _mx4_bytes(case["rows"], case["K"]) + 4.0 * n,
                "flops": 4.0 * n}
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": size * (M * K + M * N) + _mx4_bytes(N, K), "flops": 2.0 * M * N * K}
    H_kv, D = case["H_kv"], case["D"]
    if kind == "append":
        new = 2.0 * sum(_counts(case)) * H_kv
        whole = 2.0 * case["B"] * H_kv * case["S_max"]
        return {"bytes": new * D * size + _mx4_bytes(whole, D) + 4.0 * whole * D,
                "flops": 3.0 * new * D + whole * D}
    H, S_q, B = case["H"], case["S_q"], case["B"]
    lens = _lens(case)
    pairs = 0.0
    for b in range(B):
        n = lens[0 if case["shared"] else b]
        pairs += S_q * n - (S_q * (S_q - 1) / 2 if case["causal"] else 0)
    return {"bytes": 2.0 * size * B * S_q * H * D + 2 * _mx4_bytes(float(sum(lens)) * H_kv, D),
            "flops": 4.0 * pairs * H * D}


# ------------------------------------------------- the definition, in 64 bits

_STEPS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_powers():
    return torch.tensor([2.0 ** (k - 127) for k in range(256)], dtype=torch.float64, device=DEV)


def _exact_rounded(x):
    """x as MX4 holds it: the nearest of the group's eight magnitudes, the even code on ties."""
    rows, K = x.shape
    pad = -K % 32
    g = torch.cat([x.double(), x.new_zeros(rows, pad).double()], 1).view(rows, -1, 32)
    top = g.abs().max(-1, keepdim=True).values
    power = _exact_powers()
    E = torch.searchsorted(power, top, right=True) - 1  # power[E] <= top < power[E + 1]
    E = E.clamp(min=0) + (top > 1.75 * power[E.clamp(min=0)])
    unit = power[(E - 2).clamp(2, 252)]
    mag = g.abs() / unit
    best, dist = torch.zeros_like(mag), mag.clone()
    for code, step in enumerate(_STEPS):
        d = (mag - step).abs()
        take = (d < dist) | ((d == dist) & (code % 2 == 0))
        best, dist = torch.where(take, step, best), torch.where(take, d, dist)
    return (torch.sign(g) * best * unit).view(rows, -1)[:, :K]


def _exact_values(codes, scales, K):
    lead = codes.shape[:-1]
    nib = torch.zeros(*lead, codes.shape[-1] * 2, dtype=torch.long, device=codes.device)
    nib[..., 0::2], nib[..., 1::2] = codes.long() % 16, codes.long() // 16
    steps = torch.tensor(_STEPS, dtype=torch.float64, device=codes.device)
    v = steps[nib % 8] * torch.where(nib >= 8, -1.0, 1.0).double()
    return (v * _exact_powers()[scales.long()].repeat_interleave(32, -1))[..., :K]


def exact(case, seed):
    kind = case["kind"]
    x = _inputs(case, seed)
    if kind == "pack":
        return _exact_rounded(x["x"])
    if kind == "linear":
        out = torch.empty(case["M"], case["N"], dtype=torch.float64, device=DEV)
        for n in range(0, case["N"], 1024):
            w = _exact_values(x["codes"][n:n + 1024], x["scales"][n:n + 1024], case["K"])
            out[:, n:n + 1024] = x["a"].double() @ w.t()
        return out
    D, H_kv = case["D"], case["H_kv"]
    if kind == "append":
        out = []
        for n in "kv":
            shape = (case["B"], H_kv, case["S_max"])
            cache = _exact_values(x[n + "c"], x[n + "s"], D).view(*shape, D)
            for b, (at, m) in enumerate(zip(x["starts"].tolist(), _counts(case))):
                for h in range(H_kv):
                    cache[b, h, at:at + m] = _exact_rounded(x[n][b, :m, h])
            out.append(cache)
        return tuple(out)
    H, S_q, S_max = case["H"], case["S_q"], case["S"] + 7
    out = torch.zeros(case["B"], S_q, H, D, dtype=torch.float64, device=DEV)
    for bk, n in enumerate(_lens(case)):
        for hk in range(H_kv):
            at = slice(hk * S_max, hk * S_max + n)
            k, v = (_exact_values(x[c + "c"][bk, at], x[c + "s"][bk, at], D) for c in "kv")
            for b in range(case["B"]) if case["shared"] else [bk]:
                for h in range(hk * (H // H_kv), (hk + 1) * (H // H_kv)):
                    w = x["q"][b, :, h].double() @ k.t() / math.sqrt(D)
                    if case["causal"]:
                        seen = torch.ones(S_q, n, dtype=torch.bool, device=DEV).tril(n - S_q)
                        w = torch.where(seen, w, -math.inf)
                    out[b, :, h] = torch.softmax(w, -1) @ v
    return out
