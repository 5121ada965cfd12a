"""Cases of the 8-bit floating point operators: what is measured, and the operators in plain torch.

A block-scaled 8-bit tensor is e4m3 codes with one power-of-two scale per block: 1 x 128 values of a row for
activations, 128 x 128 for weights.  The scale of a block is 2^e with the smallest e >= -127 for which the block's
largest finite magnitude is at most 448 * 2^e (e = 0 for an all-zero block); the codes are the values over the
scale, rounded to nearest even, and a value that is not finite becomes the NaN code.

``own`` False: the operators in elementary torch operations.  True: the calls of ``llima_b200.fp8``.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# GGML type: (values per stored unit, bytes per stored unit)
UNITS = {"Q8_0": (32, 34), "Q4_0": (32, 18), "Q4_K": (256, 144), "Q5_K": (256, 176), "Q6_K": (256, 210)}


def listed():
    return [
        # a token's key projection of Llama-3-8B: the smallest weight that a file of it holds, q/k permutation included
        {"name": "convert Q4_K 1024x4096 heads", "op": "convert", "fmt": "Q4_K", "rows": 1024, "cols": 4096, "heads": 8},
        # Llama-3-8B's down projection
        {"name": "convert Q6_K 4096x14336", "op": "convert", "fmt": "Q6_K", "rows": 4096, "cols": 14336, "heads": 0},
        # Qwen2.5-7B's vocabulary rows, cut where a shard ends off the block grid
        {"name": "convert Q8_0 19007x3584", "op": "convert", "fmt": "Q8_0", "rows": 19007, "cols": 3584, "heads": 0},
        # the norm before a layer's projections: one decoded token, and a long prompt
        {"name": "norm 1x4096", "op": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": True},
        {"name": "norm 8192x4096", "op": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": True},
        # the down projection's input: a small batch of decoded tokens, and a prompt
        {"name": "gated 8x14336", "op": "quantize", "rows": 8, "cols": 14336, "dtype": "bf16", "gate": True},
        {"name": "gated 4096x14336", "op": "quantize", "rows": 4096, "cols": 14336, "dtype": "bf16", "gate": True},
        # the gate and up projections of one decoded token, and the output projection of a batch of 13
        {"name": "matmul 1x28672x4096", "op": "matmul", "rows": 1, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        {"name": "matmul 13x4096x4096", "op": "matmul", "rows": 13, "n": 4096, "k": 4096, "dtype": "bf16", "bias": False},
        # Qwen2.5-7B's query, key and value rows with their bias, for a prompt of odd length
        {"name": "matmul 509x4608x3584 bias", "op": "matmul", "rows": 509, "n": 4608, "k": 3584, "dtype": "f16", "bias": True},
        # the gate and up projections of Llama-3-8B, and its down projection kept in 32 bits, for long prompts
        {"name": "matmul 8192x28672x4096", "op": "matmul", "rows": 8192, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        {"name": "matmul 2048x4096x14336 f32", "op": "matmul", "rows": 2048, "n": 4096, "k": 14336, "dtype": "f32", "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["convert", "norm", "quantize", "matmul", "matmul"])
    if op == "convert":
        fmt = rng.choice(sorted(UNITS))
        unit = UNITS[fmt][0]
        cols = unit * max(1, _log(rng, 256, 16384) // unit)
        rows = max(1, min(_log(rng, 32, 30000), 60_000_000 // cols))
        heads = rng.choice([0, 0, 4, 8])
        if heads:
            rows = max(16 * heads, rows // (16 * heads) * 16 * heads)
        return {"op": op, "fmt": fmt, "rows": rows, "cols": cols, "heads": heads}
    if op in ("norm", "quantize"):
        cols = 32 * _log(rng, 4, 512)
        rows = max(1, min(_log(rng, 1, 8192), 30_000_000 // cols))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, ("residual" if op == "norm" else "gate"): rng.random() < 0.7}
    k = 32 * _log(rng, 8, 512)
    n = _log(rng, 100, 30000)
    rows = max(1, min(_log(rng, 1, 8192), 400_000_000_000 // (n * k)))
    return {"op": op, "rows": rows, "n": n, "k": k, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.3}


# ---- inputs ------------------------------------------------------------------------------


def _gguf_bytes(fmt, n_units, g):
    """Stored units with f16 constants in [1e-4, 1e-2] and uniform quants."""
    u = torch.randint(0, 256, (n_units, UNITS[fmt][1]), dtype=torch.uint8, device="cuda", generator=g)

    def constant():
        c = torch.empty(n_units, device="cuda").uniform_(1e-4, 1e-2, generator=g)
        return c.to(torch.float16).view(torch.uint8).view(n_units, 2)

    if fmt == "Q6_K":
        u[:, 192:208] = torch.randint(-64, 64, (n_units, 16), dtype=torch.int8, device="cuda", generator=g).view(torch.uint8)
        u[:, 208:210] = constant()
    else:
        u[:, 0:2] = constant()
        if fmt in ("Q4_K", "Q5_K"):
            u[:, 2:4] = constant()
    return u.view(-1)


def _activations(rows, cols, dtype, g):
    """Normal values with a few channels far larger than the rest, as hidden states have."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "convert":
        unit = UNITS[case["fmt"]][0]
        s["src"] = _gguf_bytes(case["fmt"], case["rows"] * case["cols"] // unit, g)
        return s
    rows, dtype = case["rows"], DTYPES[case["dtype"]]
    if case["op"] == "norm":
        s["x"] = _activations(rows, case["cols"], dtype, g)
        s["r"] = _activations(rows, case["cols"], dtype, g) if case["residual"] else None
        s["w"] = torch.randn(case["cols"], device="cuda", generator=g) * 0.02 + 1.0
    elif case["op"] == "quantize":
        # gate and up come side by side out of one product
        both = _activations(rows, 2 * case["cols"] if case["gate"] else case["cols"], dtype, g)
        s["x"] = both[:, case["cols"]:] if case["gate"] else both
        s["g"] = both[:, :case["cols"]] if case["gate"] else None
    else:
        s["a"], s["sa"] = _quantize_rows(_activations(rows, case["k"], torch.float32, g))
        s["b"], s["sb"] = _quantize_blocks(torch.randn(case["n"], case["k"], device="cuda", generator=g) * 0.02)
        s["bias"] = torch.randn(case["n"], device="cuda", generator=g) * 0.02 if case["bias"] else None
    return s


# ---- the operators -----------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "convert":
        return _quantize_blocks(_permute(_dequantize(s["fmt"], s["src"]).view(s["rows"], s["cols"]), s["heads"]))
    if s["op"] == "norm":
        h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
        hf = h.float()
        y = hf * torch.rsqrt((hf * hf).mean(1, keepdim=True) + 1e-5) * s["w"]
        return (*_quantize_rows(y), h) if s["r"] is not None else _quantize_rows(y)
    if s["op"] == "quantize":
        y = s["x"].float()
        if s["g"] is not None:
            gate = s["g"].float()
            y = gate / (1.0 + torch.exp(-gate)) * y
        return _quantize_rows(y)
    out = _values(s["a"], s["sa"], 1) @ _values(s["b"], s["sb"], BLOCK).T
    if s["bias"] is not None:
        out += s["bias"]
    return out.to(DTYPES[s["dtype"]])


def _run_own(s):
    from llima_b200 import fp8
    if s["op"] == "convert":
        w = fp8.convert_fp8_device(s["fmt"], s["src"], s["rows"], s["cols"], s["heads"])
        return w.codes, w.scales
    if s["op"] == "norm":
        if s["r"] is None:
            q = fp8.rms_norm_fp8(s["x"], s["w"], 1e-5)
            return q.codes, q.scales
        q, h = fp8.rms_norm_fp8(s["x"], s["w"], 1e-5, residual=s["r"])
        return q.codes, q.scales, h
    if s["op"] == "quantize":
        q = fp8.quantize_fp8(s["x"], gate=s["g"])
        return q.codes, q.scales
    a, b = fp8.Fp8Rows(s["a"], s["sa"]), fp8.Fp8Weight(s["b"], s["sb"])
    return fp8.matmul_fp8(a, b, bias=s["bias"], dtype=DTYPES[s["dtype"]])


def _halves(u, at):
    return u[:, at:at + 2].contiguous().view(torch.float16).float()


def _six_bit(u):
    """(n, 8) scales and mins of the 12 packed bytes of Q4_K and Q5_K."""
    a, b, c = u[:, 4:8], u[:, 8:12], u[:, 12:16]
    sc = torch.cat([a & 63, (c & 15) | (a >> 6 << 4)], 1)
    mn = torch.cat([b & 63, (c >> 4) | (b >> 6 << 4)], 1)
    return sc.float(), mn.float()


def _dequantize(fmt, src):
    """The f32 values of GGUF bytes, each product and difference rounded on its own."""
    u = src.view(-1, UNITS[fmt][1])
    n = u.shape[0]
    if fmt == "Q8_0":
        return _halves(u, 0) * u[:, 2:].contiguous().view(torch.int8).float()
    if fmt == "Q4_0":
        return _halves(u, 0) * (torch.cat([u[:, 2:] & 15, u[:, 2:] >> 4], 1).float() - 8.0)
    if fmt == "Q6_K":
        ql, qh = u[:, :128].reshape(n, 2, 64), u[:, 128:192].reshape(n, 2, 32)
        low = torch.stack([ql[..., :32] & 15, ql[..., 32:] & 15, ql[..., :32] >> 4, ql[..., 32:] >> 4], 2)
        high = torch.stack([qh & 3, qh >> 2 & 3, qh >> 4 & 3, qh >> 6], 2)
        q = (low | high << 4).float().view(n, 16, 16) - 32.0
        scale = _halves(u, 208) * u[:, 192:208].contiguous().view(torch.int8).float()
        return scale[:, :, None] * q
    sc, mn = _six_bit(u)
    scale, least = _halves(u, 0) * sc, _halves(u, 2) * mn
    qs = u[:, 16 if fmt == "Q4_K" else 48:].reshape(n, 4, 1, 32)
    q = torch.cat([qs & 15, qs >> 4], 2).view(n, 8, 32)
    if fmt == "Q5_K":
        bit = torch.arange(8, device=u.device, dtype=torch.uint8).view(1, 8, 1)
        q = q | ((u[:, None, 16:48] >> bit & 1) << 4)
    return scale[:, :, None] * q.float() - least[:, :, None]


def _permute(x, heads):
    """The llama q/k order: row h D + 2 a + t goes to h D + t D / 2 + a."""
    if not heads:
        return x
    rows, cols = x.shape
    return x.view(heads, rows // heads // 2, 2, cols).transpose(1, 2).reshape(rows, cols)


def _exponent(amax):
    m, e = torch.frexp(amax)
    e = torch.where(m <= E4M3_MAX / 512.0, e - 9, e - 8)
    return torch.where(amax == 0, 0, e).clamp_min(-127).to(torch.int32)


def _powers(e):
    """2^-e for -127 <= e <= 120, exactly."""
    return (127 - e << 23).view(torch.float32)


def _stored(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _quantize_rows(y):
    rows, cols = y.shape
    blocks = -(-cols // BLOCK)
    padded = torch.nn.functional.pad(y, (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    e = _exponent(torch.where(torch.isfinite(padded), padded.abs(), 0.0).amax(2))
    codes = (padded * _powers(e)[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks * BLOCK)
    return codes[:, :cols].contiguous(), _stored(e)


def _quantize_blocks(x):
    rows, cols = x.shape
    rb, cb = -(-rows // BLOCK), -(-cols // BLOCK)
    padded = torch.nn.functional.pad(x, (0, cb * BLOCK - cols, 0, rb * BLOCK - rows)).view(rb, BLOCK, cb, BLOCK)
    e = _exponent(torch.where(torch.isfinite(padded), padded.abs(), 0.0).amax((1, 3)))
    codes = (padded * _powers(e)[:, None, :, None]).to(torch.float8_e4m3fn).view(rb * BLOCK, cb * BLOCK)
    return codes[:rows, :cols].contiguous(), _stored(e)


def _values(codes, scales, rows_per_scale):
    rows, cols = codes.shape
    s = scales.float().repeat_interleave(rows_per_scale, 0)[:rows] if rows_per_scale > 1 else scales.float()
    return codes.float() * s.repeat_interleave(BLOCK, 1)[:, :cols]


# ---- the definitions in 64 bits ----------------------------------------------------------


def exact(case, seed):
    """Codes come as the unrounded quotients, scales as powers of two."""
    s = prepare(case, seed)
    if case["op"] == "convert":
        rows, cols = case["rows"], case["cols"]
        row = torch.arange(rows, device="cuda")
        if case["heads"]:
            d = rows // case["heads"]
            i = row % d
            row = row - i + 2 * (i % (d // 2)) + i // (d // 2)
        return _exact_blocks(_exact_values(case["fmt"], s["src"]).view(rows, cols)[row], BLOCK)
    if case["op"] == "norm":
        if s["r"] is None:
            return _exact_blocks(_exact_norm(s["x"].double(), s["w"]), 1)
        h = s["x"].double() + s["r"].double()
        kept = h.to(s["x"].dtype).double()      # the norm is of the sum as it is stored
        return (*_exact_blocks(_exact_norm(kept, s["w"]), 1), h)
    if case["op"] == "quantize":
        y = s["x"].double()
        if s["g"] is not None:
            y = y * s["g"].double() * torch.sigmoid(s["g"].double())
        return _exact_blocks(y, 1)
    out = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    per_row = s["sb"].double()[torch.arange(case["n"], device="cuda") // BLOCK]
    for k in range(0, case["k"], BLOCK):
        part = s["a"][:, k:k + BLOCK].double() @ s["b"][:, k:k + BLOCK].double().T
        out += part * s["sa"][:, k // BLOCK].double()[:, None] * per_row[:, k // BLOCK]
    return out if s["bias"] is None else out + s["bias"].double()


def _exact_norm(h, w):
    return h / torch.sqrt((h ** 2).sum(1, keepdim=True) / h.shape[1] + 1e-5) * w.double()


def _exact_blocks(y, tall):
    """Quotients and scales of blocks of `tall` x 128."""
    rows, cols = y.shape
    r, c = torch.arange(rows, device="cuda") // tall, torch.arange(cols, device="cuda") // BLOCK
    amax = torch.nn.functional.max_pool2d(y.abs()[None], (tall, BLOCK), ceil_mode=True)[0]
    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp_min(amax, 1e-300) / E4M3_MAX)).clamp_min(-127))
    scale = torch.where(amax == 0, 1.0, scale)
    return y / scale[r][:, c], scale


def _exact_values(fmt, src):
    """One value at a time from its place in the unit, all values at once."""
    values, size = UNITS[fmt]
    u = src.view(-1, size).long()
    v = torch.arange(values, device="cuda")

    def half(at):
        return (u[:, at] + 256 * u[:, at + 1]).to(torch.int16).view(torch.float16).double()[:, None]

    if fmt == "Q8_0":
        return half(0) * ((u[:, 2 + v] + 128) % 256 - 128)
    if fmt == "Q4_0":
        return half(0) * (u[:, 2 + v % 16] // 16 ** (v // 16) % 16 - 8)
    if fmt == "Q6_K":
        h, part, j = v // 128, v % 128 // 32, v % 32
        low = u[:, 64 * h + 32 * (part % 2) + j] // 16 ** (part // 2) % 16
        high = u[:, 128 + 32 * h + j] // 4 ** part % 4
        sub = (u[:, 192 + v // 16] + 128) % 256 - 128
        return half(208) * sub * (low + 16 * high - 32)
    k, j = v // 32, v % 32
    first, second = u[:, 4 + k % 4], u[:, 8 + k % 4]
    third = u[:, 12 + k % 4]
    sub = torch.where(k < 4, first % 64, third % 16 + first // 64 * 16)
    least = torch.where(k < 4, second % 64, third // 16 + second // 64 * 16)
    q = u[:, (16 if fmt == "Q4_K" else 48) + 32 * (k // 2) + j] // 16 ** (k % 2) % 16
    if fmt == "Q5_K":
        q = q + u[:, 16 + j] // 2 ** k % 2 * 16
    return half(0) * sub * q - half(2) * least


def work(case):
    if case["op"] == "convert":
        rows, cols = case["rows"], case["cols"]
        values, size = UNITS[case["fmt"]]
        blocks = -(-rows // BLOCK) * -(-cols // BLOCK)
        return {"bytes": rows * cols // values * size + rows * cols + blocks, "flops": 2 * rows * cols}
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "matmul":
        m, n, k = case["rows"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        read = m * k + n * k + m * kb + -(-n // BLOCK) * kb + (4 * n if case["bias"] else 0)
        return {"bytes": read + m * n * size, "flops": 2 * m * n * k}
    values = case["rows"] * case["cols"]
    written = values + case["rows"] * -(-case["cols"] // BLOCK)
    if case["op"] == "norm":
        return {"bytes": values * size * (3 if case["residual"] else 1) + 4 * case["cols"] + written, "flops": 6 * values}
    return {"bytes": values * size * (2 if case["gate"] else 1) + written, "flops": (8 if case["gate"] else 2) * values}
