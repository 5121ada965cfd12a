"""Block-scaled 8-bit floats against plain implementations in 64 bits.

Weights: the f32 values come from the CPU oracle, and scaling by a power of two is exact, so
scales and codes are compared byte for byte (any NaN code equals any other).

Activations: y is computed in 64 bits.  The kernel's f32 y is off by at most YERR (relative):
the norm takes one rounding each for the mean, the sum with eps, the square root, the
quotient and two products (2^-24 each; halved by the root for the first two) and the sum of
squares, whose relative error is at most (terms added one after another) * 2^-24 <= 2^-17 for
the 128 of a thread of the widest row here plus the tree, halved by the root: below 2^-17 in
all.  The gated product takes an exponential of at most 2 + 1.5 |x| ulp (|x| < 30 here), a
reciprocal of 1 ulp and three roundings: below 2^-17.  So a code's value is within half a
step of y (2^-4 relative, or 2^-10 of the scale below the normal range) plus 2^-17 of y, and
a scale may differ only where the block's largest |y| is that near 448 * 2^e.

Products: every product of two e4m3 values is exact in f32, and k of them summed in f32 in
any order, each sum rounded or truncated, are off by at most k 2^-23 sum|a b|; the result is
rounded once more, by half a step of its type.
"""
import ctypes

import numpy as np
import pytest
import torch
from ml_dtypes import bfloat16

from llima_b200 import _native as N
from llima_b200 import fp8
from llima_b200.formats import FORMATS
from llima_b200.synth import gen_tensor_bytes
from oracle import ggml_oracle as O

pytestmark = pytest.mark.gpu

YERR = 2.0 ** -17
DEV = "cuda"


# ---- plain forms --------------------------------------------------------------------------


def exponent(amax: np.ndarray) -> np.ndarray:
    """Smallest e >= -127 with amax <= 448 * 2^e; 0 where amax is 0."""
    m, e = np.frexp(amax.astype(np.float64))
    e = np.where(m <= 0.875, e - 9, e - 8)
    return np.where(amax == 0, 0, np.maximum(e, -127)).astype(np.int64)


def e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 code bytes of f32 values of at most 448; NaN code where not finite."""
    t = torch.from_numpy(np.where(np.isfinite(x), x, np.nan).astype(np.float32))
    return t.to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def blocks_of(x: np.ndarray, tall: int) -> np.ndarray:
    r, c = x.shape
    p = np.zeros((-(-r // tall) * tall, -(-c // 128) * 128), x.dtype)
    p[:r, :c] = x
    return p.reshape(p.shape[0] // tall, tall, p.shape[1] // 128, 128)


def quantize_plain(x: np.ndarray, tall: int):
    """Code bytes and scale bytes of f32 values."""
    p = blocks_of(x, tall)
    with np.errstate(all="ignore"):
        e = exponent(np.where(np.isfinite(p), np.abs(p), 0).max((1, 3)))
        q = e4m3(np.ldexp(p.astype(np.float64), -e[:, None, :, None].astype(np.int32)))
    return q.reshape(p.shape[0] * tall, -1)[:x.shape[0], :x.shape[1]], (e + 127).astype(np.uint8)


def bytes_of(t: torch.Tensor) -> np.ndarray:
    return t.view(torch.uint8).cpu().numpy()


def same_codes(got: np.ndarray, want: np.ndarray) -> bool:
    nan = ((got & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F)
    zero = ((got & 0x7F) == 0) & ((want & 0x7F) == 0)
    return got.shape == want.shape and bool(np.all(nan | zero | (got == want)))


def values_of(q) -> np.ndarray:
    """The values that codes and scales stand for, in 64 bits."""
    c, s = q.codes.float().cpu().double().numpy(), q.scales.float().cpu().double().numpy()
    tall = 1 if isinstance(q, fp8.Fp8Rows) else 128
    s = np.repeat(np.repeat(s, tall, 0)[:c.shape[0]], 128, 1)[:, :c.shape[1]]
    return c * s


def check_rows(q: fp8.Fp8Rows, y: np.ndarray):
    """Codes and scales of activations against y in 64 bits (see the module's comment)."""
    rows, cols = y.shape
    assert q.codes.shape == (rows, cols) and q.scales.shape == (rows, -(-cols // 128))
    p = blocks_of(y, 1)
    amax = np.where(np.isfinite(p), np.abs(p), 0).max((1, 3))
    e = bytes_of(q.scales).astype(np.int64) - 127
    low, high = exponent(amax * (1 - YERR)), exponent(amax * (1 + YERR))
    assert np.all((e == low) | (e == high)), "a scale is off"
    c = q.codes.float().cpu().double().numpy()
    s = np.ldexp(1.0, np.repeat(e, 128, 1)[:, :cols].astype(np.int32))
    bad = ~np.isfinite(y)
    assert np.array_equal(np.isnan(c), bad)
    with np.errstate(all="ignore"):
        off = np.abs(c * s - y)
        limit = np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) + np.abs(y) * YERR
    assert np.all((off <= limit) | bad), f"a code is off by {np.nanmax(off / limit)} of its limit"


# ---- weights ------------------------------------------------------------------------------

TYPES = ["Q8_0", "Q4_0", "Q4_1", "Q5_0", "Q5_1", "Q2_K", "Q3_K", "Q4_K", "Q5_K", "Q6_K", "F32", "F16", "BF16"]


def raw_bytes(fmt, rows, cols, seed):
    if fmt in ("F16", "BF16"):
        v = np.random.default_rng(seed).normal(0, 0.05, rows * cols).astype(np.float32)
        return v.astype(np.float16 if fmt == "F16" else bfloat16).view(np.uint8)
    return gen_tensor_bytes(fmt, rows * cols, seed, "bias")


def oracle_values(fmt, raw, rows, cols):
    if fmt in ("F32", "F16", "BF16"):
        t = {"F32": np.float32, "F16": np.float16, "BF16": bfloat16}[fmt]
        return raw.view(t).astype(np.float32).reshape(rows, cols)
    with np.errstate(all="ignore"):
        return O.gguf_dequantize(raw.tobytes(), fmt).reshape(rows, cols)


def permute(x, heads):
    rows = x.shape[0]
    return x.reshape(heads, rows // heads // 2, 2, -1).swapaxes(1, 2).reshape(x.shape) if heads else x


def check_weight(fmt, raw, rows, cols, heads=0):
    w = fp8.convert_fp8_device(fmt, torch.from_numpy(raw.copy()).to(DEV), rows, cols, heads)
    torch.cuda.synchronize()
    codes, scales = quantize_plain(permute(oracle_values(fmt, raw, rows, cols), heads), 128)
    assert np.array_equal(bytes_of(w.scales), scales)
    assert same_codes(bytes_of(w.codes), codes)


@pytest.mark.parametrize("fmt", TYPES)
@pytest.mark.parametrize("rows,units", [(1, 1), (37, 3), (128, 2), (129, 5), (300, 4)])
def test_weight_matches_oracle(fmt, rows, units):
    cols = units * max(32, FORMATS[fmt].unit_values)
    check_weight(fmt, raw_bytes(fmt, rows, cols, rows + units), rows, cols)


@pytest.mark.parametrize("fmt", TYPES)
def test_weight_head_permutation(fmt):
    cols = 2 * max(32, FORMATS[fmt].unit_values)
    check_weight(fmt, raw_bytes(fmt, 288, cols, 5), 288, cols, heads=3)


@pytest.mark.parametrize("fmt", TYPES)
@pytest.mark.parametrize("rows,cols,heads", [(300, 2048, 0), (129, 640, 0), (512, 2048, 4), (512, 2048, 8), (512, 768, 2), (640, 2048, 40),
                                             (512, 2048, 64), (576, 2048, 3), (1024, 512, 2), (5, 2304, 0)])
def test_weight_rows_of_whole_16_bytes_and_not(fmt, rows, cols, heads):
    """Rows whose bytes are a multiple of 16 arrive in boxes, others one by one; heads of 128, 64,
    256, 16, 8, 192 and 512 rows."""
    cols = cols // FORMATS[fmt].unit_values * FORMATS[fmt].unit_values
    check_weight(fmt, raw_bytes(fmt, rows, cols, rows + heads), rows, cols, heads)


@pytest.mark.parametrize("fmt", [t for t in TYPES if t[0] == "Q"])
def test_weight_of_random_bytes(fmt):
    """NaN, infinite, negative, subnormal and huge f16 constants."""
    f = FORMATS[fmt]
    for rows, cols in ((260, 2 * max(128, f.unit_values)), (130, 2048)):
        raw = np.frombuffer(np.random.default_rng(9).bytes(rows * cols // f.unit_values * f.unit_bytes), np.uint8)
        check_weight(fmt, raw, rows, cols)


def test_weight_float_extremes():
    """All-zero blocks, infinities and NaN beside finite values, subnormals, the largest f32,
    and largest magnitudes on both sides of 448 * 2^e."""
    x = np.random.default_rng(1).normal(0, 1, (300, 640)).astype(np.float32)
    x[:128, :128] = 0
    x[3, 130], x[4, 140], x[5, 150] = np.inf, -np.inf, np.nan
    x[:128, 256:384] *= np.float32(1e-42)
    x[:128, 384:512] *= np.float32(1e38)
    x[128:256, :128] = np.clip(x[128:256, :128], -1, 1)
    x[128, 0] = np.float32(448 / 256)                       # exactly representable: the smaller scale
    x[128:256, 128:256] = np.clip(x[128:256, 128:256], -1, 1)
    x[128, 128] = np.nextafter(np.float32(448 / 256), np.float32(2))
    x[256:, 512:] = np.inf
    check_weight("F32", x.view(np.uint8).reshape(-1), 300, 640)


def test_weight_full_size_projection():
    rows, cols = 1024, 4096
    check_weight("Q4_K", raw_bytes("Q4_K", rows, cols, 2), rows, cols, heads=8)


# ---- activations --------------------------------------------------------------------------

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def rows_of(rows, cols, dtype, seed, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if outliers:
        x[:, ::97] *= 20
    return x.to(dtype).to(DEV)


def norm_plain(h, w, eps):
    h = h.cpu().double().numpy()
    with np.errstate(all="ignore"):
        return h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w.cpu().double().numpy()


NORM_SHAPES = [(1, 32), (3, 96), (1, 4096), (5, 128), (2, 1056), (300, 512), (7, 3584), (2, 8224), (1, 32768), (2, 40992)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm(rows, cols, dtype):
    x, r = rows_of(rows, cols, dtype, 1), rows_of(rows, cols, dtype, 2)
    w = torch.randn(cols, generator=torch.Generator().manual_seed(3)).to(DEV)
    check_rows(fp8.rms_norm_fp8(x, w, 1e-5), norm_plain(x, w, 1e-5))
    q, h = fp8.rms_norm_fp8(x, w, 1e-6, residual=r)
    want = (x.float() + r.float()).to(dtype)
    assert torch.equal(h, want)
    check_rows(q, norm_plain(want, w, 1e-6))


def test_norm_in_place_and_strided():
    """x and the residual as column ranges of wider tensors, the sum over the residual or over
    x, and what lies beside them left as it was."""
    for where in ("residual", "x"):
        both, wide = rows_of(9, 1024, torch.bfloat16, 4), rows_of(9, 768, torch.bfloat16, 5)
        x, r = both[:, 512:], wide[:, 128:640]
        codes = torch.zeros(9, 1024, dtype=torch.uint8, device=DEV)
        scales = torch.zeros(9, 7, dtype=torch.uint8, device=DEV)
        out = fp8.Fp8Rows(codes[:, 256:768].view(fp8.E4M3), scales[:, 1:5].view(fp8.E8M0))
        w = torch.ones(512, device=DEV)
        want = (x.float() + r.float()).bfloat16()
        before = both.clone(), wide.clone()
        target = r if where == "residual" else x
        q, h = fp8.rms_norm_fp8(x, w, residual=r, sum_out=target, out=out)
        assert h is target and torch.equal(h, want)
        check_rows(q, norm_plain(want, w, 1e-5))
        assert torch.equal(both[:, :512], before[0][:, :512])
        assert torch.equal(wide[:, :128], before[1][:, :128]) and torch.equal(wide[:, 640:], before[1][:, 640:])
        assert not codes[:, :256].any() and not codes[:, 768:].any() and not scales[:, 0].any() and not scales[:, 5:].any()


def test_norm_zero_and_nonfinite_rows():
    x = rows_of(6, 256, torch.float32, 6, outliers=False)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 9] = float("nan")
    x[3] *= 1e-30
    x[4] *= 1e25     # squares overflow f32: the mean is infinite and the row's quotients 0
    w = torch.ones(256, device=DEV)
    q = fp8.rms_norm_fp8(x, w, 0.0)
    c = q.codes.float().cpu()
    assert torch.isnan(c[0]).all()            # 0 / 0 at eps = 0
    assert torch.isnan(c[1, 7]) and (c[1].nan_to_num() == 0).all()
    assert torch.isnan(c[2]).all()
    assert (bytes_of(q.scales)[:3] == 127).all()
    assert torch.isnan(c[3]).all() or (c[3] != 0).any()
    assert (c[4] == 0).all()
    check_rows(fp8.Fp8Rows(q.codes[5:], q.scales[5:]), norm_plain(x[5:], w, 0.0))
    z = fp8.rms_norm_fp8(x[:1], w, 1e-5)
    assert (z.codes.float() == 0).all() and (bytes_of(z.scales) == 127).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_quantize(rows, cols, dtype):
    x = rows_of(rows, cols, dtype, 7)
    q = fp8.quantize_fp8(x)
    codes, scales = quantize_plain(x.float().cpu().numpy(), 1)
    assert np.array_equal(bytes_of(q.scales), scales) and same_codes(bytes_of(q.codes), codes)
    both = rows_of(rows, 2 * cols, dtype, 8, outliers=False)
    g, u = both[:, :cols].cpu().double().numpy(), both[:, cols:].cpu().double().numpy()
    check_rows(fp8.quantize_fp8(both[:, cols:], gate=both[:, :cols]), g / (1 + np.exp(-g)) * u)


def test_quantize_extremes():
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(6, 160, device=DEV)
    x[0, :4] = torch.tensor([1.0, inf, -inf, nan])
    x[1, :2] = torch.tensor([3.4e38, -1e-45])
    x[2, :3] = torch.tensor([1e-45, 1e-40, -1e-38])
    x[3] = inf
    x[4, 128:] = torch.linspace(-448, 448, 32)
    x[5, 128:] = torch.linspace(-448.1, 448.1, 32)
    q = fp8.quantize_fp8(x)
    codes, scales = quantize_plain(x.cpu().numpy(), 1)
    assert np.array_equal(bytes_of(q.scales), scales) and same_codes(bytes_of(q.codes), codes)
    g = torch.zeros(2, 128, device=DEV)
    g[0, :5] = torch.tensor([100.0, -100.0, inf, -inf, nan])
    y = fp8.quantize_fp8(torch.ones(2, 128, device=DEV), gate=g)
    c = (y.codes.float() * y.scales.float()).cpu()
    assert abs(float(c[0, 0]) - 100) <= 100 / 16 and abs(float(c[0, 1])) <= 2.0 ** -4
    assert torch.isnan(c[0, 2:5]).all() and (c[0, 5:] == 0).all() and (c[1] == 0).all()


# ---- products -----------------------------------------------------------------------------


def operands(m, n, k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    a = fp8.quantize_fp8(torch.randn(m, k, device=DEV, generator=g) * torch.rand(m, 1, device=DEV, generator=g).exp2())
    raw = (torch.randn(n, k, device=DEV, generator=g) * 0.02).view(torch.uint8).view(-1)
    return a, fp8.convert_fp8_device("F32", raw, n, k)


def check_product(out, a, w, bias=None):
    k = a.codes.shape[1]
    av, wv = torch.from_numpy(values_of(a)).to(DEV), torch.from_numpy(values_of(w)).to(DEV)
    want = av @ wv.T
    bound = av.abs() @ wv.abs().T
    if bias is not None:
        want += bias.double()
        bound += bias.double().abs()
    half = torch.finfo(out.dtype).eps / 2
    limit = (k + 1) * 2.0 ** -23 * bound + half * want.abs() + torch.finfo(out.dtype).tiny
    off = (out.double() - want).abs()
    assert torch.isfinite(want).all() and bool((off <= limit).all()), f"off by {float((off / limit).max())} of the limit"
    # the bound above is a worst case: together the errors stay near the rounding of the result
    far = float(off.norm() / want.norm().clamp_min(1e-30))
    assert far <= max(half, 2e-6), far


MS = [1, 2, 7, 16, 17, 33, 64, 65, 100, 128, 129, 257, 300, 520]


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k", [(1, 32), (100, 96), (128, 128), (129, 160), (384, 512), (260, 640), (513, 1056), (256, 4128)])
def test_product(m, n, k):
    a, w = operands(m, n, k, m + n + k)
    dtype = FLOATS[(m + n) % 3]
    check_product(fp8.matmul_fp8(a, w, dtype=dtype), a, w)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m", [1, 5, 48, 130, 512])
@pytest.mark.parametrize("n", [64, 333, 1152])
def test_product_bias_and_types(m, n, dtype):
    a, w = operands(m, n, 1024, m)
    bias = torch.randn(n, device=DEV)
    check_product(fp8.matmul_fp8(a, w, bias=bias, dtype=dtype), a, w, bias)


@pytest.mark.parametrize("m,n,k", [(1, 28672, 4096), (13, 4096, 14336), (509, 4608, 3584), (2000, 4096, 4096), (1100, 6152, 2080),
                                   (4096, 1024, 512), (3, 128256, 256)])
def test_product_full_size(m, n, k):
    a, w = operands(m, n, k, 1)
    check_product(fp8.matmul_fp8(a, w, dtype=torch.float32), a, w)


# more weight rows than one tile per SM holds, so that k is not split: sums of 34, 67 and 99 blocks
# in two to four pieces, whose ends do not fall on a group of four
@pytest.mark.parametrize("m,n,k", [(3, 19100, 4256), (20, 19100, 4256), (50, 19100, 4256), (3, 19100, 8480), (50, 19100, 8480),
                                   (20, 19100, 12672), (600, 2600, 4256), (600, 2600, 8480)])
def test_product_pieces(m, n, k):
    a, w = operands(m, n, k, 7)
    check_product(fp8.matmul_fp8(a, w, dtype=torch.float32), a, w)


@pytest.mark.parametrize("m", [1, 3, 40, 200, 600])
def test_product_strided_operands(m):
    """Operands and output as ranges of wider tensors; what lies beside the output stays."""
    n, k = 200, 416
    a, w = operands(m, n, k, 3)
    wide_a = torch.full((m + 2, k + 48), 0x7F, dtype=torch.uint8, device=DEV)      # NaN around the codes
    wide_a[1:-1, 16:16 + k] = a.codes.view(torch.uint8)
    wide_sa = torch.full((m + 2, 11), 0xFF, dtype=torch.uint8, device=DEV)
    wide_sa[1:-1, 3:7] = a.scales.view(torch.uint8)
    wide_w = torch.full((n + 3, k + 64), 0x7F, dtype=torch.uint8, device=DEV)
    wide_w[2:-1, 32:32 + k] = w.codes.view(torch.uint8)
    wide_sw = torch.full((4, 9), 0xFF, dtype=torch.uint8, device=DEV)
    wide_sw[1:3, 1:5] = w.scales.view(torch.uint8)
    sa = fp8.Fp8Rows(wide_a[1:-1, 16:16 + k].view(fp8.E4M3), wide_sa[1:-1, 3:7].view(fp8.E8M0))
    sw = fp8.Fp8Weight(wide_w[2:-1, 32:32 + k].view(fp8.E4M3), wide_sw[1:3, 1:5].view(fp8.E8M0))
    for dtype in FLOATS:
        for left, pitch in ((8, n + 24), (1, n + 3)):
            wide = torch.full((m + 2, pitch), 7.0, dtype=dtype, device=DEV)
            out = wide[1:-1, left:left + n]
            assert fp8.matmul_fp8(sa, sw, out=out) is out
            check_product(out, a, w)
            wide[1:-1, left:left + n] = 7.0
            assert bool((wide == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [2600, 2597, 2612])
@pytest.mark.parametrize("k,layout", [(320, "plain"), (2080, "plain"), (2080, "offset"), (2080, "pitch"), (4128, "plain"), (17440, "plain")])
def test_product_many_tiles(n, k, layout, dtype):
    """More tiles than pairs of SMs, with sums of one and several batches of scales, rows of the
    output on and off 16 bytes, and scales that lie side by side, off 16 bytes, or apart."""
    m = 2500 if k < 10000 else 1900
    a, w = operands(m, n, k, 31)
    blocks = a.scales.shape[1]

    def relay(t):
        left, pitch = {"plain": (0, blocks), "offset": (3, blocks + 5), "pitch": (0, blocks + 7)}[layout]
        wide = torch.full((t.shape[0] + 1, pitch), 0xFF, dtype=torch.uint8, device=DEV)
        wide[:-1, left:left + blocks] = t.view(torch.uint8)
        return wide[:-1, left:left + blocks].view(fp8.E8M0)

    a, w = fp8.Fp8Rows(a.codes, relay(a.scales)), fp8.Fp8Weight(w.codes, relay(w.scales))
    bias = torch.randn(n, device=DEV) if k == 2080 else None
    check_product(fp8.matmul_fp8(a, w, bias=bias, dtype=dtype), a, w, bias)


def test_scales_at_the_end_of_their_memory():
    """Scales whose last byte is their allocation's last: nothing past them is read for a result."""
    for m, n, k in ((2500, 2600, 2080), (2499, 2597, 4128), (130, 300, 1056)):
        a, w = operands(m, n, k, 32)

        def at_end(t):
            room = -(-t.numel() // 512) * 512
            buf = torch.full((room,), 0xFF, dtype=torch.uint8, device=DEV)
            start = (room - t.numel()) // 16 * 16       # on 16 bytes, so that the bulk copies are taken
            buf[start:start + t.numel()] = t.view(torch.uint8).reshape(-1)
            return buf[start:start + t.numel()].view(t.shape).view(fp8.E8M0)

        b, v = fp8.Fp8Rows(a.codes, at_end(a.scales)), fp8.Fp8Weight(w.codes, at_end(w.scales))
        assert torch.equal(fp8.matmul_fp8(b, v, dtype=torch.float32), fp8.matmul_fp8(a, w, dtype=torch.float32))


def test_product_nan_reaches_its_row_and_column_only():
    for m in (5, 300):
        a, w = operands(m, 200, 256, 4)
        plain = fp8.matmul_fp8(a, w, dtype=torch.float32)
        a.codes.view(torch.uint8)[2, 17] = 0x7F
        w.codes.view(torch.uint8)[150, 200] = 0xFF
        a.scales.view(torch.uint8)[4, 1] = 0xFF
        out = fp8.matmul_fp8(a, w, dtype=torch.float32)
        want = torch.zeros(m, 200, dtype=torch.bool, device=DEV)
        want[2] = want[4] = True
        want[:, 150] = True
        assert torch.equal(torch.isnan(out), want)
        assert torch.equal(out[~want], plain[~want])


@pytest.mark.parametrize("m", [2, 200])
def test_product_wide_scales(m):
    """Scales far apart whose products are ordinary, and blocks that are negligible or zero."""
    a, w = operands(m, 256, 512, 5)
    sa, sw = a.scales.view(torch.uint8), w.scales.view(torch.uint8)
    sa[:, 0] += 100
    sw[:, 0] -= 100
    sa[:, 1] -= 90
    sw[:, 1] += 90
    sa[:, 2] -= 60
    a.codes.view(torch.uint8)[:, 384:] = 0
    check_product(fp8.matmul_fp8(a, w, dtype=torch.float32), a, w)


def test_product_empty():
    a, w = operands(4, 128, 128, 6)
    none = fp8.Fp8Rows(a.codes[:0], a.scales[:0])
    assert fp8.matmul_fp8(none, w).shape == (0, 128)
    assert fp8.matmul_fp8(a, fp8.Fp8Weight(w.codes[:0], w.scales[:0])).shape == (4, 0)
    bias = torch.randn(128, device=DEV)
    flat = fp8.Fp8Rows(a.codes[:, :0], a.scales[:, :0])
    flat_w = fp8.Fp8Weight(w.codes[:, :0], w.scales[:, :0])
    assert torch.equal(fp8.matmul_fp8(flat, flat_w, bias=bias, dtype=torch.float32), bias.expand(4, 128))
    assert (fp8.matmul_fp8(flat, flat_w) == 0).all()
    assert fp8.quantize_fp8(torch.zeros(0, 64, device=DEV)).codes.shape == (0, 64)
    q, h = fp8.rms_norm_fp8(torch.zeros(0, 64, device=DEV), torch.ones(64, device=DEV), residual=torch.zeros(0, 64, device=DEV))
    assert q.codes.shape == (0, 64) and h.shape == (0, 64)
    assert fp8.convert_fp8_device("Q8_0", torch.zeros(0, dtype=torch.uint8, device=DEV), 0, 64).codes.shape == (0, 64)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (20, 1000, 2048), (700, 1280, 1024)])
def test_product_repeats_bit_for_bit(m, n, k):
    a, w = operands(m, n, k, 8)
    first = fp8.matmul_fp8(a, w, dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(fp8.matmul_fp8(a, w, dtype=torch.float32), first)


# ---- past 32 bits ---------------------------------------------------------------------------


def test_rows_past_32_bits():
    """More than 2^31 values: the last rows come out as they do on their own."""
    rows, cols = 527_000, 4096
    x = torch.randn(1000, cols, device=DEV).bfloat16().repeat(rows // 1000, 1)
    x[-5:] *= torch.arange(1, 6, device=DEV)[:, None].bfloat16()
    w = torch.randn(cols, device=DEV)
    for call in (fp8.quantize_fp8, lambda t: fp8.rms_norm_fp8(t, w)):
        q, tail = call(x), call(x[-70:].clone())
        assert torch.equal(q.codes[-70:].view(torch.uint8), tail.codes.view(torch.uint8))
        assert torch.equal(q.scales[-70:].view(torch.uint8), tail.scales.view(torch.uint8))
        del q
    q, h = fp8.rms_norm_fp8(x, w, residual=x, sum_out=x)
    del q
    assert torch.equal(h[1000:1010], h[:10]) and torch.equal(h[-1005:-1000], h[-2005:-2000])


def test_weight_past_32_bits():
    rows, cols = 131_200, 16_416
    size = cols // 32 * 18
    raw = torch.randint(0, 256, (rows, size), dtype=torch.uint8, device=DEV)
    raw.view(rows, -1, 18)[:, :, 0:2] = torch.tensor([0x66, 0x1C], dtype=torch.uint8, device=DEV)      # an ordinary f16
    w = fp8.convert_fp8_device("Q4_0", raw.view(-1), rows, cols)
    tail = fp8.convert_fp8_device("Q4_0", raw[-256:].reshape(-1).clone(), 256, cols)
    assert torch.equal(w.codes[-256:].view(torch.uint8), tail.codes.view(torch.uint8))
    assert torch.equal(w.scales[-2:].view(torch.uint8), tail.scales.view(torch.uint8))
    # and as an operand
    a = operands(3, 1, cols, 50)[0]
    out = fp8.matmul_fp8(a, w, dtype=torch.float32)
    check_product(out[:, -256:], a, tail)


@pytest.mark.parametrize("n", [32_768, 32_765])
def test_product_past_32_bits(n):
    m, k = 66_000, 160
    a, w = operands(m, n, k, 51)
    out = fp8.matmul_fp8(a, w)
    tail = fp8.Fp8Rows(a.codes[-300:], a.scales[-300:])
    check_product(out[-300:], tail, w)


# ---- refusals of the Python layer -----------------------------------------------------------


def test_refusals():
    a, w = operands(4, 128, 256, 9)
    x = torch.zeros(4, 256, device=DEV, dtype=torch.bfloat16)
    ones = torch.ones(256, device=DEV)
    with pytest.raises(ValueError):
        fp8.quantize_fp8(torch.zeros(4, 100, device=DEV))
    with pytest.raises(ValueError):
        fp8.quantize_fp8(torch.zeros(4, 3, 32, device=DEV))
    with pytest.raises(ValueError):
        fp8.quantize_fp8(torch.zeros(256, 4, device=DEV).T)
    with pytest.raises(ValueError):
        fp8.quantize_fp8(torch.zeros(1, 256, device=DEV).expand(4, 256))
    with pytest.raises(TypeError):
        fp8.quantize_fp8(torch.zeros(4, 256, device=DEV, dtype=torch.float64))
    with pytest.raises(TypeError):
        fp8.quantize_fp8(x, gate=x.float())
    with pytest.raises(ValueError):
        fp8.quantize_fp8(x, gate=x[:2])
    with pytest.raises(N.GqError):
        fp8.quantize_fp8(torch.zeros(4, 260, device=DEV, dtype=torch.bfloat16)[:, 4:])     # rows off 16 bytes
    with pytest.raises(ValueError):
        fp8.rms_norm_fp8(x, ones[:128])
    with pytest.raises(ValueError):
        fp8.rms_norm_fp8(x, ones.bfloat16())
    with pytest.raises(ValueError):
        fp8.rms_norm_fp8(x, ones, sum_out=x)
    with pytest.raises(ValueError):
        fp8.matmul_fp8(fp8.Fp8Rows(a.codes[:, :128], a.scales[:, :1]), w)
    with pytest.raises(ValueError):
        fp8.matmul_fp8(fp8.Fp8Rows(a.codes, a.scales[:, :1]), w)
    with pytest.raises(TypeError):
        fp8.matmul_fp8(fp8.Fp8Rows(a.codes, a.scales.view(torch.uint8)), w)
    with pytest.raises(TypeError):
        fp8.matmul_fp8(a, w, dtype=torch.float64)
    with pytest.raises(ValueError):
        fp8.matmul_fp8(a, w, bias=torch.zeros(127, device=DEV))
    with pytest.raises(ValueError):
        fp8.matmul_fp8(a, w, out=torch.empty(4, 127, device=DEV))
    with pytest.raises(ValueError):
        fp8.matmul_fp8(a, w, out=torch.empty(128, 4, device=DEV).T)
    with pytest.raises(N.GqError):
        fp8.convert_fp8_device("Q4_K", torch.zeros(143, dtype=torch.uint8, device=DEV), 1, 256)


# ---- together -------------------------------------------------------------------------------


def _gguf_file(path, hidden=256, ff=384):
    import gguf
    w = gguf.GGUFWriter(str(path), "llama")
    w.add_layer_norm_rms_eps(1e-6)
    for name, fmt, rows, cols in (("ffn_gate", "Q4_K", ff, hidden), ("ffn_up", "Q5_K", ff, hidden), ("ffn_down", "Q8_0", hidden, ff),
                                  ("attn_q", "Q6_K", hidden, hidden)):
        raw = gen_tensor_bytes(fmt, rows * cols, len(name))
        f = FORMATS[fmt]
        w.add_tensor(f"blk.3.{name}.weight", raw.reshape(rows, cols // f.unit_values * f.unit_bytes),
                     raw_dtype=gguf.GGMLQuantizationType(f.type_id))
    w.add_tensor("blk.3.ffn_norm.weight", np.random.default_rng(0).normal(1, 0.1, hidden).astype(np.float32))
    w.add_tensor("blk.3.attn_q.bias", np.random.default_rng(1).normal(0, 0.1, hidden).astype(np.float32))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()


@pytest.mark.parametrize("rows", [1, 19, 200])
def test_feed_forward_of_a_gguf_file(tmp_path, rows):
    """The operators as a layer uses them: each step against its formula on what the step
    before it gave, and the block's output the last step's."""
    path = tmp_path / "m.gguf"
    _gguf_file(path)
    ffn = fp8.Fp8FeedForward.from_gguf(path, 3)
    assert ffn.eps == pytest.approx(1e-6)
    x, r = rows_of(rows, 256, torch.bfloat16, 11), rows_of(rows, 256, torch.bfloat16, 12)
    y, h = ffn(x, r)
    want = (x.float() + r.float()).bfloat16()
    assert torch.equal(h, want)
    q, _ = fp8.rms_norm_fp8(x, ffn.norm, ffn.eps, residual=r)
    check_rows(q, norm_plain(want, ffn.norm, ffn.eps))
    both = fp8.matmul_fp8(q, ffn.gate_up)
    check_product(both, q, ffn.gate_up)
    s = fp8.quantize_fp8(both[:, 384:], gate=both[:, :384])
    g, u = both[:, :384].cpu().double().numpy(), both[:, 384:].cpu().double().numpy()
    check_rows(s, g / (1 + np.exp(-g)) * u)
    check_product(y, s, ffn.down)
    # the weights are the file's: gate rows first, then up
    from gguf import GGUFReader
    t = {t.name: t for t in GGUFReader(path).tensors}
    for i, (name, fmt) in enumerate((("ffn_gate", "Q4_K"), ("ffn_up", "Q5_K"))):
        codes, scales = quantize_plain(oracle_values(fmt, np.array(t[f"blk.3.{name}.weight"].data).reshape(-1).view(np.uint8), 384, 256), 128)
        assert same_codes(bytes_of(ffn.gate_up.codes)[384 * i:384 * (i + 1)], codes)
        assert np.array_equal(bytes_of(ffn.gate_up.scales)[3 * i:3 * (i + 1)], scales)


def test_linear_of_a_gguf_file_with_bias_and_heads(tmp_path):
    path = tmp_path / "m.gguf"
    _gguf_file(path)
    from gguf import GGUFReader
    t = {t.name: t for t in GGUFReader(path).tensors}
    lin = fp8.Fp8Linear.from_gguf(t["blk.3.attn_q.weight"], t["blk.3.attn_q.bias"], heads=4)
    b = permute(np.array(t["blk.3.attn_q.bias"].data, np.float32).reshape(-1, 1), 4).reshape(-1)
    assert np.array_equal(lin.bias.cpu().numpy(), b)
    codes, scales = quantize_plain(permute(oracle_values("Q6_K", np.array(t["blk.3.attn_q.weight"].data).reshape(-1).view(np.uint8), 256, 256), 4), 128)
    assert same_codes(bytes_of(lin.weight.codes), codes) and np.array_equal(bytes_of(lin.weight.scales), scales)
    x = rows_of(33, 256, torch.float16, 13)
    out = lin(x, dtype=torch.float32)
    check_product(out, fp8.quantize_fp8(x), lin.weight, lin.bias)
    assert torch.equal(lin(fp8.quantize_fp8(x), dtype=torch.float32), out)


@pytest.mark.parametrize("rows", [1, 150, 600])
def test_captured_and_replayed(tmp_path, rows):
    """The block in a CUDA graph: replayed on new inputs it gives what eager calls give."""
    path = tmp_path / "m.gguf"
    _gguf_file(path)
    ffn = fp8.Fp8FeedForward.from_gguf(path, 3)
    x, r = rows_of(rows, 256, torch.bfloat16, 14), rows_of(rows, 256, torch.bfloat16, 15)
    ffn(x, r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = ffn(x, r)
    for seed in (16, 17):
        x.copy_(rows_of(rows, 256, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone(), h.clone()
        want = ffn(x, r)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_with_copies_and_a_fork():
    """A graph in which these kernels follow a copy, a fill, each other on two streams, and the
    join of both."""
    a, w = operands(200, 512, 1024, 60)
    _, v = operands(1, 1024, 512, 61)
    host = torch.randn(200, 1024).bfloat16().pin_memory()
    x = torch.empty(200, 1024, dtype=torch.bfloat16, device=DEV)
    ones = torch.ones(1024, device=DEV)

    def work(side):
        main = torch.cuda.current_stream()
        x.copy_(host, non_blocking=True)
        q = fp8.rms_norm_fp8(x, ones)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            left = fp8.matmul_fp8(q, w)
            left_q = fp8.quantize_fp8(left)
        right = fp8.matmul_fp8(q, w, dtype=torch.float16)
        right.zero_()
        right_q = fp8.quantize_fp8(right)
        main.wait_stream(side)
        both = fp8.matmul_fp8(left_q, v, dtype=torch.float32)
        return both, fp8.matmul_fp8(right_q, v), left

    side = torch.cuda.Stream()
    want = [t.clone() for t in work(side)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(side)
    for _ in range(3):
        for t in got:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for g, t in zip(got, want):
            assert torch.equal(g, t)


@pytest.mark.parametrize("m", [1, 40, 300, 1500])
def test_back_to_back_on_the_same_buffers(m):
    """Kernels of this module begin under the one before them: a chain that writes what the last
    link still reads, over and over on the same buffers, gives what single calls give."""
    w1, w2 = operands(1, 512, 1024, 40)[1], operands(1, 1024, 256, 41)[1]
    norm = torch.randn(1024, device=DEV)
    x0 = rows_of(m, 1024, torch.bfloat16, 42)

    def links(x, out, wait):
        q, h = fp8.rms_norm_fp8(x, norm, residual=x, **({} if out is None else {"out": out[0], "sum_out": out[1]}))
        wait()
        both = fp8.matmul_fp8(q, w1, out=None if out is None else out[2])
        wait()
        s = fp8.quantize_fp8(both[:, 256:], gate=both[:, :256], out=None if out is None else out[3])
        wait()
        fp8.matmul_fp8(s, w2, out=x)
        wait()
        return h

    x = x0.clone()
    want = []
    for _ in range(6):
        h = links(x, None, torch.cuda.synchronize)
        want.append((x.clone(), h.clone()))
    x = x0.clone()
    q = fp8.Fp8Rows(torch.empty(m, 1024, dtype=fp8.E4M3, device=DEV), torch.empty(m, 8, dtype=fp8.E8M0, device=DEV))
    s = fp8.Fp8Rows(torch.empty(m, 256, dtype=fp8.E4M3, device=DEV), torch.empty(m, 2, dtype=fp8.E8M0, device=DEV))
    out = (q, torch.empty_like(x), torch.empty(m, 512, dtype=torch.bfloat16, device=DEV), s)
    got = []
    for _ in range(6):
        h = links(x, out, lambda: None)
        got.append((x.clone(), h.clone()))
    for (xa, ha), (xb, hb) in zip(got, want):
        assert torch.equal(xa, xb) and torch.equal(ha, hb)
    # and with nothing but these kernels on the stream between the copies out
    x.copy_(x0)
    for _ in range(6):
        links(x, out, lambda: None)
    assert torch.equal(x, want[-1][0])


@pytest.mark.parametrize("m", [1, 24, 600])
def test_two_streams_at_once(m):
    """Products on two streams share nothing: each gives what it gives alone."""
    pairs = [operands(m, 1536, 2048, s) for s in (20, 21)]
    want = [fp8.matmul_fp8(*p) for p in pairs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fp8.matmul_fp8(*pairs[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert torch.equal(g, want[i])


def test_a_wait_of_the_product_that_nothing_ends_gives_up(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    from llima_b200.build import ARCH, CSRC
    root = Path(__file__).resolve().parents[1]
    so = tmp_path / "libwait.so"
    subprocess.run([shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc", *ARCH, "-O2", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
                    f"-I{CSRC}", f"-I{root / 'include'}", "-o", str(so), str(root / "tests" / "cuda" / "tensor_wait_timeout.cu")],
                   check=True, capture_output=True)
    status, waited = ctypes.c_int(-1), ctypes.c_ulonglong(0)
    assert ctypes.CDLL(str(so)).run_wait_never(ctypes.byref(status), ctypes.byref(waited)) == 0
    assert status.value == 0 and 0.9e9 <= waited.value <= 5e9


def test_no_kernel_reported_an_error():
    flags = ctypes.c_uint32(99)
    N.check(N.lib().gq_kernel_errors(0, 0, ctypes.byref(flags)), "gq_kernel_errors")
    assert flags.value == 0
