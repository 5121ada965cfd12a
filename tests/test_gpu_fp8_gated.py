"""silu(gate) * x over the whole range of its exponential, against 64 bits.

The kernel takes exp(-|g| / 2) = 2^h, h = -|g| / (2 ln 2).  The product and the constant put h off
by at most 1.25 * 2^-24 |h|, so the square of the exponential by 1.25 * 2^-24 |g|.  The hardware's
exponential is off by 2^-22 in each of two factors, its reciprocal by 2^-23, and each of four
roundings by 2^-24; in the sum with 1 these errors cancel in part.  Together the f32 value is off
by less than |g| 2^-23 + 2^-20 relative for |g| < 174, so a code's value is within half a step of
the exact one (2^-4 relative, or 2^-10 of the scale below the normal range) plus that."""
import numpy as np
import pytest
import torch

from llima_b200 import fp8
from test_gpu_fp8 import FLOATS, exponent

pytestmark = pytest.mark.gpu


def check(x, g):
    q = fp8.quantize_fp8(x, gate=g)
    xd, gd = x.cpu().double().numpy(), g.cpu().double().numpy()
    y = xd * gd / (1 + np.exp(-gd))                 # 64 bits overflow at g = -709
    rows, cols = y.shape
    err = np.abs(gd) * 2.0 ** -23 + 2.0 ** -20
    # y is held in f32: 0 below 2^-150
    low, high = (exponent((np.abs(y) * (1 + d)).reshape(rows, cols // 128, 128).max(2).astype(np.float32)) for d in (-err, err))
    e = q.scales.view(torch.uint8).cpu().numpy().astype(np.int64) - 127
    assert np.all((e == low) | (e == high))
    s = np.repeat(np.ldexp(1.0, e.astype(np.int32)), 128, 1)
    off = np.abs(q.codes.cpu().double().numpy() * s - y)
    limit = np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) + np.abs(y) * err + 2.0 ** -149
    assert np.all(off <= limit), np.max(off / limit)
    return q


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gate", [-103.5, -95.0, -88.7, -88.0, -87.4, -80.0, -40.0, -1e-3, 0.0, 3.0, 87.5, 200.0])
@pytest.mark.parametrize("size", [1.0, 3e4])
def test_blocks_of_one_gate(gate, size, dtype):
    """Every gate of a block near one value: the scale follows it however small it makes the block."""
    g = (torch.full((3, 256), gate, device="cuda") + torch.linspace(0, 0.25, 256, device="cuda")).to(dtype)
    x = torch.randn(3, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * size
    q = check(x.to(dtype).clamp(-6e4, 6e4), g)
    if size * abs(gate) * np.exp(min(gate, 0)) > 1e-36:
        assert bool((q.codes.float() != 0).any(1).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_gates_of_large_values(dtype):
    """Gates down to -170, whose quotients f32 cannot hold by themselves, times values up to 2e36."""
    g = torch.linspace(-170, 90, 64 * 128, device="cuda").reshape(64, 128).to(dtype)
    for size in (1.0, 1e20, 5e35):
        check((torch.randn(64, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * size).to(dtype), g)


def test_gates_that_are_not_finite():
    g = torch.ones(2, 128, device="cuda")
    g[0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    g[1, 0], g[1, 1] = 3e38, -3e38
    c = fp8.quantize_fp8(torch.ones(2, 128, device="cuda"), gate=g).codes.float().cpu()
    assert torch.isnan(c[0, :3]).all() and not torch.isnan(c[0, 3:]).any() and not torch.isnan(c[1]).any()
    assert float(c[0, 3]) != 0 and float(c[1, 0]) == 224 and float(c[1, 1]) == 0


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("strided", [False, True])
def test_far_gates_among_ordinary_ones(dtype, strided):
    """Some lanes of a warp with far gates and some without, on rows that start on 32 bytes and off
    them, with a ragged last block; and a block of far gates beside ordinary blocks."""
    gen = torch.Generator("cuda").manual_seed(3)
    rows, cols = 37, 416
    pad = 16 // torch.empty(0, dtype=dtype).element_size() if strided else 0
    wide = torch.zeros(2, rows, cols + 2 * pad, dtype=dtype, device="cuda")
    x, g = wide[0, :, pad:pad + cols], wide[1, :, pad:pad + cols]
    x.copy_(torch.randn(rows, cols, device="cuda", generator=gen))
    gates = torch.randn(rows, cols, device="cuda", generator=gen) * 4
    far = torch.rand(rows, cols, device="cuda", generator=gen) < 0.02
    g.copy_(torch.where(far, -87.0 - 10 * torch.rand(rows, cols, device="cuda", generator=gen), gates))
    g[5, 128:256] = -89
    g[6, 384:] = -88
    q = fp8.quantize_fp8(x, gate=g)
    pd = torch.nn.functional.pad
    whole = check(pd(x, (0, 512 - cols)), pd(g, (0, 512 - cols)))
    assert torch.equal(q.codes.view(torch.uint8), whole.codes.view(torch.uint8)[:, :cols])
    assert torch.equal(q.scales.view(torch.uint8), whole.scales.view(torch.uint8))
    assert bool((q.codes.float()[5, 128:256] != 0).any()) and bool((q.codes.float()[6, 384:] != 0).any())
