"""Argument checks of the block-scaled 8-bit float entry points: they come before any CUDA
call, so they run without a GPU."""
import ctypes

import pytest
import torch

from llima_b200 import _native as N
from llima_b200 import fp8

SIZE, ALIGN, NULL, TYPE, ARG = -2, -3, -4, -1, -5
F32, F16, BF16 = 0, 1, 30
P = 0x1000   # a 16-byte-aligned address that no call here may read


def _convert(scales=P, **fields):
    t = N.Tensor(**{"type": 12, "rows": 130, "cols": 512, "src": P, "src_bytes": 130 * 288, "codes": P, **fields})
    return N.lib().gq_convert_fp8(ctypes.byref(t), scales, None)


def test_convert_refusals():
    assert N.lib().gq_convert_fp8(None, P, None) == NULL
    assert _convert(type=99) == TYPE
    assert _convert(cols=500) == SIZE
    assert _convert(rows=-1) == SIZE
    assert _convert(src_bytes=130 * 288 - 1) == SIZE
    assert _convert(type=F32, cols=33, src_bytes=1 << 20) == SIZE       # 32-column granularity for float types too
    assert _convert(perm_heads=3) == ARG
    assert _convert(perm_heads=-1) == ARG
    assert _convert(src=None) == NULL and _convert(codes=None) == NULL and _convert(scales=None) == NULL
    assert _convert(src=P + 8) == ALIGN and _convert(codes=P + 8) == ALIGN
    assert _convert(rows=0, src=None, codes=None, scales=None) == 0
    assert _convert(rows=1 << 62, cols=1 << 32) == SIZE


def _norm(dtype=BF16, x=P, ld_x=256, residual=P, ld_r=256, weight=P, rows=4, cols=256, out=P, ld_s=256, codes=P, ld_c=256,
          scales=P, ld_sc=2):
    return N.lib().gq_rms_norm_fp8(dtype, x, ld_x, residual, ld_r, weight, 1e-5, rows, cols, out, ld_s, codes, ld_c, scales,
                                   ld_sc, None)


def test_rms_norm_refusals():
    assert _norm(dtype=12) == TYPE
    assert _norm(cols=250) == SIZE and _norm(rows=-1) == SIZE and _norm(rows=1 << 31) == SIZE
    assert _norm(ld_x=255) == SIZE and _norm(ld_r=255) == SIZE and _norm(ld_s=255) == SIZE
    assert _norm(ld_c=255) == SIZE and _norm(ld_sc=1) == SIZE
    assert _norm(x=None) == NULL and _norm(weight=None) == NULL and _norm(out=None) == NULL
    assert _norm(codes=None) == NULL and _norm(scales=None) == NULL
    for name in ("x", "residual", "weight", "out", "codes"):
        assert _norm(**{name: P + 8}) == ALIGN
    assert _norm(ld_x=260) == ALIGN and _norm(ld_r=260) == ALIGN and _norm(ld_s=260) == ALIGN and _norm(ld_c=264) == ALIGN
    assert _norm(rows=0, x=None) == 0 and _norm(cols=0, ld_sc=0, x=None) == 0


def _quantize(dtype=F16, x=P, ld_x=96, gate=P, ld_g=96, rows=3, cols=96, codes=P, ld_c=96, scales=P, ld_sc=1):
    return N.lib().gq_quantize_fp8(dtype, x, ld_x, gate, ld_g, rows, cols, codes, ld_c, scales, ld_sc, None)


def test_quantize_refusals():
    assert _quantize(dtype=8) == TYPE
    assert _quantize(cols=95) == SIZE and _quantize(rows=-3) == SIZE
    assert _quantize(ld_x=95) == SIZE and _quantize(ld_g=95) == SIZE and _quantize(ld_c=95) == SIZE and _quantize(ld_sc=0) == SIZE
    assert _quantize(x=None) == NULL and _quantize(codes=None) == NULL and _quantize(scales=None) == NULL
    assert _quantize(x=P + 2) == ALIGN and _quantize(gate=P + 4) == ALIGN and _quantize(codes=P + 1) == ALIGN
    assert _quantize(ld_x=100) == ALIGN and _quantize(ld_g=98) == ALIGN and _quantize(ld_c=104) == ALIGN
    assert _quantize(rows=0) == 0


def _matmul(a=P, ld_a=256, sa=P, ld_sa=2, b=P, ld_b=256, sb=P, ld_sb=2, bias=None, m=5, n=7, k=256, dtype=BF16, out=P, ld_o=7):
    return N.lib().gq_matmul_fp8(a, ld_a, sa, ld_sa, b, ld_b, sb, ld_sb, bias, m, n, k, dtype, out, ld_o, None)


def test_matmul_refusals():
    assert _matmul(dtype=2) == TYPE
    assert _matmul(k=250) == SIZE and _matmul(m=-1) == SIZE and _matmul(n=-1) == SIZE and _matmul(k=-32) == SIZE
    assert _matmul(m=1 << 31) == SIZE and _matmul(n=1 << 31, ld_o=1 << 31) == SIZE
    assert _matmul(ld_a=255) == SIZE and _matmul(ld_b=255) == SIZE and _matmul(ld_o=6) == SIZE
    assert _matmul(ld_sa=1) == SIZE and _matmul(ld_sb=1) == SIZE
    assert _matmul(ld_a=1 << 40) == SIZE
    for name in ("a", "sa", "b", "sb", "out"):
        assert _matmul(**{name: None}) == NULL
    assert _matmul(a=P + 8) == ALIGN and _matmul(b=P + 8) == ALIGN and _matmul(out=P + 1) == ALIGN and _matmul(bias=P + 2) == ALIGN
    assert _matmul(ld_a=264) == ALIGN and _matmul(ld_b=264) == ALIGN
    assert _matmul(m=0, a=None) == 0 and _matmul(n=0, ld_o=0) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(4, 128)
    with pytest.raises(TypeError):
        fp8.quantize_fp8(x)
    with pytest.raises(TypeError):
        fp8.rms_norm_fp8(x, torch.ones(128))
    with pytest.raises(TypeError):
        fp8.convert_fp8_device("Q8_0", torch.zeros(34, dtype=torch.uint8), 1, 32)
    c, s = torch.zeros(4, 128).to(fp8.E4M3), torch.ones(4, 1).to(fp8.E8M0)
    with pytest.raises(TypeError):
        fp8.matmul_fp8(fp8.Fp8Rows(c, s), fp8.Fp8Weight(c, s[:1]))
