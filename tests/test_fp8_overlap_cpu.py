"""Outputs that share memory with another operand are refused, before any CUDA call; those that only
lie between the rows of one are not (held to a count of shared bytes)."""
import ctypes
import os
import random
import subprocess
import sys
from pathlib import Path

from llima_b200 import _native as N

ARG = -5
A, B, C, D, E, F = (i << 32 for i in range(1, 7))     # addresses far apart that no call here reads
BF16 = 30


def norm(x=A, ld_x=256, residual=B, ld_r=256, weight=C, rows=4, cols=256, out=D, ld_s=256, codes=E, ld_c=256, scales=F, ld_sc=2):
    return N.lib().gq_rms_norm_fp8(BF16, x, ld_x, residual, ld_r, weight, 1e-5, rows, cols, out, ld_s, codes, ld_c, scales, ld_sc, None)


def test_norm():
    assert norm(out=A + 512) == ARG and norm(out=B - 512) == ARG            # a row further, a row before
    assert norm(out=A, ld_s=512) == ARG and norm(out=A + 16) == ARG
    assert norm(codes=A) == ARG and norm(codes=B + 1024) == ARG and norm(codes=C) == ARG and norm(codes=D + 256) == ARG
    assert norm(scales=A + 3) == ARG and norm(scales=D) == ARG and norm(scales=E + 1) == ARG
    assert norm(out=C) == ARG
    assert norm(residual=None, out=None, codes=A) == ARG


def test_quantize():
    def call(x=A, gate=B, codes=C, scales=D):
        return N.lib().gq_quantize_fp8(BF16, x, 256, gate, 256, 4, 256, codes, 256, scales, 2, None)

    assert call(codes=A + 512) == ARG and call(codes=B) == ARG and call(scales=A) == ARG and call(scales=B + 100) == ARG
    assert call(scales=C + 1023) == ARG and call(gate=None, codes=A) == ARG


def test_matmul():
    def call(out=E, bias=F, ld_o=256):
        return N.lib().gq_matmul_fp8(A, 256, B, 2, C, 256, D, 2, bias, 5, 256, 256, BF16, out, ld_o, None)

    for operand in (A, B, C, D, F):
        assert call(out=operand) == ARG
    assert call(out=A + 256 * 4 + 240) == ARG and call(out=A - 16) == ARG and call(out=F + 1022) == ARG


def test_convert():
    def call(src=A, codes=B, scales=C):
        t = N.Tensor(type=8, rows=130, cols=512, src=src, src_bytes=130 * 544, codes=codes)
        return N.lib().gq_convert_fp8(ctypes.byref(t), scales, None)

    assert call(codes=A + 544 * 129) == ARG and call(scales=A) == ARG and call(scales=B + 130 * 512 - 1) == ARG


def test_against_a_count_of_bytes():
    """Random places of the sum beside x in one buffer, where no device is seen: a call that is not
    refused ends with the missing device."""
    code = "import sys\nsys.path.insert(0, 'tests')\nimport test_fp8_overlap_cpu as t\nt.random_places()"
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=str(root)),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def random_places():
    rng = random.Random(1)
    refused = 0
    for _ in range(3000):
        rows, cols = rng.choice([1, 2, 3, 7]), 32 * rng.randint(1, 4)
        ld = cols + 8 * rng.randint(0, 40)
        at = 16 * rng.randint(-rows * ld // 8 - 20, rows * ld // 8 + 20)

        def cells(base, pitch):
            return {base + 2 * (r * pitch + c) for r in range(rows) for c in range(0, cols, 8)}

        shared = bool(cells(0, ld) & cells(at, ld)) and at != 0
        got = norm(x=A, ld_x=ld, rows=rows, cols=cols, out=A + at, ld_s=ld)
        assert got == (ARG if shared else -6), (rows, cols, ld, at, got)
        refused += shared
    assert 500 < refused < 2500
