"""The 8-bit float entry points where there is no device: an error code, never the process's end.
Each runs in a child process that sees no GPU, so that its operands' addresses are never read."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CALLS = {
    "convert boxes": "lib.gq_convert_fp8(ctypes.byref(N.Tensor(type=12, rows=130, cols=512, src=A, src_bytes=130 * 288, codes=B)), C, None)",
    "convert rows": "lib.gq_convert_fp8(ctypes.byref(N.Tensor(type=8, rows=130, cols=96, src=A, src_bytes=130 * 102, codes=B)), C, None)",
    "convert floats": "lib.gq_convert_fp8(ctypes.byref(N.Tensor(type=0, rows=130, cols=96, src=A, src_bytes=130 * 384, codes=B)), C, None)",
    "norm": "lib.gq_rms_norm_fp8(30, A, 256, B, 256, C, 1e-5, 4000, 256, D, 256, E, 256, F, 2, None)",
    "long norm": "lib.gq_rms_norm_fp8(30, A, 32768, None, 0, B, 1e-5, 4, 32768, None, 0, C, 32768, D, 256, None)",
    "rows": "lib.gq_quantize_fp8(1, A, 96, B, 96, 3, 96, C, 96, D, 1, None)",
    "product of a token": "lib.gq_matmul_fp8(A, 256, B, 2, C, 256, D, 2, None, 1, 7, 256, 30, E, 7, None)",
    "product of a prompt": "lib.gq_matmul_fp8(A, 4096, B, 32, C, 4096, D, 32, None, 2048, 8192, 4096, 0, E, 8192, None)",
    "product over nothing": "lib.gq_matmul_fp8(None, 0, None, 0, None, 0, None, 0, None, 3, 7, 0, 30, A, 7, None)",
}


@pytest.mark.parametrize("name", CALLS)
def test_status_without_a_device(name):
    code = f"import ctypes\nfrom llima_b200 import _native as N\nlib = N.lib()\nA, B, C, D, E, F = (i << 32 for i in range(1, 7))\nprint('status', {CALLS[name]})"
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=str(ROOT))
    r = subprocess.run([sys.executable, "-c", code], env=env, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, f"ended with {r.returncode}: {r.stderr[-300:]}"
    assert r.stdout.split() == ["status", "-6"]
