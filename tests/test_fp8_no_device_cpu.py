"""The 8-bit float entry points where there is no device: an error code, never the process's end.
Each runs in a child process that sees no GPU, so that its operands' addresses are never read."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CALLS = {
    "convert boxes": "lib.gq_convert_fp8(ctypes.byref(N.Tensor(type=12, rows=130, cols=512, src=P, src_bytes=130 * 288, codes=P)), P, None)",
    "convert rows": "lib.gq_convert_fp8(ctypes.byref(N.Tensor(type=8, rows=130, cols=96, src=P, src_bytes=130 * 102, codes=P)), P, None)",
    "convert floats": "lib.gq_convert_fp8(ctypes.byref(N.Tensor(type=0, rows=130, cols=96, src=P, src_bytes=130 * 384, codes=P)), P, None)",
    "norm": "lib.gq_rms_norm_fp8(30, P, 256, P, 256, P, 1e-5, 4000, 256, P, 256, P, 256, P, 2, None)",
    "long norm": "lib.gq_rms_norm_fp8(30, P, 32768, None, 0, P, 1e-5, 4, 32768, None, 0, P, 32768, P, 256, None)",
    "rows": "lib.gq_quantize_fp8(1, P, 96, P, 96, 3, 96, P, 96, P, 1, None)",
    "product of a token": "lib.gq_matmul_fp8(P, 256, P, 2, P, 256, P, 2, None, 1, 7, 256, 30, P, 7, None)",
    "product of a prompt": "lib.gq_matmul_fp8(P, 4096, P, 32, P, 4096, P, 32, None, 2048, 8192, 4096, 0, P, 8192, None)",
    "product over nothing": "lib.gq_matmul_fp8(None, 0, None, 0, None, 0, None, 0, None, 3, 7, 0, 30, P, 7, None)",
}


@pytest.mark.parametrize("name", CALLS)
def test_status_without_a_device(name):
    code = f"import ctypes\nfrom llima_b200 import _native as N\nlib, P = N.lib(), 0x1000\nprint('status', {CALLS[name]})"
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", PYTHONPATH=str(ROOT))
    r = subprocess.run([sys.executable, "-c", code], env=env, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, f"ended with {r.returncode}: {r.stderr[-300:]}"
    assert r.stdout.split() == ["status", "-6"]
