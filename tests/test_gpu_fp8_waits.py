"""The answer of the product's bounded wait is the warp's, not a lane's."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_a_warp_gets_one_answer(tmp_path):
    from llima_b200.build import ARCH, CSRC
    root = Path(__file__).resolve().parents[1]
    so = tmp_path / "liblanes.so"
    subprocess.run([shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc", *ARCH, "-O2", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
                    f"-I{CSRC}", f"-I{root / 'include'}", "-o", str(so), str(root / "tests" / "cuda" / "tensor_wait_lanes.cu")],
                   check=True, capture_output=True)
    answers, elected = (ctypes.c_int * 64)(), (ctypes.c_int * 3)()
    assert ctypes.CDLL(str(so)).run_lanes(answers, elected) == 0
    assert list(answers) == [0] * 32 + [1] * 32
    assert list(elected) == [1, 1, 3]


def test_check_kernels_after_ordinary_work():
    import torch
    from llima_b200 import fp8
    x = fp8.quantize_fp8(torch.randn(300, 512, device="cuda"))
    w = fp8.convert_fp8_device("F32", torch.randn(512 * 512, device="cuda").view(torch.uint8), 512, 512)
    fp8.matmul_fp8(x, w)
    for device in (None, 0, "cuda", torch.device("cuda", 0)):
        fp8.check_kernels(device)
