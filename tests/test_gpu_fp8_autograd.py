"""What autograd is told: outputs have no history, and a tensor written through out= or sum_out= counts
as changed."""
import pytest
import torch

from llima_b200 import fp8
from test_gpu_fp8 import operands, rows_of

pytestmark = pytest.mark.gpu


def test_a_saved_tensor_that_is_written_over_fails_its_backward_pass():
    a, w = operands(4, 128, 256, 1)
    ones = torch.ones(256, device="cuda")
    for write in (lambda t: fp8.matmul_fp8(a, w, out=t[:, :128]), lambda t: fp8.rms_norm_fp8(t, ones, residual=t, sum_out=t)):
        saved = torch.randn(4, 256, device="cuda")
        leaf = torch.ones(4, 256, device="cuda", requires_grad=True)
        loss = (leaf * saved).sum()
        write(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_versions_of_what_is_written():
    x = rows_of(4, 256, torch.bfloat16, 1)
    q = fp8.Fp8Rows(torch.empty(4, 256, dtype=fp8.E4M3, device="cuda"), torch.empty(4, 2, dtype=fp8.E8M0, device="cuda"))
    raw = torch.zeros(4 * 8 * 34, dtype=torch.uint8, device="cuda")
    v = fp8.Fp8Weight(torch.empty(4, 256, dtype=fp8.E4M3, device="cuda"), torch.empty(1, 2, dtype=fp8.E8M0, device="cuda"))
    for out, call in ((q, lambda: fp8.quantize_fp8(x, out=q)), (q, lambda: fp8.rms_norm_fp8(x, torch.ones(256, device="cuda"), out=q)),
                      (v, lambda: fp8.convert_fp8_device("Q8_0", raw, 4, 256, out=v))):
        before = [t._version for t in out] + [x._version]
        call()
        assert [t._version for t in out] + [x._version] == [before[0] + 1, before[1] + 1, before[2]]


def test_under_no_grad_and_inference_mode():
    a, w = operands(4, 128, 256, 2)
    want = fp8.matmul_fp8(a, w)
    x = rows_of(4, 256, torch.float32, 1).requires_grad_()
    with torch.no_grad():
        assert not fp8.quantize_fp8(x).codes.requires_grad
    with torch.inference_mode():
        out = torch.empty(4, 128, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(fp8.matmul_fp8(a, w, out=out), want)
        assert fp8.quantize_fp8(x).codes.shape == (4, 256)
    p = torch.nn.Parameter(torch.ones(256, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradients"):
        fp8.rms_norm_fp8(x.detach(), p)
    fp8.rms_norm_fp8(x.detach(), p.detach())
