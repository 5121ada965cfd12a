"""Operands that a gradient is asked for are refused, before anything else is looked at: no GPU is
needed to see it."""
import pytest
import torch

from llima_b200 import fp8


def f8(*shape):
    return torch.zeros(*shape).to(fp8.E4M3), torch.ones(shape[0], 1).to(fp8.E8M0)


def calls():
    x, w = torch.zeros(4, 128), torch.ones(128)
    leaf, wleaf = x.clone().requires_grad_(), w.clone().requires_grad_()
    q, weight = fp8.Fp8Rows(*f8(4, 128)), fp8.Fp8Weight(*f8(4, 128))
    yield "x", lambda: fp8.quantize_fp8(leaf)
    yield "not a leaf", lambda: fp8.quantize_fp8(leaf * 2)
    yield "gate", lambda: fp8.quantize_fp8(x, gate=leaf)
    yield "norm x", lambda: fp8.rms_norm_fp8(leaf, w)
    yield "norm weight", lambda: fp8.rms_norm_fp8(x, wleaf)
    yield "residual", lambda: fp8.rms_norm_fp8(x, w, residual=leaf)
    yield "sum_out", lambda: fp8.rms_norm_fp8(x, w, residual=x, sum_out=leaf)
    yield "bias", lambda: fp8.matmul_fp8(q, weight, bias=torch.ones(4, requires_grad=True))
    yield "out", lambda: fp8.matmul_fp8(q, weight, out=torch.zeros(4, 4, requires_grad=True))
    yield "linear", lambda: fp8.Fp8Linear(weight)(leaf)
    yield "feed forward", lambda: fp8.Fp8FeedForward(w, weight, weight)(leaf, x)


@pytest.mark.parametrize("name,call", list(calls()), ids=lambda v: v if isinstance(v, str) else "")
def test_gradients_are_refused(name, call):
    with pytest.raises(RuntimeError, match="no gradients"):
        call()
    with torch.no_grad(), pytest.raises(TypeError, match="CUDA"):
        call()      # on to the next check
