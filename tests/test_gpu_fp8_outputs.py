"""What lies beside an output that is a range of a wider tensor stays as it was: rows that start on 16
bytes and end off them, for tiles of every kernel."""
import pytest
import torch

from llima_b200 import fp8
from test_gpu_fp8 import DEV, FLOATS, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k", [(3, 416), (50, 2080), (130, 96), (600, 2080), (1300, 2080)])
@pytest.mark.parametrize("n", [2593, 2594, 2597, 2599, 2600, 2604, 333])
def test_columns_beside_the_output_stay(n, m, k, dtype):
    a, w = operands(m, n, k, m + n)
    want = fp8.matmul_fp8(a, w, dtype=dtype)
    for left, pitch in ((8, 8 * -(-(n + 24) // 8)), (8, 8 * -(-(n + 8) // 8)), (3, n + 5)):
        wide = torch.full((m + 2, pitch), 7.0, dtype=dtype, device=DEV)
        out = wide[1:-1, left:left + n]
        fp8.matmul_fp8(a, w, out=out)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert bool((wide == 7.0).all())


def test_outputs_between_the_rows_of_an_input():
    """Ranges of columns of one tensor share no byte: they are taken."""
    wide = torch.randn(6, 1024, device=DEV).bfloat16()
    x, s = wide[:, :512], wide[:, 512:]
    want = (x.float() + x.float()).bfloat16()
    left = wide[:, :512].clone()
    q, h = fp8.rms_norm_fp8(x, torch.ones(512, device=DEV), residual=x, sum_out=s)
    assert h is s and torch.equal(s, want) and torch.equal(wide[:, :512], left)
    buf = torch.zeros(6, 1024, dtype=torch.uint8, device=DEV)
    out = fp8.Fp8Rows(buf[:, :512].view(fp8.E4M3), buf[:, 512:516].view(fp8.E8M0))
    fp8.quantize_fp8(x, out=out)
    ref = fp8.quantize_fp8(left)
    assert torch.equal(out.codes.view(torch.uint8), ref.codes.view(torch.uint8)) and not buf[:, 516:].any()
    assert torch.equal(out.scales.view(torch.uint8), ref.scales.view(torch.uint8))


def test_outputs_over_an_operand_are_refused():
    from llima_b200 import _native as N
    x = torch.randn(6, 512, device=DEV).bfloat16()
    ones = torch.ones(512, device=DEV)
    kept = x.clone()
    with pytest.raises(N.GqError):
        fp8.rms_norm_fp8(x[:-1], ones, residual=x[:-1].clone(), sum_out=x[1:])
    flat = x.view(torch.uint8)
    with pytest.raises(N.GqError):
        fp8.quantize_fp8(x, out=fp8.Fp8Rows(flat[:, :512].view(fp8.E4M3), torch.empty(6, 4, dtype=fp8.E8M0, device=DEV)))
    a, w = operands(6, 128, 512, 1)
    with pytest.raises(N.GqError):
        fp8.matmul_fp8(a, w, out=a.codes.view(torch.bfloat16)[:, :128])
    assert torch.equal(x, kept)
