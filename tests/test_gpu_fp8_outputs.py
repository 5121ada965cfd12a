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
