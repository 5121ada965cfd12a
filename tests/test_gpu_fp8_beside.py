"""Products beside other work that takes tensor memory: kernels of another library on a second stream."""
import pytest
import torch

from llima_b200 import fp8
from test_gpu_fp8 import operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (13, 4096, 4096), (60, 1536, 2048), (120, 1024, 4096), (600, 2600, 2080)])
def test_beside_products_of_another_stream(m, n, k):
    """Split over clusters, one CTA per tile, and pairs: each gives what it gives alone, and so does
    the other stream's."""
    a, w = operands(m, n, k, 1)
    x, y = torch.randn(2048, 2048, device="cuda").bfloat16(), torch.randn(2048, 2048, device="cuda").bfloat16()
    small = x[:64].contiguous()
    want, other, few = fp8.matmul_fp8(a, w), x @ y, small @ y
    torch.cuda.synchronize()
    mine, theirs = torch.cuda.Stream(), torch.cuda.Stream()
    got, beside = [], []
    for _ in range(40):
        with torch.cuda.stream(theirs):
            beside.append((x @ y, small @ y))
        with torch.cuda.stream(mine):
            got.append(fp8.matmul_fp8(a, w))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    assert all(torch.equal(b, other) and torch.equal(f, few) for b, f in beside)
