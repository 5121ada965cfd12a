"""Every kernel of the product, at shapes that reach it (fp8_shapes, held to the choice on the CPU):
all output types, output rows on 16 bytes (boxes) and off them (plain stores), with a bias, into a
range of a wider tensor whose other values stay; and the pair kernel repeated, captured, chained and
on two streams.

Products of two e4m3 values are exact; sums of k of them in f32, each rounded or truncated, are off
by at most k 2^-23 sum|a b|, and the result by half a step of its type.  Together the errors of an f32
result are far smaller: 1.7e-6 of its norm was measured for sums of 112 blocks of 128 columns in one
piece.  They grow at least as fast as a piece, and none is longer than 48 blocks: 48 / 112 * 1.7e-6 <
8e-7.  A sum in one piece of 62 blocks or more is beyond that."""
import pytest
import torch

from fp8_shapes import ANY_TYPE, F32_ONLY, WIDE
from llima_b200 import fp8
from test_gpu_fp8 import DEV, FLOATS, operands, rows_of

pytestmark = pytest.mark.gpu


def values(q, rows_per_scale, rows=slice(None)):
    c = q.codes[rows].double()
    s = q.scales.double().repeat_interleave(rows_per_scale, 0)[:q.codes.shape[0]][rows]
    return c.mul_(s.repeat_interleave(128, 1)[:, :c.shape[1]])


def check(out, a, w, bias=None):
    m, k = a.codes.shape
    av = values(a, 1)
    half = torch.finfo(out.dtype).eps / 2
    step = 2048
    off2 = want2 = 0.0
    for n0 in range(0, out.shape[1], step):
        wv = values(w, 128, slice(n0, n0 + step))
        got, want = out[:, n0:n0 + step].double(), av @ wv.T
        bound = av.abs() @ wv.abs_().T
        if bias is not None:
            want += bias[n0:n0 + step].double()
            bound += bias[n0:n0 + step].double().abs()
        off = (got - want).abs()
        assert bool((off <= (k + 1) * 2.0 ** -23 * bound + half * want.abs() + torch.finfo(out.dtype).tiny).all()), f"columns from {n0}"
        off2, want2 = off2 + float((off * off).sum()), want2 + float((want * want).sum())
    far = (off2 / want2) ** 0.5
    assert far <= max(half, 8e-7), far


def run_both_layouts(m, n, k, dtype):
    a, w = operands(m, n, k, m + n)
    bias = torch.randn(n, device=DEV) * 0.1
    boxes = 16 // (2 if dtype != torch.float32 else 4)
    for left, pitch in ((boxes, -(-(n + 2 * boxes) // boxes) * boxes), (1, n + 2 + (n & 1))):
        wide = torch.full((m + 2, pitch), 7.0, dtype=dtype, device=DEV)
        out = wide[1:-1, left:left + n]
        fp8.matmul_fp8(a, w, bias=bias, out=out)
        check(out, a, w, bias)
        out.fill_(7.0)
        assert bool((wide == 7.0).all()), "beside the output"


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("choice,split,m,n,k", ANY_TYPE)
def test_every_kernel(choice, split, m, n, k, dtype):
    run_both_layouts(m, n, k, dtype)


@pytest.mark.parametrize("choice,split,m,n,k", F32_ONLY)
def test_long_sums_to_f32(choice, split, m, n, k):
    a, w = operands(m, n, k, 3)
    check(fp8.matmul_fp8(a, w, dtype=torch.float32), a, w)


@pytest.mark.parametrize("m,n,k", [(3, 19100, 12672), (20, 19100, 14336), (50, 19100, 14336), (2048, 4096, 14336), (600, 2597, 14336)])
def test_sums_in_pieces(m, n, k):
    """Sums of 99 and 112 blocks, which in one piece would be off by 1.5e-6 and more."""
    a, w = operands(m, n, k, 5)
    check(fp8.matmul_fp8(a, w, dtype=torch.float32), a, w)


def test_biased_f16_projection():
    a, w = operands(509, 4608, 3584, 6)
    bias = torch.randn(4608, device=DEV)
    check(fp8.matmul_fp8(a, w, bias=bias, dtype=torch.float16), a, w, bias)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("choice,split,m,n,k", WIDE)
def test_pairs_repeat_bit_for_bit(choice, split, m, n, k, dtype):
    a, w = operands(m, n, k, 8)
    first = fp8.matmul_fp8(a, w, dtype=dtype)
    check(first, a, w)
    for _ in range(5):
        assert torch.equal(fp8.matmul_fp8(a, w, dtype=dtype), first)


@pytest.mark.parametrize("choice,split,m,n,k", WIDE)
def test_nan_reaches_its_row_and_column_only(choice, split, m, n, k):
    a, w = operands(m, n, k, 4)
    plain = fp8.matmul_fp8(a, w, dtype=torch.float32)
    a.codes.view(torch.uint8)[2, 17] = 0x7F
    w.codes.view(torch.uint8)[n - 3, k - 1] = 0xFF
    a.scales.view(torch.uint8)[m - 1, 1] = 0xFF
    out = fp8.matmul_fp8(a, w, dtype=torch.float32)
    want = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    want[2] = want[m - 1] = True
    want[:, n - 3] = True
    assert torch.equal(torch.isnan(out), want) and torch.equal(out[~want], plain[~want])


def test_pairs_on_two_streams_at_once():
    pairs = [operands(m, n, k, 20) for _, _, m, n, k in WIDE[:4]]
    want = [fp8.matmul_fp8(*p) for p in pairs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [[] for _ in pairs]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fp8.matmul_fp8(*pairs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(4) for g in got[i])


def test_two_graphs_of_pairs_replayed_at_once():
    """Two captured products with operands and outputs of their own, replayed on two streams."""
    made = []
    for seed, (_, _, m, n, k) in enumerate(WIDE[:2]):
        a, w = operands(m, n, k, seed)
        want = fp8.matmul_fp8(a, w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = [fp8.matmul_fp8(a, w) for _ in range(4)]
        made.append((g, outs, want, torch.cuda.Stream(), a, w))      # a graph keeps no operand alive
    for _ in range(5):
        for g, outs, _, s, *_ in made:
            with torch.cuda.stream(s):
                for o in outs:
                    o.zero_()
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, outs, want, *_ in made for o in outs)


@pytest.mark.parametrize("m", [700, 1500])
def test_chain_of_pairs_on_the_same_buffers(m):
    """norm -> gate and up -> gated rows -> down, over and over on the same buffers, eager and
    captured, against single calls with a wait after each."""
    hidden, half = 2048, 1280
    w1, w2 = operands(1, 2 * half, hidden, 40)[1], operands(1, hidden, half, 41)[1]
    norm = torch.randn(hidden, device=DEV)
    x0 = rows_of(m, hidden, torch.bfloat16, 42)
    new = lambda r, c: fp8.Fp8Rows(torch.empty(r, c, dtype=fp8.E4M3, device=DEV), torch.empty(r, c // 128, dtype=fp8.E8M0, device=DEV))
    q, s, both, h = new(m, hidden), new(m, half), torch.empty(m, 2 * half, dtype=torch.bfloat16, device=DEV), torch.empty_like(x0)

    def links(x, wait=lambda: None):
        fp8.rms_norm_fp8(x, norm, residual=x, sum_out=h, out=q)
        wait()
        fp8.matmul_fp8(q, w1, out=both)
        wait()
        fp8.quantize_fp8(both[:, half:], gate=both[:, :half], out=s)
        wait()
        fp8.matmul_fp8(s, w2, out=x)
        wait()

    x, want = x0.clone(), []
    for _ in range(4):
        links(x, torch.cuda.synchronize)
        want.append(x.clone())
    x = x0.clone()
    for i in range(4):
        links(x)
        assert torch.equal(x, want[i])
    x.copy_(x0)
    for _ in range(4):
        links(x)
    assert torch.equal(x, want[3])
    graph = torch.cuda.CUDAGraph()
    x.copy_(x0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for _ in range(4):
            links(x)
    for _ in range(3):
        x.copy_(x0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want[3])
