"""Calls from host threads: a thread's first CUDA work may be any of them, and two at once share nothing."""
import threading

import pytest
import torch

from llima_b200 import fp8
from llima_b200.synth import gen_tensor_bytes
from test_gpu_fp8 import operands, rows_of

pytestmark = pytest.mark.gpu


def in_thread(*calls):
    """The calls' results, each made as the first work of a thread of its own, all at once."""
    results = [None] * len(calls)

    def work(i):
        try:
            results[i] = calls[i]()
        except Exception as e:
            results[i] = e

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in results:
        if isinstance(r, Exception):
            raise r
    return results


@pytest.mark.parametrize("m,n,k", [(3, 256, 512), (600, 2600, 416), (600, 2597, 416)])
def test_product_first_in_a_thread(m, n, k):
    a, w = operands(m, n, k, 1)
    want = fp8.matmul_fp8(a, w)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    in_thread(lambda: fp8.matmul_fp8(a, w, out=out))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("fmt,heads", [("Q8_0", 0), ("Q4_K", 2), ("Q6_K", 0), ("F32", 0)])
def test_conversion_first_in_a_thread(fmt, heads):
    raw = torch.from_numpy(gen_tensor_bytes(fmt, 256 * 2048, 1).copy()).cuda()
    want = fp8.convert_fp8_device(fmt, raw, 256, 2048, heads)
    out = fp8.Fp8Weight(torch.zeros_like(want.codes.view(torch.uint8)).view(fp8.E4M3), torch.zeros_like(want.scales.view(torch.uint8)).view(fp8.E8M0))
    torch.cuda.synchronize()
    in_thread(lambda: fp8.convert_fp8_device(fmt, raw, 256, 2048, heads, out=out))
    torch.cuda.synchronize()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(out, want))


def test_rows_first_in_a_thread():
    x, w = rows_of(5, 512, torch.bfloat16, 1), torch.ones(512, device="cuda")
    want = fp8.quantize_fp8(x), fp8.rms_norm_fp8(x, w)
    out = [fp8.Fp8Rows(torch.empty_like(q.codes), torch.empty_like(q.scales)) for q in want]
    torch.cuda.synchronize()
    in_thread(lambda: fp8.quantize_fp8(x, out=out[0]), lambda: fp8.rms_norm_fp8(x, w, out=out[1]))
    torch.cuda.synchronize()
    for q, v in zip(out, want):
        assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(q, v))


def test_threads_at_once_on_streams_of_their_own():
    """Four threads, each a chain of all the operators on its own stream, over and over."""
    raw = torch.from_numpy(gen_tensor_bytes("Q8_0", 256 * 512, 2).copy()).cuda()
    norm = torch.randn(512, device="cuda")
    xs = [rows_of(m, 512, torch.bfloat16, m) for m in (1, 40, 300, 700)]

    def chain(x):
        w = fp8.convert_fp8_device("Q8_0", raw, 256, 512)
        y = fp8.matmul_fp8(fp8.rms_norm_fp8(x, norm), w)
        return fp8.quantize_fp8(y[:, 128:], gate=y[:, :128])

    want = [chain(x) for x in xs]
    torch.cuda.synchronize()

    def work(x):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [chain(x) for _ in range(20)]
        s.synchronize()
        return got

    for got, ref in zip(in_thread(*[lambda x=x: work(x) for x in xs]), want):
        for q in got:
            assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(q, ref))
