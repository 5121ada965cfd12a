"""The matrix product's choice of kernel: that the table of shapes reaches every kernel, and that no
sum to an f32 output is taken in pieces longer than the stated ones."""
import subprocess
from pathlib import Path

import pytest

from fp8_shapes import ANY_TYPE, F32_ONLY, SMS, WIDE

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    exe = tmp_path_factory.mktemp("choice") / "choice"
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{ROOT / 'llima_b200' / 'csrc'}", "-o", str(exe),
                    str(ROOT / "tests" / "numerics" / "product_choice.cpp")], check=True)

    def run(rows):
        text = "\n".join(" ".join(str(int(v)) for v in r) for r in rows)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
        return [tuple(int(v) for v in line.split()) for line in out if line]

    return run


def test_the_table_is_what_is_chosen(choose):
    rows = [(m, n, k, f32, SMS) for _, _, m, n, k in ANY_TYPE + WIDE for f32 in (0, 1)] + [(m, n, k, 1, SMS) for _, _, m, n, k in F32_ONLY]
    want = [(c, s) for c, s, *_ in ANY_TYPE + WIDE for _ in (0, 1)] + [(c, s) for c, s, *_ in F32_ONLY]
    assert [(c, s) for c, s, _ in choose(rows)] == want


def test_the_table_reaches_every_kernel(choose):
    ms = [1, 2, 5, 13, 20, 33, 50, 70, 100, 130, 200, 257, 300, 509, 600, 1100, 1900, 8192]
    ns = [100, 333, 1024, 1152, 1536, 2600, 4096, 4608, 8200, 19100, 28672, 128256]
    ks = [32, 96, 416, 1056, 2080, 3584, 4128, 8480, 14336, 32768, 65536]
    for f32 in (0, 1):
        found = {(c, s) for c, s, _ in choose([(m, n, k, f32, SMS) for m in ms for n in ns for k in ks])}
        table = {(c, s) for c, s, *_ in ANY_TYPE + (F32_ONLY if f32 else [])}
        assert {c for c, _ in found} == {c for c, _ in table} == {16, 32, 64, 128, 256, 512}
        assert not f32 or {s for _, s in found} == {s for _, s in table}


def test_pieces_of_f32_sums_stay_short(choose):
    """At most 48 blocks of 128 columns to an accumulator, whatever k, rows and channels."""
    rows = [(m, n, k, 1, sms) for m in (1, 3, 16, 20, 50, 64, 100, 128, 300, 5000) for n in (1, 128, 1000, 4096, 19100, 28672, 128256)
            for k in (32, 4096, 8480, 14336, 16384, 18464, 24608, 32768, 65536, 131072, 400000, 1 << 20, (1 << 31) - 544)
            for sms in (SMS, 132, 2)]
    worst = max(zip(choose(rows), rows), key=lambda x: x[0][2])
    assert worst[0][2] <= 48, worst
