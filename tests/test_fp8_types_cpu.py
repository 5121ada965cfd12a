"""GGML types that the conversion does not take raise the same error on every way to it."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from llima_b200 import fp8


@pytest.mark.parametrize("fmt", ["IQ4_NL", "TQ1_0", "Q8_K", "F64", "nothing"])
def test_types_that_are_not_handled(fmt):
    with pytest.raises(NotImplementedError, match=fmt):
        fp8.convert_fp8_device(fmt, torch.zeros(64, dtype=torch.uint8), 1, 32)


def test_a_reader_tensor_of_such_a_type():
    gguf = pytest.importorskip("gguf")
    t = SimpleNamespace(name="w", tensor_type=gguf.GGMLQuantizationType.IQ4_NL, shape=np.array([32, 1]), data=np.zeros((1, 18), np.uint8))
    with pytest.raises(NotImplementedError, match="IQ4_NL"):
        fp8.fp8_from_gguf(t)
