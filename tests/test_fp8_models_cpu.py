"""Which GGUF files a feed-forward block is made of: the refusals come before any CUDA call, so
they run without a GPU."""
import numpy as np
import pytest

from llima_b200 import fp8
from llima_b200.formats import FORMATS
from llima_b200.synth import gen_tensor_bytes

gguf = pytest.importorskip("gguf")


class Reached(Exception):
    pass


def write_file(path, arch="llama", extra=(), fmts=("Q8_0", "Q8_0", "Q8_0"), shapes=((256, 128), (256, 128), (128, 256)), norm=128):
    w = gguf.GGUFWriter(str(path), arch)
    w.add_layer_norm_rms_eps(1e-6)
    for name, fmt, (rows, cols) in zip(("gate", "up", "down"), fmts, shapes):
        f = FORMATS[fmt]
        raw = gen_tensor_bytes(fmt, rows * cols, len(name))
        w.add_tensor(f"blk.0.ffn_{name}.weight", raw.reshape(rows, cols // f.unit_values * f.unit_bytes),
                     raw_dtype=gguf.GGMLQuantizationType(f.type_id))
    w.add_tensor("blk.0.ffn_norm.weight", np.ones(norm, np.float32))
    for name in extra:
        w.add_tensor(name, np.ones(128, np.float32))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    return path


@pytest.fixture
def no_gpu(monkeypatch):
    """Stands for everything after the file was accepted."""
    def reached(*_, **__):
        raise Reached

    monkeypatch.setattr(fp8, "_new", reached)
    monkeypatch.setattr(fp8, "convert_fp8_device", reached)
    monkeypatch.setattr(fp8.torch, "empty", reached)


@pytest.mark.parametrize("arch", ["llama", "mistral", "qwen2", "qwen3"])
def test_architectures_with_this_block(tmp_path, arch, no_gpu):
    """Layers with other tensors beside them are no obstacle: blk.01 is not blk.0's."""
    path = write_file(tmp_path / "m.gguf", arch, extra=["blk.0.attn_norm.weight", "blk.01.ffn_up.bias", "blk.0.attn_q.bias"])
    with pytest.raises(Reached):
        fp8.Fp8FeedForward.from_gguf(path, 0, device="cpu")


@pytest.mark.parametrize("arch", ["gemma", "gemma2", "gemma3", "unheard_of"])
def test_architectures_with_another_block(tmp_path, arch, no_gpu):
    """The same tensors under the same names, and another activation, scale or norm."""
    path = write_file(tmp_path / "m.gguf", arch)
    with pytest.raises(NotImplementedError, match=arch):
        fp8.Fp8FeedForward.from_gguf(path, 0, device="cpu")


@pytest.mark.parametrize("name", ["post_ffw_norm.weight", "ffn_gate.bias", "ffn_up.bias", "ffn_down.bias", "ffn_norm.bias",
                                  "ffn_sub_norm.weight", "ffn_gate_inp.weight"])
def test_layers_with_more_tensors(tmp_path, name, no_gpu):
    path = write_file(tmp_path / "m.gguf", extra=[f"blk.0.{name}"])
    with pytest.raises(NotImplementedError, match=name):
        fp8.Fp8FeedForward.from_gguf(path, 0, device="cpu")


@pytest.mark.parametrize("change", [{"shapes": ((256, 128), (384, 128), (128, 256))}, {"shapes": ((256, 128), (256, 160), (128, 256))},
                                    {"shapes": ((256, 128), (256, 128), (128, 288))}, {"shapes": ((256, 128), (256, 128), (160, 256))},
                                    {"norm": 160}, {"shapes": ((256, 160), (256, 160), (160, 256))}])
def test_shapes_that_do_not_belong_together(tmp_path, change, no_gpu):
    path = write_file(tmp_path / "m.gguf", **change)
    with pytest.raises(ValueError, match="do not belong together"):
        fp8.Fp8FeedForward.from_gguf(path, 0, device="cpu")


def test_feed_forward_channels_off_the_block(tmp_path, no_gpu):
    path = write_file(tmp_path / "m.gguf", shapes=((320, 128), (320, 128), (128, 320)))
    with pytest.raises(ValueError, match="multiple of 128"):
        fp8.Fp8FeedForward.from_gguf(path, 0, device="cpu")


def test_a_bias_of_another_length(tmp_path, no_gpu):
    path = write_file(tmp_path / "m.gguf", extra=["blk.0.attn_q.bias"])
    t = {t.name: t for t in gguf.GGUFReader(path).tensors}
    with pytest.raises(ValueError, match="256 output channels"):
        fp8.Fp8Linear.from_gguf(t["blk.0.ffn_gate.weight"], t["blk.0.attn_q.bias"], device="cpu")
    with pytest.raises(Reached):
        fp8.Fp8Linear.from_gguf(t["blk.0.ffn_down.weight"], t["blk.0.attn_q.bias"], device="cpu")
