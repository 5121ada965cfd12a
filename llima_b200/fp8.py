"""Block-scaled 8-bit floats: a GGUF file's projections on the GPU itself.

The reference prepares integer weights and leaves the products to the Modalix accelerator
(``ModelGraph.linear``, ``sima_lmm/model/model_graph.py:351-403``).  Here the same GGUF
tensors become e4m3 weights that the B200's tensor cores multiply directly, with the two
operators that feed them:

* ``convert_fp8_device`` / ``fp8_from_gguf``: a GGUF tensor to e4m3 codes with one
  power-of-two scale per 128 x 128 block (``Fp8Weight``);
* ``rms_norm_fp8``: RMS norm, with the residual's addition, to e4m3 rows with one scale per
  1 x 128 block (``Fp8Rows``);
* ``quantize_fp8``: rows, or silu(gate) * rows, quantized the same way;
* ``matmul_fp8``: ``Fp8Rows`` times ``Fp8Weight``, for one token as for a long prompt;
* ``Fp8Linear`` and ``Fp8FeedForward``: a projection, and a layer's gated feed-forward block,
  from a GGUF file's tensors;
* ``check_kernels``: whether a kernel gave up waiting and left its result incomplete.

Scales are ``float8_e8m0fnu``: 2^e with the smallest e >= -127 for which the block's largest
finite magnitude is at most 448 * 2^e.  A value that is not finite becomes the NaN code.
Row counts are free; column counts are multiples of 32, as every quantized GGUF row's are.

Work is enqueued on the current stream of the operands' device, whichever device is
current, and no call waits for it.  There are no gradients: outside ``torch.no_grad()`` an operand
that requires one is refused.  A tensor given as ``out`` or ``sum_out`` shares no memory with
another operand except where stated (refused as well).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import numpy as np
import torch

from . import _native as N
from .formats import FORMATS

__all__ = ["Fp8Rows", "Fp8Weight", "convert_fp8_device", "fp8_from_gguf", "rms_norm_fp8", "quantize_fp8",
           "matmul_fp8", "check_kernels", "Fp8Linear", "Fp8FeedForward"]

BLOCK = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_TYPE_IDS = {torch.float32: FORMATS["F32"].type_id, torch.float16: FORMATS["F16"].type_id,
             torch.bfloat16: FORMATS["BF16"].type_id}
# Architectures (general.architecture of a GGUF file) whose feed-forward block is the one of
# Fp8FeedForward.  Others hold tensors under the same names and compute something else with
# them: Gemma takes tanh-GELU and, from its second version, a norm of the block's output.
_GATED_SILU = ("llama", "mistral", "qwen2", "qwen3")


class Fp8Rows(NamedTuple):
    """Activations: codes (rows, cols) float8_e4m3fn and scales (rows, ceil(cols / 128))
    float8_e8m0fnu."""
    codes: torch.Tensor
    scales: torch.Tensor


class Fp8Weight(NamedTuple):
    """Weights: codes (rows, cols) float8_e4m3fn, rows = output channels, and scales
    (ceil(rows / 128), ceil(cols / 128)) float8_e8m0fnu."""
    codes: torch.Tensor
    scales: torch.Tensor


def _call(name: str, device: int, *args) -> None:
    """The C entry point `name` with the current stream of CUDA device `device`, which is made
    current for the call.  (``torch.cuda.current_stream`` builds a Stream object, 3 us a call;
    its handle alone is what the C ABI takes.)"""
    if device == _current_device():
        status = getattr(N.lib(), name)(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = getattr(N.lib(), name)(*args, _raw_stream(device))
    if status:
        N.check(status, name)


def _no_backward(*tensors: torch.Tensor | None) -> None:
    """These operators have no backward pass: an operand that a gradient is asked for is refused
    rather than detached in silence.  (Callers look at ``requires_grad`` themselves first: a call
    costs half a microsecond.)"""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("no gradients through the 8-bit float operators: detach the operand, or call under torch.no_grad()")


def _written(*tensors: torch.Tensor) -> None:
    """Tells autograd that these tensors of the caller's were written, so that a backward pass that
    saved what was there before fails instead of using what is there now."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _matrix(t: torch.Tensor, name: str, dtype, device: int, rows: int | None = None, cols: int | None = None) -> int:
    """Checks a 2-D operand on CUDA device `device` whose rows are consecutive elements;
    returns its row stride."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the other operands on cuda:{device}")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, not {t.dim()}")
    r, c = t.shape
    if (rows is not None and r != rows) or (cols is not None and c != cols):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected "
                         f"{(r if rows is None else rows, c if cols is None else cols)}")
    s0, s1 = t.stride()
    if s1 != 1 and c > 1:
        raise ValueError(f"the elements of a row of {name} must be consecutive (strides {t.stride()})")
    if r <= 1:
        return c
    if s0 < c:
        raise ValueError(f"the rows of {name} overlap (strides {t.stride()})")
    return s0


def _new(rows: int, cols: int, dtype, device) -> torch.Tensor:
    """An uninitialized row-major tensor (empty_strided: the cheapest of torch's ways)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _device_of(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _vector(t: torch.Tensor, name: str, n: int, device: int) -> int:
    """Checks `n` consecutive float32 values on CUDA device `device`; returns their address."""
    if t.dtype is not torch.float32 or t.shape != (n,) or t.get_device() != device or (t.stride(0) != 1 and n > 1):
        raise ValueError(f"{name} must be a contiguous float32 tensor of {n} values on cuda:{device}")
    return t.data_ptr()


def _float_rows(x: torch.Tensor, name: str) -> int:
    if x.dtype not in _TYPE_IDS:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, not {x.dtype}")
    ld = _matrix(x, name, x.dtype, _device_of(x, name))
    if x.shape[1] % 32:
        raise ValueError(f"{name} has {x.shape[1]} columns: a multiple of 32 is needed")
    return ld


def _rows_out(x: torch.Tensor, device: int, out: Fp8Rows | None):
    """The codes and scales that rows shaped like x go to, with their row strides."""
    rows, cols = x.shape
    blocks = (cols + 127) >> 7
    if out is None:
        return (torch.empty_like(x, dtype=E4M3, memory_format=torch.contiguous_format), cols,
                _new(rows, blocks, E8M0, x.device), blocks)
    codes, scales = out
    return (codes, _matrix(codes, "out.codes", E4M3, device, rows, cols),
            scales, _matrix(scales, "out.scales", E8M0, device, rows, blocks))


def _known(fmt: str) -> str:
    if fmt not in FORMATS:
        raise NotImplementedError(f"GGML type {fmt} is not handled by the B200 GGUF path")
    return fmt


def convert_fp8_device(fmt: str, src: torch.Tensor, rows: int, cols: int, heads: int = 0,
                       out: Fp8Weight | None = None) -> Fp8Weight:
    """GGUF bytes already on the GPU (uint8, 16-byte aligned) -> ``Fp8Weight``.  The values
    quantized are those of the f32 conversion, bit for bit; heads > 0 applies the llama q/k
    row permutation (``GgufModel._permute_qk_proj``, gguf_conversion.py:314-332)."""
    f = FORMATS[_known(fmt)]
    if src.dtype != torch.uint8 or not src.is_cuda or not src.is_contiguous():
        raise TypeError("src must be a contiguous CUDA uint8 tensor of GGUF bytes")
    dev = src.get_device()
    shape = ((rows + BLOCK - 1) // BLOCK, (cols + BLOCK - 1) // BLOCK)
    given = out
    if out is None:
        if rows < 0 or cols < 0:
            raise ValueError(f"negative shape ({rows}, {cols})")
        out = Fp8Weight(_new(rows, cols, E4M3, src.device), _new(*shape, E8M0, src.device))
    else:
        _no_backward(*out)
        _matrix(out.codes, "out.codes", E4M3, dev, rows, cols)
        _matrix(out.scales, "out.scales", E8M0, dev, *shape)
        if not out.codes.is_contiguous() or not out.scales.is_contiguous():
            raise ValueError("out must be contiguous")
    t = N.Tensor(type=f.type_id, perm_heads=heads, rows=rows, cols=cols, src=src.data_ptr(), src_bytes=src.numel(),
                 codes=out.codes.data_ptr())
    _call("gq_convert_fp8", dev, ctypes.byref(t), out.scales.data_ptr())
    if given is not None:
        _written(*out)
    return out


def fp8_from_gguf(gguf_tensor, heads: int = 0, device=None) -> Fp8Weight:
    """``Fp8Weight`` of one reader tensor (rows = output channels).  ``device``: a CUDA
    device, the current one by default."""
    from .gguf_conversion import _type_name
    fmt = _known(_type_name(gguf_tensor.tensor_type))
    shape = tuple(int(x) for x in gguf_tensor.shape[::-1])
    if len(shape) != 2:
        raise ValueError(f"{gguf_tensor.name}: a weight has two dimensions, not {len(shape)}")
    raw = np.ascontiguousarray(gguf_tensor.data).reshape(-1).view(np.uint8)
    src = torch.from_numpy(raw if raw.flags.writeable else raw.copy()).to("cuda" if device is None else device)
    return convert_fp8_device(fmt, src, *shape, heads)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: torch.Tensor | None = None,
                 sum_out: torch.Tensor | None = None, out: Fp8Rows | None = None):
    """RMS norm of the rows of ``x`` (rows, cols), quantized: ``Fp8Rows`` of
    h / sqrt(mean(h^2) + eps) * weight, weight float32 (cols).  With ``residual`` (of x's
    type and shape), h = x + residual rounded to that type and (``Fp8Rows``, h) is returned;
    ``sum_out`` receives h and may be ``residual`` or ``x`` itself."""
    if x.requires_grad or weight.requires_grad or residual is not None and residual.requires_grad or \
            sum_out is not None and sum_out.requires_grad or out is not None:
        _no_backward(x, weight, residual, sum_out, *(out or ()))
    ld_x = _float_rows(x, "x")
    rows, cols = x.shape
    dev = x.get_device()
    w = _vector(weight, "weight", cols, dev)
    ld_r = ld_s = 0
    r = s = None
    given = sum_out
    if residual is not None:
        ld_r = _matrix(residual, "residual", x.dtype, dev, rows, cols)
        if sum_out is None:
            sum_out, ld_s = torch.empty_like(x, memory_format=torch.contiguous_format), cols
        else:
            ld_s = _matrix(sum_out, "sum_out", x.dtype, dev, rows, cols)
        r, s = residual.data_ptr(), sum_out.data_ptr()
    elif sum_out is not None:
        raise ValueError("sum_out without residual")
    codes, ld_c, scales, ld_sc = _rows_out(x, dev, out)
    _call("gq_rms_norm_fp8", dev, _TYPE_IDS[x.dtype], x.data_ptr(), ld_x, r, ld_r, w, eps, rows, cols, s, ld_s,
          codes.data_ptr(), ld_c, scales.data_ptr(), ld_sc)
    if out is not None:
        _written(*out)
    if given is not None:
        _written(given)
    q = Fp8Rows(codes, scales)
    return q if residual is None else (q, sum_out)


def quantize_fp8(x: torch.Tensor, gate: torch.Tensor | None = None, out: Fp8Rows | None = None) -> Fp8Rows:
    """Rows of ``x`` (rows, cols), or silu(gate) * x with ``gate`` of x's type and shape, as
    ``Fp8Rows``.  Both may be column ranges of one wider tensor, as a fused gate and up
    product leaves them."""
    if x.requires_grad or gate is not None and gate.requires_grad or out is not None:
        _no_backward(x, gate, *(out or ()))
    ld_x = _float_rows(x, "x")
    rows, cols = x.shape
    dev = x.get_device()
    ld_g, g = 0, None
    if gate is not None:
        ld_g, g = _matrix(gate, "gate", x.dtype, dev, rows, cols), gate.data_ptr()
    codes, ld_c, scales, ld_sc = _rows_out(x, dev, out)
    _call("gq_quantize_fp8", dev, _TYPE_IDS[x.dtype], x.data_ptr(), ld_x, g, ld_g, rows, cols, codes.data_ptr(), ld_c,
          scales.data_ptr(), ld_sc)
    if out is not None:
        _written(*out)
    return Fp8Rows(codes, scales)


def matmul_fp8(a: Fp8Rows, w: Fp8Weight, bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """a (m, k) times w (n, k) transposed, plus ``bias`` (n, float32): (m, n) of ``dtype``
    (bfloat16, float16 or float32; that of ``out`` when given), accumulated in float32 and
    rounded once.  The tensor cores truncate as they accumulate; for float32 results they take
    sums of at most 6144 columns, which are added with rounding."""
    codes, scales = a
    w_codes, w_scales = w
    if codes.requires_grad or w_codes.requires_grad or scales.requires_grad or w_scales.requires_grad or \
            bias is not None and bias.requires_grad or out is not None and out.requires_grad:
        _no_backward(codes, scales, w_codes, w_scales, bias, out)
    dev = _device_of(codes, "a.codes")
    ld_a = _matrix(codes, "a.codes", E4M3, dev)
    m, k = codes.shape
    if k % 32:
        raise ValueError(f"a.codes has {k} columns: a multiple of 32 is needed")
    blocks = (k + 127) >> 7
    ld_sa = _matrix(scales, "a.scales", E8M0, dev, m, blocks)
    ld_b = _matrix(w_codes, "w.codes", E4M3, dev, None, k)
    n = w_codes.shape[0]
    ld_sb = _matrix(w_scales, "w.scales", E8M0, dev, (n + 127) >> 7, blocks)
    given = out
    if out is None:
        if dtype not in _TYPE_IDS:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
        out, ld_o = _new(m, n, dtype, codes.device), n
    else:
        dtype = out.dtype
        if dtype not in _TYPE_IDS:
            raise TypeError(f"out must be float32, float16 or bfloat16, not {dtype}")
        ld_o = _matrix(out, "out", dtype, dev, m, n)
    _call("gq_matmul_fp8", dev, codes.data_ptr(), ld_a, scales.data_ptr(), ld_sa, w_codes.data_ptr(), ld_b,
          w_scales.data_ptr(), ld_sb, None if bias is None else _vector(bias, "bias", n, dev), m, n, k, _TYPE_IDS[dtype],
          out.data_ptr(), ld_o)
    if given is not None:
        _written(out)
    return out


def check_kernels(device=None) -> None:
    """Waits for the work on ``device`` (a CUDA device, the current one by default) and raises
    ``RuntimeError`` when one of the library's kernels there gave up a wait (for a tile copy, or
    for the tensor cores, after a second) since the last call.  Such a kernel ends with its
    result incomplete, and nothing else tells: a program that must not pass one on calls this
    before it uses results, as seldom as it likes.  The record is cleared."""
    torch.cuda.synchronize(device)
    index = torch.device("cuda" if device is None else device).index if not isinstance(device, int) else device
    if index is None:
        index = torch.cuda.current_device()
    flags = ctypes.c_uint32(0)
    N.check(N.lib().gq_kernel_errors(index, 1, ctypes.byref(flags)), "gq_kernel_errors")
    if flags.value:
        raise RuntimeError(f"a kernel on cuda:{index} gave up waiting (flags {flags.value}): results since the last check may "
                           "be incomplete")


class Fp8Linear:
    """One projection: ``Fp8Weight`` and an optional float32 bias."""

    def __init__(self, weight: Fp8Weight, bias: torch.Tensor | None = None):
        self.weight = weight
        self.bias = bias

    @classmethod
    def from_gguf(cls, gguf_tensor, bias_tensor=None, heads: int = 0, device=None) -> "Fp8Linear":
        """From a reader's weight tensor and, where the model has one, its bias tensor;
        heads > 0 applies the llama q/k row permutation to both."""
        if bias_tensor is not None and math.prod(int(x) for x in bias_tensor.shape) != int(gguf_tensor.shape[-1]):
            raise ValueError(f"{bias_tensor.name} has shape {tuple(bias_tensor.shape)}: {gguf_tensor.name} has "
                             f"{int(gguf_tensor.shape[-1])} output channels")
        weight = fp8_from_gguf(gguf_tensor, heads, device)
        bias = None
        if bias_tensor is not None:
            from .gguf_conversion import load_tensor
            b = np.array(load_tensor(bias_tensor, True, heads)[1], dtype=np.float32).reshape(-1)
            bias = torch.from_numpy(b).to(weight.codes.device)
        return cls(weight, bias)

    def __call__(self, x: Fp8Rows | torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """x as ``Fp8Rows``, or float rows that are quantized first."""
        if not isinstance(x, Fp8Rows):
            x = quantize_fp8(x)
        return matmul_fp8(x, self.weight, self.bias, dtype)


class Fp8FeedForward:
    """A layer's gated feed-forward block: x + residual -> RMS norm -> gate and up products ->
    silu(gate) * up -> down product, every product on e4m3 operands.  The gate and up weights
    sit in one tensor and are one product."""

    def __init__(self, norm: torch.Tensor, gate_up: Fp8Weight, down: Fp8Weight, eps: float = 1e-5):
        self.norm, self.gate_up, self.down, self.eps = norm, gate_up, down, eps

    @classmethod
    def from_gguf(cls, reader, layer: int, device=None) -> "Fp8FeedForward":
        """From a ``gguf.GGUFReader`` (or a path) by the tensors' GGUF names: ``blk.N.ffn_norm``,
        ``ffn_gate``, ``ffn_up`` and ``ffn_down``; the epsilon from the file's metadata.  For files
        of the architectures llama, mistral, qwen2 and qwen3; a file of another one, or a layer
        with further feed-forward tensors (biases, a norm after the block, experts), computes
        something else and is refused (``NotImplementedError``)."""
        if not hasattr(reader, "tensors"):
            from gguf import GGUFReader
            reader = GGUFReader(reader)
        from .gguf_conversion import _type_name, load_tensor
        arch = reader.fields["general.architecture"].contents()
        if arch not in _GATED_SILU:
            raise NotImplementedError(f"the feed-forward block of architecture {arch!r} is not known to be norm -> "
                                      f"silu(gate) * up -> down (known: {', '.join(_GATED_SILU)})")
        names = {t.name: t for t in reader.tensors}
        parts = [f"blk.{layer}.ffn_{part}.weight" for part in ("norm", "gate", "up", "down")]
        more = sorted(n for n in names if n.startswith((f"blk.{layer}.ffn_", f"blk.{layer}.post_ffw_")) and n not in parts)
        if more:
            raise NotImplementedError(f"layer {layer} has feed-forward tensors that this block does not take: {', '.join(more)}")
        norm, gate, up, down = (names[part] for part in parts)
        eps = float(reader.fields[f"{arch}.attention.layer_norm_rms_epsilon"].contents())
        dev = torch.device("cuda" if device is None else device)
        shapes = [tuple(int(x) for x in t.shape[::-1]) for t in (gate, up, down, norm)]
        if len(shapes[0]) != 2:
            raise ValueError(f"{gate.name}: a weight has two dimensions, not {len(shapes[0])}")
        rows, cols = shapes[0]
        if shapes != [(rows, cols), (rows, cols), (cols, rows), (cols,)]:
            raise ValueError("the shapes of gate, up, down and norm do not belong together: " + ", ".join(map(str, shapes)))
        for t in (gate, up, down):
            _known(_type_name(t.tensor_type))
        if rows % BLOCK:
            raise ValueError(f"{rows} feed-forward channels: a multiple of {BLOCK} is needed to keep the gate and up "
                             "weights in one tensor")
        both = Fp8Weight(torch.empty((2 * rows, cols), dtype=E4M3, device=dev),
                         torch.empty((2 * rows // BLOCK, -(-cols // BLOCK)), dtype=E8M0, device=dev))
        for i, t in enumerate((gate, up)):
            part = slice(i * rows, (i + 1) * rows), slice(i * rows // BLOCK, (i + 1) * rows // BLOCK)
            raw = torch.from_numpy(np.array(t.data).reshape(-1).view(np.uint8)).to(dev)
            convert_fp8_device(_type_name(t.tensor_type), raw, rows, cols,
                               out=Fp8Weight(both.codes[part[0]], both.scales[part[1]]))
        w = torch.from_numpy(np.array(load_tensor(norm, True)[1], dtype=np.float32).reshape(-1)).to(dev)
        return cls(w, both, fp8_from_gguf(down, device=dev), eps)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor):
        """x and residual (rows, hidden) -> (the block's output, the residual that it is to be
        added to: x + residual), both of x's type."""
        q, h = rms_norm_fp8(x, self.norm, self.eps, residual=residual)
        both = matmul_fp8(q, self.gate_up, dtype=x.dtype)
        half = both.shape[1] // 2
        return matmul_fp8(quantize_fp8(both[:, half:], gate=both[:, :half]), self.down, dtype=x.dtype), h
