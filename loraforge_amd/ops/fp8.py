"""FP8 weights and activations (e4m3 with an fp32 scale for each block of 128) and their linear, on gfx950.

A scale belongs to 128 values of a row (activations, ``block_rows=1``) or to a block of
128 rows x 128 columns (weights, ``block_rows=128``); the last block of a dimension
may be shorter. It is the format that checkpoints with block-scaled FP8 weights ship
in, used as it is stored. ``fp8_linear`` keeps bf16 activations as they are, or
multiplies activations that ``quantize_fp8`` brought into the format at the matrix
cores' 8-bit rate (which drops low bits within eight products: see ``fp8_linear``); a block's products are summed first
and scaled once, in fp32.

``expert_linear`` and ``expert_mlp`` take FP8 weights too. The operators are for
inference: tensors that require gradients are refused.
"""

from __future__ import annotations

from dataclasses import dataclass

from .. import _lib
from ..annotations import ExperimentalAPI
from . import mxfp4
from ._checks import distinct_output, require_arch, tensor

BLOCK = 128


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


@dataclass
class FP8Tensor:
    """``codes`` ``float8_e4m3fn`` ``[..., R, K]`` and fp32 ``scales``, both contiguous.

    ``scales`` is ``[..., R, ceil(K / 128)]`` (a scale for 128 values of a row) or
    ``[..., ceil(R / 128), ceil(K / 128)]`` (a scale for a block).
    """

    codes: object
    scales: object

    @property
    def shape(self) -> tuple:
        return tuple(self.codes.shape)

    @property
    def ndim(self) -> int:
        return self.codes.ndim

    @property
    def device(self):
        return self.codes.device


def scaled(t, name, ndim=None, device=None, *, block_rows=None):
    """Checks of an ``FP8Tensor`` (of ``ndim`` dimensions, its scales for ``block_rows`` rows); returns the rows of a scale."""
    import torch

    if not isinstance(t, FP8Tensor):
        raise TypeError(f"{name} must be an FP8Tensor")
    if ndim is None:
        ndim = getattr(t.codes, "ndim", 0)
        if ndim < 2:
            raise ValueError(f"{name} must have rows and columns")
    tensor(t.codes, f"{name}.codes", ndim, torch.float8_e4m3fn, device)
    tensor(t.scales, f"{name}.scales", ndim, torch.float32, t.codes.device)
    rows, k = t.codes.shape[-2:]
    if k == 0 or k % 16:
        raise ValueError(f"{name}'s last dimension must be a positive multiple of 16")
    held = tuple(t.scales.shape)
    lead = tuple(t.codes.shape[:-2])
    kinds = [b for b in ((1, BLOCK) if block_rows is None else (block_rows,)) if held == (*lead, -(-rows // b), _blocks(k))]
    if not kinds:
        raise ValueError(f"{name} must hold one scale for each block of 128 values"
                         + ("" if block_rows is None else " of a row" if block_rows == 1 else " x 128 rows"))
    if not t.codes.is_contiguous() or not t.scales.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.codes.data_ptr() % 16:
        raise ValueError(f"{name} codes must be 16-byte aligned")
    return kinds[0]


@ExperimentalAPI(reason="Block-scaled FP8 quantisation; gfx950 HIP kernel.")
def quantize_fp8(x, *, block_rows: int = 1) -> FP8Tensor:
    """``x`` (bf16 ``[..., R, K]``, 16-byte aligned rows, K a multiple of 16) in FP8.

    ``block_rows`` 1 gives 128 values of a row a scale, 128 a block of 128 x 128.
    With ``A`` the block's largest magnitude, but at least 2^-100, the scale is
    ``A / 448`` and the codes are ``448 x / A`` rounded to nearest, ties to even. A
    block that holds infinity or NaN becomes NaN.
    """
    import torch

    if getattr(x, "is_cuda", False):
        done = _lib.binding().fp8_quantize(x, block_rows)
        if done is not None:
            return FP8Tensor(*done)
    if type(block_rows) is not int or block_rows not in (1, BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if x.ndim < 2 or x.dtype != torch.bfloat16:
        raise ValueError("x must have rows and columns and dtype torch.bfloat16")
    if x.device.type != "cuda":
        raise ValueError("x must be on the same CUDA/ROCm GPU")
    if x.requires_grad:
        raise ValueError("FP8 operators are inference-only")
    if any(size >= 2**31 for size in x.shape):
        raise ValueError("x dimensions must fit signed int32 indexing")
    rows, k = x.shape[-2:]
    if k == 0 or k % 16:
        raise ValueError("the last dimension must be a positive multiple of 16")
    if x.ndim != 2 and not x.is_contiguous():
        raise ValueError("x of other than two dimensions must be contiguous")
    lead = x.shape[:-2]
    matrices = lead.numel()
    stride = x.stride(0) if x.ndim == 2 and rows > 1 else k
    if x.numel() and (x.stride(-1) != 1 or stride < k or stride % 8 or x.data_ptr() % 16):
        raise ValueError("x rows must be 16-byte aligned with unit stride")
    if matrices >= 2**31:
        raise ValueError("x dimensions must fit signed int32 indexing")
    require_arch(x.device)
    out = FP8Tensor(
        torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device),
        torch.empty((*lead, -(-rows // block_rows), _blocks(k)), dtype=torch.float32, device=x.device),
    )
    if x.numel():
        with torch.cuda.device(x.device):
            _lib.check(
                _lib.library().lf_fp8_quantize(
                    x.data_ptr(), matrices, rows, k, stride, block_rows, out.codes.data_ptr(), out.scales.data_ptr(),
                    _lib.stream_of(x.device)))
    return out


@ExperimentalAPI(reason="Block-scaled FP8 dequantisation; gfx950 HIP kernel.")
def dequantize_fp8(t: FP8Tensor, *, out=None):
    """The values of ``t``, a code times its scale, rounded once to bf16."""
    import torch

    if not isinstance(t, FP8Tensor):
        raise TypeError("t must be an FP8Tensor")
    if out is None and getattr(t.codes, "is_cuda", False):
        done = _lib.binding().fp8_dequantize(t)
        if done is not None:
            return done
    scale_rows = scaled(t, "t")
    rows, k = t.shape[-2:]
    if out is None:
        out = torch.empty(t.shape, dtype=torch.bfloat16, device=t.device)
    tensor(out, "out", t.ndim, torch.bfloat16, t.device)
    if tuple(out.shape) != t.shape or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous, 16-byte aligned and of the values' shape")
    distinct_output(out, (t.codes, t.scales))
    require_arch(t.device)
    if out.numel():
        with torch.cuda.device(t.device):
            _lib.check(
                _lib.library().lf_fp8_dequantize(
                    t.codes.data_ptr(), t.scales.data_ptr(), out.numel() // (rows * k), rows, k, scale_rows, out.data_ptr(),
                    _lib.stream_of(t.device)))
    return out


@ExperimentalAPI(reason="Block-scaled FP8 linear; gfx950 HIP kernel.")
def fp8_linear(x, weight: FP8Tensor, *, bias=None, swiglu: bool = False, out=None):
    """``x @ weight.T (+ bias)`` in bf16 for an FP8 ``weight`` ``[N, K]`` with a scale for each 128 x 128 block.

    ``x`` is bf16 ``[M, K]`` with 16-byte aligned rows, or an ``FP8Tensor`` ``[M, K]``
    with a scale for each 128 values of a row (``quantize_fp8``): both operands then go
    through the 8-bit matrix instructions. Sums in fp32: each block's products first,
    then times the scales (whose product is formed first), rounded once. With an FP8 ``x`` the
    matrix instructions add eight products of consecutive k at a time, aligned to the largest of them, and drop what lies
    2^-13 below it: beside bf16's rounding little for most activations, but a sum whose large terms cancel
    is not exact. bf16 ``x`` has no such loss. ``swiglu``: the weight is a merged
    ``[gate | up]`` (each a multiple of 128 rows) and the result ``silu(gate) * up``,
    ``[M, N / 2]``, in fp32 before its rounding.
    """
    if not isinstance(weight, FP8Tensor):
        raise TypeError("weight must be an FP8Tensor")
    return mxfp4.product(x, weight, experts=None, offsets=None, tokens=None, bias=bias, swiglu=swiglu, out=out)
