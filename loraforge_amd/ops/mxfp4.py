"""MXFP4 weights and activations (OCP microscaling, 4 bits) and their linear, on gfx950.

A block of 32 values along the last dimension shares one e8m0 scale byte ``s``;
a value is ``level * 2 ** (s - 127)`` with a sign and a level out of 0, 0.5, 1,
1.5, 2, 3, 4, 6, two codes a byte (the low nibble is the even index). It is
the format that checkpoints with 4-bit floating point experts ship and that
gfx950's matrix instructions multiply directly, so weights are used as they
are stored: no codebook, no second layout.

``mxfp4_linear`` keeps bf16 activations as they are, or multiplies activations
that ``quantize_mxfp4`` brought into the same format at the matrix cores' 4-bit
rate. The operators are for inference: tensors that require gradients are
refused. LoRA adapters are added to the output with ``lora_apply``.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

from .. import _lib
from ..annotations import ExperimentalAPI
from . import fp8
from ._checks import distinct_output, require_arch, tensor, vector

BLOCK = 32


@dataclass
class MXFP4Tensor:
    """``codes`` uint8 ``[..., K / 2]`` and ``scales`` uint8 ``[..., K / 32]``, contiguous, of the same leading shape."""

    codes: object
    scales: object

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:-1], self.codes.shape[-1] * 2)

    @property
    def ndim(self) -> int:
        return self.codes.ndim

    @property
    def device(self):
        return self.codes.device


def packed(t, name, ndim, device=None):
    """Checks of an ``MXFP4Tensor`` of ``ndim`` dimensions; returns its shape."""
    import torch

    if not isinstance(t, MXFP4Tensor):
        raise TypeError(f"{name} must be an MXFP4Tensor")
    tensor(t.codes, f"{name}.codes", ndim, torch.uint8, device)
    tensor(t.scales, f"{name}.scales", ndim, torch.uint8, t.codes.device)
    k = t.codes.shape[-1] * 2
    if k == 0 or k % BLOCK or tuple(t.scales.shape) != (*t.codes.shape[:-1], k // BLOCK):
        raise ValueError(f"{name} must hold one scale for each block of 32 along its last dimension")
    if not t.codes.is_contiguous() or not t.scales.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.codes.data_ptr() % 16:
        raise ValueError(f"{name} codes must be 16-byte aligned")
    return t.shape


@ExperimentalAPI(reason="MXFP4 quantisation; gfx950 HIP kernel.")
def quantize_mxfp4(x) -> MXFP4Tensor:
    """``x`` (bf16 or fp32, 16-byte aligned rows, last dimension a multiple of 32) in MXFP4.

    A block's scale is ``2 ** (floor(log2(max |x|)) - 2)`` (its byte at least
    0; 0 for a block of zeros), codes are rounded to nearest, ties to even, and
    saturate at 6. A block that holds infinity or NaN becomes NaN.
    """
    import torch

    if getattr(x, "is_cuda", False):
        done = _lib.binding().mx_quantize(x)
        if done is not None:
            return MXFP4Tensor(*done)
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if x.ndim < 1 or x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("x must have dtype torch.bfloat16 or torch.float32")
    if x.device.type != "cuda":
        raise ValueError("x must be on the same CUDA/ROCm GPU")
    if x.requires_grad:
        raise ValueError("MXFP4 operators are inference-only")
    k = x.shape[-1]
    if k == 0 or k % BLOCK:
        raise ValueError("the last dimension must be a positive multiple of 32")
    if x.ndim != 2 and not x.is_contiguous():
        raise ValueError("x of other than two dimensions must be contiguous")
    rows = x.numel() // k
    stride = x.stride(0) if x.ndim == 2 and rows > 1 else k
    unit = 16 // x.element_size()
    if x.stride(-1) != 1 or stride < k or stride % unit or x.data_ptr() % 16:
        raise ValueError("x rows must be 16-byte aligned with unit stride")
    require_arch(x.device)
    out = MXFP4Tensor(
        torch.empty((*x.shape[:-1], k // 2), dtype=torch.uint8, device=x.device),
        torch.empty((*x.shape[:-1], k // BLOCK), dtype=torch.uint8, device=x.device),
    )
    if rows:
        with torch.cuda.device(x.device):
            _lib.check(
                _lib.library().lf_mxfp4_quantize(
                    x.data_ptr(), x.dtype == torch.float32, rows, k, stride, out.codes.data_ptr(), out.scales.data_ptr(),
                    _lib.stream_of(x.device)))
    return out


@ExperimentalAPI(reason="MXFP4 dequantisation; gfx950 HIP kernel.")
def dequantize_mxfp4(t: MXFP4Tensor, *, out=None):
    """The bf16 values of ``t`` (exact: a level times a power of two)."""
    import torch

    if not isinstance(t, MXFP4Tensor):
        raise TypeError("t must be an MXFP4Tensor")
    if out is None and getattr(t.codes, "is_cuda", False):
        done = _lib.binding().mx_dequantize(t)
        if done is not None:
            return done
    shape = packed(t, "t", t.ndim)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=t.device)
    tensor(out, "out", len(shape), torch.bfloat16, t.device)
    if tuple(out.shape) != shape or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous, 16-byte aligned and of the values' shape")
    distinct_output(out, (t.codes, t.scales))
    require_arch(t.device)
    if out.numel():
        with torch.cuda.device(t.device):
            _lib.check(
                _lib.library().lf_mxfp4_dequantize(
                    t.codes.data_ptr(), t.scales.data_ptr(), out.numel() // BLOCK, out.data_ptr(), _lib.stream_of(t.device)))
    return out


def product(x, weight, *, experts, offsets, tokens, bias, swiglu, out, plan=None):
    """The product that ``mxfp4_linear``, ``fp8_linear`` and ``expert_linear`` share; ``experts`` is None for the dense ones.

    ``plan`` (``_lib.ExpertPlan``) forces a kernel; by default the library chooses.
    """
    import torch

    grouped = experts is not None
    quantised = isinstance(weight, (MXFP4Tensor, fp8.FP8Tensor))
    eight = isinstance(weight, fp8.FP8Tensor)
    if plan is None and (offsets is not None) == grouped and getattr(weight.codes if quantised else weight, "is_cuda", False):
        done = _lib.binding().product(x, weight, offsets, tokens, bias, swiglu, out)
        if done is not None:
            return done
    if eight:
        fp8.scaled(weight, "weight", 3 if grouped else 2, block_rows=fp8.BLOCK)
        shape, device = weight.shape, weight.device
    elif quantised:
        shape = packed(weight, "weight", 3 if grouped else 2)
        device = weight.device
    else:
        tensor(weight, "weight", 3, torch.bfloat16)
        if not weight.is_contiguous() or weight.data_ptr() % 16:
            raise ValueError("weight must be contiguous and 16-byte aligned")
        shape, device = tuple(weight.shape), weight.device
    n, k = shape[-2:]
    if n == 0 or k == 0 or (grouped and shape[0] == 0):
        raise ValueError("weight must not be empty")
    a = _lib.ExpertProduct()
    if isinstance(x, fp8.FP8Tensor):
        if not eight:
            raise ValueError("an FP8 x needs an FP8 weight")
        fp8.scaled(x, "x", 2, device, block_rows=1)
        x_rows = x.shape[0]
        if x.shape[1] != k:
            raise ValueError("x must have the weight's inner dimension")
        read = (x.codes, x.scales)
        a.x, a.x_fp8_scales = x.codes.data_ptr(), x.scales.data_ptr()
    elif isinstance(x, MXFP4Tensor):
        if not quantised or eight:
            raise ValueError("an MXFP4 x needs an MXFP4 weight")
        x_rows = packed(x, "x", 2, device)[0]
        if x.shape[1] != k:
            raise ValueError("x must have the weight's inner dimension")
        read = (x.codes, x.scales)
        a.x, a.x_scales = x.codes.data_ptr(), x.scales.data_ptr()
    else:
        tensor(x, "x", 2, torch.bfloat16, device)
        x_rows = x.shape[0]
        if x.shape[1] != k:
            raise ValueError("x must have the weight's inner dimension")
        a.x_stride = x.stride(0) if x_rows > 1 else k
        if k % 8 or x.stride(1) != 1 or a.x_stride < k or a.x_stride % 8 or x.data_ptr() % 16:
            raise ValueError("x rows must be 16-byte aligned with unit stride")
        read = (x,)
        a.x = x.data_ptr()
    if type(swiglu) is not bool:
        raise TypeError("swiglu must be a bool")
    if swiglu and n % 2:
        raise ValueError("swiglu needs as many gate as up rows")
    if swiglu and eight and n % (2 * fp8.BLOCK):
        raise ValueError("swiglu needs whole blocks of 128 FP8 gate and up rows")
    width = n // 2 if swiglu else n
    rows = x_rows
    if grouped:
        vector(offsets, "offsets", torch.int32, device, experts + 1)
        a.offsets = offsets.data_ptr()
        if tokens is not None:
            vector(tokens, "tokens", torch.int32, device)
            rows = tokens.numel()
            a.tokens = tokens.data_ptr()
            if rows and not x_rows:
                raise ValueError("x must hold the rows that tokens name")
    if bias is not None:
        tensor(bias, "bias", 2 if grouped else 1, torch.bfloat16, device)
        if tuple(bias.shape) != (shape[:2] if grouped else (n,)) or not bias.is_contiguous():
            raise ValueError("bias must be contiguous with an entry for each weight row")
        a.bias = bias.data_ptr()
    if out is None:
        out = torch.empty(rows, width, dtype=torch.bfloat16, device=device)
    tensor(out, "out", 2, torch.bfloat16, device)
    if out.shape != (rows, width) or (out.numel() and out.stride(1) != 1) or (rows > 1 and out.stride(0) < width):
        raise ValueError("out must be [rows, columns] with unit column stride")
    weights = (weight.codes, weight.scales) if quantised else (weight,)
    distinct_output(out, (*read, *weights, bias, offsets, tokens))
    require_arch(device)
    if rows == 0:
        return out
    a.x_rows, a.rows, a.n, a.k, a.experts = x_rows, rows, n, k, experts if grouped else 1
    a.w = weights[0].data_ptr()
    if eight:
        a.w_fp8_scales = weights[1].data_ptr()
    elif quantised:
        a.w_scales = weights[1].data_ptr()
    a.y, a.y_stride, a.swiglu = out.data_ptr(), out.stride(0) if rows > 1 else width, swiglu
    if plan is not None:
        a.plan = ctypes.pointer(plan)
    with torch.cuda.device(device):
        _lib.check(_lib.library().lf_expert_linear(ctypes.byref(a), _lib.stream_of(device)))
    return out


@ExperimentalAPI(reason="MXFP4 linear; gfx950 HIP kernel.")
def mxfp4_linear(x, weight: MXFP4Tensor, *, bias=None, swiglu: bool = False, out=None):
    """``x @ weight.T (+ bias)`` in bf16 for an MXFP4 ``weight`` ``[N, K]``, fp32 sums, rounded once.

    ``x`` is bf16 ``[M, K]`` with 16-byte aligned rows, or an ``MXFP4Tensor``
    ``[M, K]`` (``quantize_mxfp4``): both operands then go through the scaled
    4-bit matrix instructions. ``swiglu``: the weight is a merged ``[gate | up]``
    and the result ``silu(gate) * up``, ``[M, N / 2]``, in fp32 before its rounding.
    """
    if not isinstance(weight, MXFP4Tensor):
        raise TypeError("weight must be an MXFP4Tensor")
    return product(x, weight, experts=None, offsets=None, tokens=None, bias=bias, swiglu=swiglu, out=out)
