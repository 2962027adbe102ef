"""What the FP8 operators and the whole expert MLP refuse, without a GPU."""

import ctypes

import pytest
import torch

from loraforge_amd import _lib
from loraforge_amd.ops import FP8Tensor, MXFP4Tensor, dequantize_fp8, expert_linear, expert_mlp, fp8_linear, mxfp4_linear, quantize_fp8
from loraforge_amd.ops.fp8 import scaled

BF16 = torch.bfloat16


def f8(*shape, rows=128):
    return FP8Tensor(torch.zeros(*shape, dtype=torch.float8_e4m3fn),
                     torch.zeros(*shape[:-2], -(-shape[-2] // rows), -(-shape[-1] // 128)))


def test_python_checks():
    x = torch.zeros(4, 64, dtype=BF16)
    with pytest.raises(TypeError, match="torch.Tensor"):
        quantize_fp8([1.0])
    for bad in (x.half(), x.float(), x[0]):
        with pytest.raises(ValueError, match="dtype"):
            quantize_fp8(bad)
    for rows in (2, 64, True, 128.0):
        with pytest.raises(ValueError, match="1 or 128"):
            quantize_fp8(x, block_rows=rows)
    with pytest.raises(ValueError, match="same CUDA"):
        quantize_fp8(x)
    with pytest.raises(TypeError, match="FP8Tensor"):
        dequantize_fp8(x)
    with pytest.raises(ValueError, match="same CUDA"):
        dequantize_fp8(f8(4, 64))
    with pytest.raises(TypeError, match="FP8Tensor"):
        fp8_linear(x, x)
    with pytest.raises(TypeError, match="FP8Tensor"):
        fp8_linear(x, MXFP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)))
    with pytest.raises(TypeError, match="MXFP4Tensor"):
        mxfp4_linear(x, f8(8, 64))
    with pytest.raises(ValueError, match="same CUDA"):
        fp8_linear(x, f8(8, 64))
    with pytest.raises(ValueError, match="3D"):
        expert_linear(x, f8(8, 64), None)
    with pytest.raises(TypeError, match="FP8Tensor"):
        scaled(x, "t")
    with pytest.raises(ValueError, match="rows and columns"):
        scaled(FP8Tensor(torch.zeros(16, dtype=torch.float8_e4m3fn), torch.zeros(1)), "t")
    assert f8(3, 130, 272).shape == (3, 130, 272) and f8(3, 130, 272).scales.shape == (3, 2, 3)


def test_expert_mlp_checks():
    x, logits = torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 8)
    w = torch.zeros(8, 256, 256, dtype=BF16), torch.zeros(8, 256, 128, dtype=BF16)
    with pytest.raises(TypeError, match="gate_up"):
        expert_mlp(x, logits, None, w[1], 2)
    with pytest.raises(TypeError, match="down"):
        expert_mlp(x, logits, w[0], [1], 2)
    with pytest.raises(ValueError, match="3D"):
        expert_mlp(x, logits, w[0][0], w[1], 2)
    with pytest.raises(ValueError, match="same CUDA"):
        expert_mlp(x, logits, *w, 2)


def refused(match, status):
    with pytest.raises(ValueError, match=match):
        _lib.check(status)


def test_c_entry_points_refuse_without_device_work():
    lib = _lib.library()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(8)
    quantize = lambda x=p, m=1, r=2, k=64, stride=64, b=1, codes=p, scales=p: lib.lf_fp8_quantize(  # noqa: E731
        x, m, r, k, stride, b, codes, scales, None)
    refused("multiple of 16", quantize(k=40))
    refused("multiple of 16", quantize(k=0))
    refused("1 or 128", quantize(b=64))
    refused("x_stride", quantize(stride=48))
    refused("16-byte", quantize(x=odd))
    refused("16-byte", quantize(stride=68))
    refused("8-byte", quantize(codes=ctypes.c_void_p(4)))
    refused("null", quantize(scales=None))
    refused("int32", quantize(r=2**31))
    assert quantize(x=None, m=0) == quantize(x=None, r=0) == _lib.LF_OK
    refused("null", lib.lf_fp8_dequantize(p, None, 1, 2, 64, 1, p, None))
    refused("16-byte", lib.lf_fp8_dequantize(p, p, 1, 2, 64, 1, odd, None))
    refused("1 or 128", lib.lf_fp8_dequantize(p, p, 1, 2, 64, 2, p, None))


@pytest.mark.parametrize(
    "change,match",
    [
        (dict(k=40), "16 "),
        (dict(x_fp8_scales=16, w_fp8_scales=None), "needs an FP8 weight"),
        (dict(w_scales=16), "one type"),
        (dict(x_scales=16, x_fp8_scales=16), "one type"),
        (dict(x_scales=16), "needs an MXFP4 weight"),
        (dict(n=128, swiglu=1, y_stride=64), "whole blocks"),
        (dict(n=300, swiglu=1, y_stride=150), "whole blocks"),
        (dict(x=8), "16-byte"),
        (dict(w=4), "16-byte"),
        (dict(x_stride=68), "16-byte"),
        (dict(k=2**30), "a row's bytes"),
    ],
)
def test_c_product_refusals(change, match):
    a = _lib.ExpertProduct(x=16, w=16, w_fp8_scales=16, y=16, x_stride=64, x_rows=2, rows=2, n=32, k=64, experts=1, y_stride=32)
    for name, value in change.items():
        setattr(a, name, value)
    refused(match, _lib.library().lf_expert_linear(ctypes.byref(a), None))
