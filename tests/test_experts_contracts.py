"""What the MXFP4 and expert operators refuse, without a GPU."""

import ctypes

import pytest
import torch

from loraforge_amd import _lib
from loraforge_amd.ops import (
    MXFP4Tensor,
    combine_experts,
    dequantize_mxfp4,
    expert_linear,
    mxfp4_linear,
    quantize_mxfp4,
    route_experts,
)

BF16 = torch.bfloat16


def mx(*shape):
    return MXFP4Tensor(torch.zeros(*shape[:-1], shape[-1] // 2, dtype=torch.uint8),
                       torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.uint8))


def test_python_checks():
    x = torch.zeros(4, 64, dtype=BF16)
    with pytest.raises(TypeError, match="torch.Tensor"):
        quantize_mxfp4([1.0])
    with pytest.raises(ValueError, match="dtype"):
        quantize_mxfp4(x.half())
    with pytest.raises(ValueError, match="same CUDA"):
        quantize_mxfp4(x)
    with pytest.raises(TypeError, match="MXFP4Tensor"):
        dequantize_mxfp4(x)
    with pytest.raises(ValueError, match="same CUDA"):
        dequantize_mxfp4(mx(4, 64))
    with pytest.raises(TypeError, match="MXFP4Tensor"):
        mxfp4_linear(x, x)
    with pytest.raises(ValueError, match="same CUDA"):
        mxfp4_linear(x, mx(8, 64))
    with pytest.raises(ValueError, match="3D"):
        expert_linear(x, x, None)
    with pytest.raises(TypeError, match="weight"):
        expert_linear(x, None, None)
    with pytest.raises(ValueError, match="same CUDA"):
        route_experts(torch.zeros(2, 4), 2)
    with pytest.raises(ValueError, match="dtype"):
        route_experts(torch.zeros(2, 4, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="same CUDA"):
        combine_experts(x, torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 1))
    assert mx(3, 5, 64).shape == (3, 5, 64)


def refused(match, status):
    with pytest.raises(ValueError, match=match):
        _lib.check(status)


def test_c_entry_points_refuse_without_device_work():
    lib = _lib.library()
    p = ctypes.c_void_p(16)
    refused("multiple of 32", lib.lf_mxfp4_quantize(p, 0, 1, 48, 48, p, p, None))
    refused("x_stride", lib.lf_mxfp4_quantize(p, 0, 2, 64, 32, p, p, None))
    refused("16-byte", lib.lf_mxfp4_quantize(ctypes.c_void_p(8), 0, 1, 64, 64, p, p, None))
    refused("16-byte", lib.lf_mxfp4_quantize(p, 0, 2, 64, 68, p, p, None))
    refused("null", lib.lf_mxfp4_dequantize(p, None, 4, p, None))
    refused("16-byte", lib.lf_mxfp4_dequantize(p, p, 4, ctypes.c_void_p(2), None))
    assert lib.lf_mxfp4_quantize(None, 0, 0, 64, 64, None, None, None) == _lib.LF_OK
    route = lambda experts=8, top=2, stride=8, tokens=3, ws=None, size=0: lib.lf_route_experts(  # noqa: E731
        p, 0, tokens, experts, stride, top, 1, p, p, p, p, p, ws, size, None)
    refused("1..1024", route(experts=1025))
    refused("top_k", route(top=9))
    refused("top_k", route(experts=100, top=65, stride=100))
    refused("stride", route(stride=7))
    refused("int32", route(tokens=2**30))
    refused("workspace", route(tokens=65))
    assert lib.lf_route_experts_workspace_size(64, 8) == 0
    assert lib.lf_route_experts_workspace_size(65, 7) >= 3 * 8 * 4
    assert lib.lf_route_experts_workspace_size(10, 2000) == -1
    refused("cover n", lib.lf_combine_experts(p, 4, 7, p, p, 2, 1, 8, None, 0, p, 8, None))
    refused("null", lib.lf_combine_experts(p, 4, 8, None, p, 2, 1, 8, None, 0, p, 8, None))


@pytest.mark.parametrize(
    "change,match",
    [
        (dict(k=40), "multiple of 32"),
        (dict(w_scales=None, k=36), "or 8"),
        (dict(w_scales=None, x_scales=16), "needs an MXFP4 weight"),
        (dict(n=33, swiglu=1), "equal number"),
        (dict(experts=2), "offsets required"),
        (dict(tokens=16), "offsets required"),
        (dict(x=8), "16-byte"),
        (dict(w=4), "16-byte"),
        (dict(x_stride=68), "16-byte"),
        (dict(y_stride=31), "y_stride"),
        (dict(x_rows=1), "each row"),
        (dict(y=None), "null"),
        (dict(rows=2**31), "int32"),
        (dict(k=2**30, x_stride=2**30), "a row's bytes"),
        (dict(w_scales=None, k=2**30, x_stride=2**30), "a row's bytes"),
        (dict(n=0), "positive"),
    ],
)
def test_c_product_refusals(change, match):
    a = _lib.ExpertProduct(x=16, w=16, w_scales=16, y=16, x_stride=64, x_rows=2, rows=2, n=32, k=64, experts=1, y_stride=32)
    for name, value in change.items():
        setattr(a, name, value)
    refused(match, _lib.library().lf_expert_linear(ctypes.byref(a), None))


def plan(**sizes):
    a = _lib.ExpertProduct(**{**dict(x=16, w=16, y=16, x_rows=64, rows=64, n=4096, k=4096, experts=1), **sizes})
    p = _lib.ExpertPlan()
    _lib.check(_lib.library().lf_expert_linear_plan(ctypes.byref(a), ctypes.byref(p)))
    return p


def test_stream_plans_of_few_weight_rows():
    """Rows in passes of their own where a product's weight rows would leave CUs idle; refusal of other heights."""
    p = plan(rows=96, x_rows=96, n=528, k=7424, w_scales=16)
    assert (p.kernel, p.rows) == (_lib.LF_EXPERT_STREAM, 16)
    assert plan(rows=1024, x_rows=1024, n=528, k=7424, w_scales=16).kernel == _lib.LF_EXPERT_TILE
    a = _lib.ExpertProduct(x=16, w=16, w_scales=16, y=16, x_stride=64, x_rows=2, rows=2, n=32, k=64, experts=1, y_stride=32)
    a.plan = ctypes.pointer(_lib.ExpertPlan(_lib.LF_EXPERT_STREAM, 48, 16))
    refused("16, 32 or 64 rows", _lib.library().lf_expert_linear(ctypes.byref(a), None))


def test_plans():
    """Few rows stream the weights, many run in tiles, and what a kernel cannot take does not."""
    for rows in (1, 8, 16):
        assert plan(rows=rows, x_rows=rows, w_scales=16).kernel != _lib.LF_EXPERT_TILE
    for types in ({}, dict(w_scales=16), dict(w_scales=16, x_scales=16)):
        p = plan(rows=4096, x_rows=4096, **types)
        assert (p.kernel, p.rows, p.columns) == (_lib.LF_EXPERT_TILE, 256, 256)
        spread = plan(rows=32, x_rows=32, experts=128, offsets=16, **types)
        assert spread.kernel != _lib.LF_EXPERT_TILE
    assert plan(rows=4096, k=480, w_scales=16, x_scales=16).kernel == _lib.LF_EXPERT_STREAM
    assert plan(rows=4096, k=96, w_scales=16).kernel == _lib.LF_EXPERT_STREAM
    assert plan(rows=4096, x_rows=2**22, w_scales=16, x_scales=16).kernel == _lib.LF_EXPERT_STREAM
    forced = _lib.ExpertPlan(_lib.LF_EXPERT_TILE, 256, 256)
    a = _lib.ExpertProduct(x=16, x_scales=16, w=16, w_scales=16, y=16, x_rows=2, rows=2, n=32, k=480, experts=1, y_stride=32)
    for p, match in ((forced, "cannot run in tiles"), (_lib.ExpertPlan(_lib.LF_EXPERT_TILE, 96, 256), "64, 128, 192 or 256 rows"),
                     (_lib.ExpertPlan(_lib.LF_EXPERT_TILE, 64, 96), "columns"), (_lib.ExpertPlan(_lib.LF_EXPERT_STREAM, 0, 48), "columns"),
                     (_lib.ExpertPlan(7, 64, 64), "tiles")):
        a.k = 480 if p is forced else 512
        a.plan = ctypes.pointer(p)
        refused(match, _lib.library().lf_expert_linear(ctypes.byref(a), None))
