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


# --------------------------------------------------------------------------
# The whole expert MLP
# --------------------------------------------------------------------------


def mlp(**change):
    """A call that holds together but for ``change``; refused before any pointer is followed."""
    call = dict(x=16, x_stride=256, logits=16, logits_stride=8, tokens=4, hidden=256, inter=128, experts=8, top=2, type=_lib.LF_EXPERT_BF16,
                gate_up=16, down=16, y=16, y_stride=256)
    workspace, size = change.pop("workspace", 16), change.pop("size", None)
    a = _lib.ExpertMlp(**{**call, **change})
    if size is None:
        size = 1 << 30
    return _lib.library().lf_expert_mlp(ctypes.byref(a), ctypes.c_void_p(workspace), size, None)


@pytest.mark.parametrize(
    "change,match",
    [
        (dict(tokens=0), "as routing, products and sum"),
        (dict(tokens=129), "as routing, products and sum"),  # 258 choices of 8 experts
        (dict(tokens=2**62), "as routing, products and sum"),
        (dict(experts=1025, logits_stride=1025), "as routing, products and sum"),
        (dict(top=9), "as routing, products and sum"),
        (dict(top=0), "as routing, products and sum"),
        (dict(experts=200, top=65, logits_stride=200), "as routing, products and sum"),
        (dict(hidden=260, x_stride=264, y_stride=260), "as routing, products and sum"),
        (dict(inter=100), "as routing, products and sum"),
        (dict(inter=192, type=_lib.LF_EXPERT_FP8), "as routing, products and sum"),
        (dict(hidden=272, type=_lib.LF_EXPERT_MXFP4), "as routing, products and sum"),
        (dict(type=3), "as routing, products and sum"),
        (dict(type=-1), "as routing, products and sum"),
        (dict(workspace=None), "workspace of"),
        (dict(size=64), "workspace of"),
        (dict(workspace=24), "16-byte"),
        (dict(x=None), "null"),
        (dict(logits=None), "null"),
        (dict(gate_up=None), "null"),
        (dict(down=None), "null"),
        (dict(y=None), "null"),
        (dict(type=_lib.LF_EXPERT_FP8), "need scales"),
        (dict(type=_lib.LF_EXPERT_MXFP4, gate_up_scales=16), "need scales"),
        (dict(gate_up_scales=16, down_scales=16), "need scales"),
        (dict(type=_lib.LF_EXPERT_MXFP4, gate_up_scales=17, down_scales=16), "4-byte"),
        (dict(x=8), "16-byte"),
        (dict(x_stride=260), "16-byte"),
        (dict(x_stride=248), "16-byte"),
        (dict(gate_up=24), "16-byte"),
        (dict(down=8), "16-byte"),
        (dict(logits_stride=7), "row stride"),
        (dict(y_stride=255), "row strides"),
        (dict(x_stride=2**29), "within 2 GiB"),
        (dict(x_stride=2**62), "within 2 GiB"),
        (dict(base=16, base_stride=255), "row strides"),
    ],
)
def test_c_expert_mlp_refusals(change, match):
    refused(match, mlp(**change))


def test_c_expert_mlp_null_call():
    refused("null", _lib.library().lf_expert_mlp(None, ctypes.c_void_p(16), 64, None))


def test_expert_mlp_workspace():
    size = _lib.library().lf_expert_mlp_workspace_size
    bf16, mx, f8 = _lib.LF_EXPERT_BF16, _lib.LF_EXPERT_MXFP4, _lib.LF_EXPERT_FP8
    # Two launches: pairs of the intermediate and a table. Four: also the routing and rows of fp32.
    for kind in (bf16, mx, f8):
        assert 8 * 4 * 256 * 4 <= size(8, 64, 4, 512, 256, kind) < 8 * 4 * 256 * 4 + 4096
        assert size(9, 64, 4, 512, 256, kind) >= 9 * 4 * (256 + 512) * 4
        assert size(512, 64, 4, 512, 256, kind) > 0 > size(513, 64, 4, 512, 256, kind)
        assert size(1, 1024, 64, 512, 256, kind) > 0
        assert size(1, 64, 4, 2**24, 256, kind) == size(1, 64, 4, 512, 2**24, kind) == -1
    assert size(1, 64, 4, 520, 264, bf16) > 0 > size(1, 64, 4, 516, 264, bf16)
    assert size(1, 64, 4, 528, 256, f8) > 0 > size(1, 64, 4, 520, 256, f8)
    assert size(1, 64, 4, 544, 288, mx) > 0 > size(1, 64, 4, 528, 256, mx)


def test_fp8_plans():
    """Few rows stream the weights, many run in tiles of a height that leaves registers for a block's products."""
    def plan(**sizes):
        a = _lib.ExpertProduct(**{**dict(x=16, w=16, y=16, w_fp8_scales=16, x_stride=4096, x_rows=64, rows=64, n=4096, k=4096, experts=1), **sizes})
        p = _lib.ExpertPlan()
        _lib.check(_lib.library().lf_expert_linear_plan(ctypes.byref(a), ctypes.byref(p)))
        return p

    for types in ({}, dict(x_fp8_scales=16)):
        for rows in (1, 8, 16):
            assert plan(rows=rows, x_rows=rows, **types).kernel != _lib.LF_EXPERT_TILE
        for rows in (300, 1024, 4096, 8192):
            for n, k in ((4096, 4096), (11008, 4096), (12288, 4096), (1024, 8192)):
                p = plan(rows=rows, x_rows=rows, n=n, k=k, **types)
                assert p.kernel == _lib.LF_EXPERT_TILE
                assert p.rows <= ((192 if p.columns == 256 else 256) if types else (128 if p.columns == 256 else 192))
        assert plan(rows=32, x_rows=32, experts=128, offsets=16, **types).kernel != _lib.LF_EXPERT_TILE
        # Offsets of 31 bits in tiles: above, the weights are streamed.
        assert plan(rows=4096, x_rows=2**20, **types).kernel == _lib.LF_EXPERT_STREAM or not types
    assert plan(rows=4096, x_rows=2**19, x_fp8_scales=16).kernel != _lib.LF_EXPERT_TILE
    a = _lib.ExpertProduct(x=16, w=16, w_fp8_scales=16, y=16, x_stride=64, x_rows=2, rows=2, n=32, k=64, experts=1, y_stride=32)
    for rows, columns, x_scales in ((256, 64, None), (192, 256, None), (256, 256, 16)):
        a.x_fp8_scales = x_scales
        a.plan = ctypes.pointer(_lib.ExpertPlan(_lib.LF_EXPERT_TILE, rows, columns))
        refused("at most", _lib.library().lf_expert_linear(ctypes.byref(a), None))
