"""The MXFP4 and expert operators' native call path against their Python path: the same bits, and what it declines is served."""

import io

import pytest
import torch

from loraforge_amd.ops import MXFP4Tensor, combine_experts, dequantize_mxfp4, expert_linear, mxfp4_linear, quantize_mxfp4, route_experts
from tests.test_native_calls_gpu import both

pytestmark = pytest.mark.gpu


def parts(result):
    if isinstance(result, MXFP4Tensor):
        return [result.codes, result.scales]
    return list(vars(result).values()) if hasattr(result, "positions") else [result]


def agree(monkeypatch, call, native=True):
    for a, b in zip(*map(parts, both(monkeypatch, call, native)), strict=True):
        assert a.dtype == b.dtype and a.shape == b.shape and a.is_contiguous()
        assert torch.equal(torch.nan_to_num(a.float(), nan=7.0), torch.nan_to_num(b.float(), nan=7.0))


def randn(device, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=device).to(dtype)


def test_quantise_and_back(monkeypatch, device):
    store = randn(device, 9, 200)
    for x in (store[:, 8:168], randn(device, 2, 3, 64), randn(device, 96, dtype=torch.float32), store[:1, :64]):
        agree(monkeypatch, lambda x=x: quantize_mxfp4(x))
        agree(monkeypatch, lambda t=quantize_mxfp4(x): dequantize_mxfp4(t))
    empty = quantize_mxfp4(store[:0, :64])
    agree(monkeypatch, lambda: quantize_mxfp4(store[:0, :64]), native=False)
    agree(monkeypatch, lambda: dequantize_mxfp4(empty), native=False)


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_products(monkeypatch, rows, device):
    store = randn(device, rows, 1040)
    x = store[:, 8:1032]
    w = quantize_mxfp4(randn(device, 3, 192, 1024) * 0.05)
    dense = MXFP4Tensor(w.codes[1], w.scales[1])
    offsets = torch.tensor([0, rows // 2, rows // 2, rows], dtype=torch.int32, device=device)
    tokens = torch.randint(0, rows, (rows + 5,), dtype=torch.int32, device=device)
    whole = torch.tensor([0, 2, 3, rows + 5], dtype=torch.int32, device=device)
    for xi in (x, quantize_mxfp4(x)):
        for swiglu in (False, True):
            agree(monkeypatch, lambda: mxfp4_linear(xi, dense, bias=store[0, :192].contiguous(), swiglu=swiglu))
            agree(monkeypatch, lambda: expert_linear(xi, w, offsets, bias=randn_like(w), swiglu=swiglu))
        agree(monkeypatch, lambda: expert_linear(xi, w, whole, tokens=tokens))
    agree(monkeypatch, lambda: expert_linear(x, dequantize_mxfp4(w), offsets))
    apart = torch.zeros(rows, 210, dtype=torch.bfloat16, device=device)
    for out in (torch.empty(rows, 192, dtype=torch.bfloat16, device=device), apart[:, 5:197]):
        for a in both(monkeypatch, lambda: mxfp4_linear(x, dense, out=out)):
            assert a is out and torch.equal(out, mxfp4_linear(x, dense))
    assert not apart[:, :5].any() and not apart[:, 197:].any()


def randn_like(w):
    return torch.linspace(-1, 1, w.shape[0] * w.shape[1], device=w.device).bfloat16().reshape(w.shape[:2])


@pytest.mark.parametrize("tokens", [5, 100])
def test_routing_and_combine(monkeypatch, tokens, device):
    logits = randn(device, tokens, 80, dtype=torch.float32)[:, 3:43]
    for renormalize in (True, False):
        agree(monkeypatch, lambda: route_experts(logits, 4, renormalize=renormalize))
        agree(monkeypatch, lambda: route_experts(logits.bfloat16(), 1, renormalize=renormalize))
    r = route_experts(logits, 4)
    rows = randn(device, tokens * 4, 264)[:, :256]
    base = randn(device, tokens, 264)[:, 4:260]
    agree(monkeypatch, lambda: combine_experts(rows, r.positions, r.weights))
    agree(monkeypatch, lambda: combine_experts(rows, r.positions, r.weights, base=base))
    agree(monkeypatch, lambda: route_experts(logits[:0], 4), native=False)
    expected = combine_experts(rows, r.positions, r.weights, base=base)
    out = torch.empty(tokens, 264, dtype=torch.bfloat16, device=device)[:, 8:]
    for a in both(monkeypatch, lambda: combine_experts(rows, r.positions, r.weights, base=base, out=out)):
        assert a is out and torch.equal(out, expected)
    bases = iter([base.clone() for _ in range(3)])  # in place, each call on a base of its own

    def onto():
        b = next(bases)
        return combine_experts(rows, r.positions, r.weights, base=b, out=b)

    for a in both(monkeypatch, onto):
        assert torch.equal(a, expected)
    for other in (dict(), dict(base=rows[:tokens])):
        with pytest.raises(ValueError, match="share storage"):
            combine_experts(rows, r.positions, r.weights, out=rows[1 : tokens + 1], **other)


def test_refusals_stay_the_operators_own(device):
    x = randn(device, 4, 64)
    w = quantize_mxfp4(randn(device, 2, 32, 64))
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device=device)
    dense = MXFP4Tensor(w.codes[0], w.scales[0])
    cases = [
        (lambda: quantize_mxfp4(x[:, :48]), "multiple of 32"),
        (lambda: quantize_mxfp4(x[:, 1:33]), "16-byte aligned"),
        (lambda: quantize_mxfp4(x.float().requires_grad_()), "inference-only"),
        (lambda: dequantize_mxfp4(MXFP4Tensor(w.codes, w.scales[..., :1].contiguous())), "one scale"),
        (lambda: mxfp4_linear(x[:, :32], dense), "inner dimension"),
        (lambda: mxfp4_linear(x.t(), quantize_mxfp4(randn(device, 8, 32)).__class__(w.codes[0][:, :16].contiguous(), w.scales[0][:, :1].contiguous())), "inner dimension"),
        (lambda: mxfp4_linear(x.requires_grad_(), dense), "inference-only"),
        (lambda: expert_linear(x.detach(), w, offsets[:2]), "offsets must be contiguous"),
        (lambda: expert_linear(x.detach(), w, offsets.long()), "offsets must be 1D"),
        (lambda: expert_linear(x.detach(), w, offsets, tokens=offsets.float()), "tokens must be 1D"),
        (lambda: expert_linear(x.detach(), w, offsets, bias=randn(device, 2, 16)), "bias must be contiguous"),
        (lambda: expert_linear(quantize_mxfp4(x.detach()), dequantize_mxfp4(w), offsets), "needs an MXFP4 weight"),
        (lambda: mxfp4_linear(x.detach(), dense, out=dense.codes), "out must be"),
        (lambda: mxfp4_linear(x.detach(), dense, out=torch.empty(4, 31, dtype=torch.bfloat16, device=device)), "out must be"),
        (lambda: mxfp4_linear(x.detach(), MXFP4Tensor(w.codes[0, :31], w.scales[0, :31]), swiglu=True), "as many gate as up"),
        (lambda: route_experts(x.detach(), 0), "top_k"),
        (lambda: route_experts(x.detach(), 65), "top_k"),
        (lambda: route_experts(x.detach().t(), 2), "unit column stride"),
        (lambda: combine_experts(x.detach(), offsets.reshape(1, 3), torch.ones(1, 2, device=device)), "positions and weights"),
        (lambda: combine_experts(x.detach(), offsets.reshape(1, 3), torch.ones(1, 3, device=device), base=x.detach()), "base must be"),
    ]
    for call, match in cases:
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: mxfp4_linear(x.detach(), dense, swiglu=1), lambda: route_experts(x.detach(), 2, renormalize=1)):
        with pytest.raises(TypeError, match="bool"):
            call()
    shared = torch.zeros(8, 64, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="share storage"):
        mxfp4_linear(shared[:4], dense, out=shared[4:, :32])


@pytest.mark.parametrize("tokens", [5, 100])
def test_routing_can_be_saved(tokens, device):
    """No two results of different types lie in one storage: torch.save refuses such tensors."""
    r = route_experts(randn(device, tokens, 40), 3)
    results = (r.weights, r.experts, r.offsets, r.tokens, r.positions)
    file = io.BytesIO()
    torch.save(results, file)
    file.seek(0)
    for a, b in zip(results, torch.load(file, weights_only=True)):
        assert torch.equal(a, b)
