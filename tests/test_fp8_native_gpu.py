"""The FP8 operators and the whole expert MLP on the native call path, and a step that runs them together."""

import pytest
import torch

from loraforge_amd import _lib
from loraforge_amd.ops import (FP8Tensor, MXFP4Tensor, dequantize_fp8, expert_linear, expert_mlp, fp8_linear, quantize_fp8, quantize_mxfp4,
                               route_experts)
from oracle import experts as ox
from oracle import fp8 as of
from tests.test_expert_mlp_gpu import KINDS, case, close, expected, randn
from tests.test_native_calls_gpu import both, standing_in

pytestmark = pytest.mark.gpu


def same(a, b):
    if isinstance(a, FP8Tensor):
        return torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_forms(rows, device, monkeypatch):
    x = randn(1, 300, 528).to(device)
    for v in (x, x[:, :272], x[::2], x[:1], x.view(3, 100, 528)):
        taken, python = both(monkeypatch, lambda: quantize_fp8(v, block_rows=rows))
        assert same(taken, python)
        back, slow = both(monkeypatch, lambda: dequantize_fp8(taken))
        assert same(back, slow)


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_linear_forms(act, device, monkeypatch):
    w = quantize_fp8(randn(2, 512, 400).to(device), block_rows=128)
    bias = randn(3, 512).to(device)
    for m in (1, 17, 200):
        x = randn(m, m, 400).to(device)
        x = quantize_fp8(x) if act == "fp8" else x
        out = torch.empty(m, 600, dtype=torch.bfloat16, device=device)
        for kw in (dict(), dict(bias=bias), dict(swiglu=True), dict(bias=bias, swiglu=True), dict(out=out[:, 3:515])):
            taken, python = both(monkeypatch, lambda: fp8_linear(x, w, **kw).clone())
            assert same(taken, python), kw


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_expert_linear_forms(act, device, monkeypatch):
    w = quantize_fp8(randn(4, 6, 256, 272).to(device), block_rows=128)
    x = randn(5, 40, 272).to(device)
    r = route_experts(torch.randn(40, 6, generator=torch.Generator().manual_seed(6)).to(device), 2)
    xa = quantize_fp8(x) if act == "fp8" else x
    for kw in (dict(tokens=r.tokens), dict(tokens=r.tokens, swiglu=True), dict(tokens=r.tokens, bias=randn(7, 6, 256).to(device))):
        taken, python = both(monkeypatch, lambda: expert_linear(xa, w, r.offsets, **kw))
        assert same(taken, python), kw


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 8, 9, 70])
def test_expert_mlp_forms(kind, tokens, device, monkeypatch):
    x, logits, gate_up, down = case(kind, tokens, 12, 256, 128, device)
    base = randn(8, tokens, 256).to(device)
    out = torch.empty(tokens, 300, dtype=torch.bfloat16, device=device)
    wide = torch.zeros(tokens, 20, device=device)
    wide[:, 2:14] = logits
    for kw in (dict(), dict(base=base), dict(renormalize=False), dict(out=out[:, 5:261]), dict(base=base, out=base.clone())):
        for lo in (logits, logits.bfloat16(), wide[:, 2:14]):
            taken, python = both(monkeypatch, lambda: expert_mlp(x, lo, gate_up, down, 3, **kw).clone())
            assert same(taken, python), kw
    onto = [base.clone(), base.clone()]
    both(monkeypatch, lambda: expert_mlp(x, logits, gate_up, down, 3, base=onto[0], out=onto[0]))
    assert torch.isfinite(onto[0].float()).all()


def test_expert_mlp_that_the_native_path_declines(device, monkeypatch):
    """More choices than the one call takes, and weights of two types: the operators in a chain."""
    x, logits, gate_up, down = case("bf16", 70, 4, 256, 128, device)
    taken, python = both_chain(monkeypatch, lambda: expert_mlp(x, logits, gate_up, down, 2))
    assert same(taken, python)
    close(taken, expected(x, logits, gate_up, down, 2))
    mixed = quantize_fp8(down, block_rows=128)
    x, logits = x[:5], logits[:5]
    taken, python = both_chain(monkeypatch, lambda: expert_mlp(x, logits, gate_up, mixed, 2))
    assert same(taken, python)
    close(taken, expected(x, logits, gate_up, mixed, 2))


def both_chain(monkeypatch, call):
    """``call`` on either path, where the native one takes the chain's operators but not the call itself."""
    call()
    native = _lib.binding()

    class Noting:
        declined = []

        def __getattr__(self, name):
            def run(*args):
                answer = getattr(native, name)(*args)
                if name == "mlp":
                    self.declined.append(answer is None)
                return answer

            return run

    class Declines:
        def __getattr__(self, name):
            return lambda *args: None

    results = []
    for path in (Noting(), Declines()):
        with monkeypatch.context() as patch:
            patch.setattr(_lib, "_binding_module", path)
            results.append(call())
    torch.cuda.synchronize()
    assert Noting.declined and all(Noting.declined)
    return results


def test_scales_of_any_alignment(device):
    """MXFP4 scales at an odd address: the one call reads words, so the operators run in a chain."""
    x, logits, gate_up, down = case("mxfp4", 6, 8, 256, 128, device)
    store = torch.zeros(gate_up.scales.numel() + 1, dtype=torch.uint8, device=device)
    store[1:] = gate_up.scales.view(-1)
    odd = MXFP4Tensor(gate_up.codes, store[1:].view(gate_up.scales.shape))
    assert odd.scales.data_ptr() % 4
    close(expert_mlp(x, logits, odd, down, 3), expected(x, logits, gate_up, down, 3))


def test_library_calls_run_without_the_gil(device):
    """In the library's place stands PyGILState_Check: 0 (no GIL held) reads as success, 1 as a refused call."""
    import ctypes

    check = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
    native = _lib.binding()
    x, logits, gate_up, down = case("fp8", 4, 8, 256, 128, device)
    q = quantize_fp8(x)
    expert_mlp(x, logits, gate_up, down, 2)
    calls = {
        "lf_fp8_quantize": lambda: native.fp8_quantize(x, 1),
        "lf_fp8_dequantize": lambda: native.fp8_dequantize(q),
        "lf_expert_mlp": lambda: native.mlp(x, logits, gate_up, down, 2, True, None, None),
    }
    for name, call in calls.items():
        assert call() is not None, name
        with standing_in(**{name: check}):
            assert call() is not None, name


def test_no_gradients_through_the_native_path(device):
    x, logits, gate_up, down = case("bf16", 4, 8, 256, 128, device)
    native = _lib.binding()
    for i in range(4):
        args = [x, logits, gate_up, down]
        args[i] = args[i].clone().requires_grad_()
        assert native.mlp(*args, 2, True, None, None) is None
        with pytest.raises(ValueError, match="inference-only"):
            expert_mlp(*args, 2)
    assert native.fp8_quantize(x.clone().requires_grad_(), 1) is None


class Block:
    """A projection and a mixture of experts with FP8 weights on top of it, as a serving step runs them."""

    def __init__(self, hidden, experts, inter, device):
        self.proj = quantize_fp8(randn(20, hidden, hidden, std=hidden**-0.5).to(device), block_rows=128)
        self.router = randn(21, experts, hidden, std=hidden**-0.5).to(device)
        self.gate_up = quantize_fp8(randn(22, experts, 2 * inter, hidden, std=hidden**-0.5).to(device), block_rows=128)
        self.down = quantize_fp8(randn(23, experts, hidden, inter, std=inter**-0.5).to(device), block_rows=128)

    def __call__(self, x):
        a = quantize_fp8(x) if x.shape[0] > 16 else x  # (a decode step is bound by the weights' bytes)
        h = fp8_linear(a, self.proj)
        logits = h @ self.router.T
        return h, logits, expert_mlp(h, logits, self.gate_up, self.down, 4, base=x)


@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_a_step_of_the_operators_together(tokens, device):
    """Eager and captured: each operator's result from its own inputs, and every replay as the eager step."""
    block = Block(512, 16, 256, device)
    x = randn(24, tokens, 512).to(device)
    h, logits, y = block(x)
    if tokens > 16:
        a = quantize_fp8(x)
        want, bound = of.product(of.values(a.codes.view(torch.uint8).cpu().numpy(), a.scales.cpu().numpy()),
                                 of.values(block.proj.codes.view(torch.uint8).cpu().numpy(), block.proj.scales.cpu().numpy()), both=True)
    else:
        want, bound = ox.product(x.double().cpu().numpy(), of.values(block.proj.codes.view(torch.uint8).cpu().numpy(), block.proj.scales.cpu().numpy()))
    close(h, (want, bound))
    close(y, expected(h, logits, block.gate_up, block.down, 4, base=x, between=2.0**-16 + 2.0**-20))
    xs = x.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(xs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        _, _, ys = block(xs)
    for seed in range(4):
        xs.copy_(randn(30 + seed, tokens, 512).to(device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys, block(xs)[2])
        torch.cuda.synchronize()
