"""The mixture-of-experts block of ``examples/moe_block.py`` against the 64-bit oracle, eagerly and in a graph.

With bf16 activations a token's output passes four roundings to bf16 in a
chain (half 2^-8 each) beside fp32 sums: within 2^-6 of the largest output.
Quantised activations: an intermediate that differs by 2^-9 falls to another e2m1 code
for about one value in a hundred, by at most a third of it, so the relative L2
distance stays below sqrt(0.01) / 3 = 0.033; 2^-4 is allowed.
"""

import numpy as np
import pytest
import torch

from examples.moe_block import MoeBlock, adapters, capture, random_block
from oracle import experts as ox

pytestmark = pytest.mark.gpu

HIDDEN, INTER, SHARED, EXPERTS, TOP = 512, 576, 640, 12, 3


def f64(t):
    return t.double().cpu().numpy()


def values(t):
    return ox.values(t.codes.cpu().numpy(), t.scales.cpu().numpy())


def expected(block: MoeBlock, x, lora, rank):
    # (The product rounds the logits to bf16, which decides near ties: taken from the same product.)
    weights, chosen, *_ = ox.route(f64(x @ block.router.T), block.top_k)
    quantized = block.quantize_from is not None and len(x) >= block.quantize_from
    act = (lambda a: ox.values(*ox.quantize(a))) if quantized else (lambda a: a)
    gate_up, down = values(block.gate_up), values(block.down)
    xv = act(f64(x))
    s = ox.product(xv, values(block.shared_gate_up), swiglu=True)[0]
    y = act(s) @ values(block.shared_down).T
    if lora is not None:
        a = f64(lora.a_store).reshape(-1, rank, SHARED)
        b = f64(lora.b_store).reshape(len(a), HIDDEN, -1)[:, :, :rank]
        for t, slot in enumerate(lora.token_slots.tolist()):
            if slot >= 0:
                y[t] += float(lora.scales[slot]) * (b[slot] @ (a[slot] @ s[t]))
    for t in range(len(x)):
        for j in range(block.top_k):
            h = ox.product(xv[t : t + 1], gate_up[chosen[t, j]], swiglu=True)[0]
            y[t] += weights[t, j] * (act(h) @ down[chosen[t, j]].T)[0]
    return y


@pytest.mark.parametrize("quantize_from", [None, 100])
@pytest.mark.parametrize("tokens", [1, 24, 150])
def test_block(tokens, quantize_from, device):
    g = torch.Generator().manual_seed(tokens)
    block = random_block(HIDDEN, INTER, SHARED, EXPERTS, TOP, device, g, quantize_from)
    rank = 16
    lora = adapters(3, rank, SHARED, HIDDEN, tokens, device, g)
    lora.token_slots[::5] = -1
    x = torch.randn(tokens, HIDDEN, generator=g).bfloat16().to(device)
    for batch in (None, lora):
        y, want = f64(block(x, batch)), expected(block, x, batch, rank)
        if quantize_from is None or tokens < quantize_from:
            assert np.abs(y - want).max() <= 2.0**-6 * np.abs(want).max()
        else:
            assert np.linalg.norm(y - want) <= 2.0**-4 * np.linalg.norm(want)


@pytest.mark.parametrize("tokens", [3, 150])
def test_block_in_a_graph(tokens, device):
    g = torch.Generator().manual_seed(tokens)
    block = random_block(HIDDEN, INTER, SHARED, EXPERTS, TOP, device, g, quantize_from=100)
    lora = adapters(3, 8, SHARED, HIDDEN, tokens, device, g)
    x = torch.randn(tokens, HIDDEN, generator=g).bfloat16().to(device)
    graph, y = capture(block, x, lora)
    for _ in range(3):
        x.copy_(torch.randn(tokens, HIDDEN, generator=g).bfloat16().to(device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, block(x, lora))
