"""Expert routing and the weighted sum of the experts' rows on gfx950, against the 64-bit oracle.

Choices, order and places have to be equal. Weights are fp32 quotients of
exponentials: each exponential is within 2 ulp plus the rounding of its
argument (2^-24 of up to 100), each sum of E terms within E 2^-24.
"""

import numpy as np
import pytest
import torch

from loraforge_amd.ops import MXFP4Tensor, combine_experts, expert_linear, quantize_mxfp4, route_experts
from oracle import experts as ox

pytestmark = pytest.mark.gpu


def check_route(logits, top, renormalize=True):
    r = route_experts(logits, top, renormalize=renormalize)
    weights, experts, offsets, tokens, positions = ox.route(logits.double().cpu().numpy(), top, renormalize)
    assert np.array_equal(r.experts.cpu().numpy(), experts)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.tokens.cpu().numpy(), tokens)
    assert np.array_equal(r.positions.cpu().numpy(), positions)
    got = r.weights.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(weights))
    limit = (logits.shape[1] + 250) * 2.0**-24 * np.abs(weights) + 2.0**-126
    assert np.nanmax(np.abs(got - weights) - limit, initial=-1.0) <= 0


def logits_of(seed, tokens, experts, dtype, device, scale=2.0):
    return (torch.randn(tokens, experts, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(
    "tokens,experts,top",
    [(1, 1, 1), (1, 8, 2), (3, 60, 6), (16, 128, 8), (64, 64, 64), (65, 8, 8), (130, 128, 8), (300, 257, 5), (77, 1024, 64),
     (2, 1024, 9), (1000, 63, 3), (5000, 16, 4)],
)
def test_route(tokens, experts, top, dtype, device):
    check_route(logits_of(tokens, tokens, experts, dtype, device), top, renormalize=tokens % 2 == 0)


@pytest.mark.parametrize("tokens", [5, 200])
def test_route_ties_go_to_the_lowest_expert(tokens, device):
    logits = torch.randint(-2, 3, (tokens, 70), generator=torch.Generator().manual_seed(1)).float()
    logits[0] = 0.0
    logits[1, ::2] = -0.0  # equal to +0
    logits[1, 1::2] = 0.0
    check_route(logits.to(device), 7)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens", [9, 150])
def test_route_masked(tokens, renormalize, device):
    """Experts that are not allowed, tokens that may choose fewer than k or none, masks of the type's lowest value."""
    logits = logits_of(2, tokens, 40, torch.float32, "cpu")
    logits[torch.rand(tokens, 40, generator=torch.Generator().manual_seed(3)) < 0.85] = -np.inf
    logits[0] = -np.inf
    logits[1] = -np.inf
    logits[1, 39] = -3.0
    logits[2] = torch.finfo(torch.float32).min  # a number: allowed, equal probabilities
    logits[3, :20] = torch.finfo(torch.float32).min
    check_route(logits.to(device), 6, renormalize)


def test_route_all_masked(device):
    logits = torch.full((70, 12), -np.inf, device=device)
    r = route_experts(logits, 3)
    assert not r.offsets.any() and (r.experts == -1).all() and (r.tokens == -1).all() and (r.positions == -1).all()
    assert not r.weights.any()


def test_route_not_finite_logits(device):
    logits = logits_of(5, 8, 20, torch.float32, "cpu")
    logits[2, 4], logits[3, 7], logits[4, :] = float("nan"), float("inf"), float("nan")
    logits = logits.to(device)
    r = route_experts(logits, 3)
    assert torch.isnan(r.weights[2]).all() and torch.isnan(r.weights[3]).all()
    assert r.experts[3, 0] == 7 and 4 not in r.experts[2].tolist() and (r.experts[4] == -1).all()
    assert torch.isfinite(r.weights[[0, 1, 5, 6, 7]]).all()


def test_route_large_logits_and_strided_rows(device):
    store = logits_of(6, 33, 90, torch.float32, device, scale=30.0)
    check_route(store[:, 5:85], 8, renormalize=False)
    check_route(logits_of(7, 0, 16, torch.float32, device), 2)


@pytest.mark.parametrize("tokens,top,n", [(1, 1, 8), (24, 4, 4096), (7, 3, 1001), (300, 8, 520), (5, 64, 64)])
@pytest.mark.parametrize("base", [False, True])
def test_combine(tokens, top, n, base, device):
    rng = np.random.default_rng(tokens)
    rows = torch.from_numpy(rng.standard_normal((tokens * top, n))).bfloat16()
    positions = rng.permutation(tokens * top).reshape(tokens, top).astype(np.int32)
    positions[rng.random((tokens, top)) < 0.2] = -1
    weights = rng.random((tokens, top)).astype(np.float32)
    weights[positions < 0] = np.nan  # beside a position of -1 nothing is read
    b = torch.from_numpy(rng.standard_normal((tokens, n))).bfloat16() if base else None
    y = combine_experts(rows.to(device), torch.from_numpy(positions).to(device), torch.from_numpy(weights).to(device),
                        base=None if b is None else b.to(device))
    term = np.where(positions[..., None] >= 0, np.nan_to_num(weights)[..., None] * rows.double().numpy()[np.maximum(positions, 0)], 0.0)
    start = np.zeros((tokens, n)) if b is None else b.double().numpy()
    expected, magnitude = start + term.sum(1), np.abs(start) + np.abs(term).sum(1)
    error = np.abs(y.double().cpu().numpy() - expected)
    assert (error <= 2.0**-8 * np.abs(expected) + (top + 1) * 2.0**-23 * magnitude).all()


def test_combine_onto_its_base_strided(device):
    rows = torch.randn(12, 40, device=device).bfloat16()[:, 8:32]
    store = torch.randn(4, 48, device=device).bfloat16()
    before = store.clone()
    positions = torch.arange(12, dtype=torch.int32, device=device).reshape(4, 3)
    weights = torch.rand(4, 3, device=device)
    expected = combine_experts(rows.contiguous(), positions, weights, base=store[:, 4:28].contiguous())
    y = combine_experts(rows, positions, weights, base=store[:, 4:28], out=store[:, 4:28])
    assert torch.equal(y, expected) and torch.equal(store[:, 4:28], expected)
    assert torch.equal(store[:, :4], before[:, :4]) and torch.equal(store[:, 28:], before[:, 28:])


@pytest.mark.parametrize("tokens", [3, 90])
def test_routed_experts_end_to_end(tokens, device):
    """Router to output in a captured graph, replayed on new inputs: each replay equals the eager chain."""
    g = torch.Generator().manual_seed(tokens)
    hidden, inter, experts, top = 256, 192, 12, 3
    w1 = quantize_mxfp4((torch.randn(experts, 2 * inter, hidden, generator=g) * 0.05).bfloat16().to(device))
    w2 = (torch.randn(experts, hidden, inter, generator=g) * 0.05).bfloat16().to(device)
    assert isinstance(w1, MXFP4Tensor)

    def block(x, logits):
        r = route_experts(logits, top)
        h = expert_linear(x, w1, r.offsets, tokens=r.tokens, swiglu=True)
        return combine_experts(expert_linear(h, w2, r.offsets), r.positions, r.weights, base=x)

    x = torch.randn(tokens, hidden, generator=g).bfloat16().to(device)
    logits = torch.randn(tokens, experts, generator=g).to(device)
    eager = block(x, logits)
    weights, chosen, *_ = ox.route(logits.double().cpu().numpy(), top)
    xv, w1v, w2v = x.double().cpu().numpy(), ox.values(w1.codes.cpu().numpy(), w1.scales.cpu().numpy()), w2.double().cpu().numpy()
    expected = xv.copy()
    for t in range(tokens):
        for j in range(top):
            h = ox.product(xv[t : t + 1], w1v[chosen[t, j]], swiglu=True)[0]
            expected[t] += weights[t, j] * (h @ w2v[chosen[t, j]].T)[0]
    scale = np.abs(expected).max()
    assert np.abs(eager.double().cpu().numpy() - expected).max() <= 2.0**-6 * scale  # three bf16 roundings in a chain
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, logits)
    for seed in range(3):
        x.copy_(torch.randn(tokens, hidden, generator=g).bfloat16().to(device))
        logits.copy_(torch.randn(tokens, experts, generator=g).to(device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, block(x, logits))
