"""The whole mixture-of-experts MLP (``expert_mlp``) against the 64-bit oracle.

With a = silu(gate) up of an expert in 64 bits, a call of more than 32 choices an expert holds a in bf16: off by
2^-8 of it (half a step; a second 2^-9 for a weight's or the fp32
sums' share), so an output by (2^-8 + 2^-9) of the sum of magnitudes of its down terms, plus the fp32
bound of both products, plus half a bf16 step of itself. All others hold a (or a times its routing weight) as a pair of bf16,
off by 2^-16: they are within that bound too, and at 2^-16 + 2^-20 in
``test_keeps_16_bits_between_the_products`` and in ``test_expert_mlp_edges_gpu.py``.
"""

import numpy as np
import pytest
import torch

from loraforge_amd.ops import (FP8Tensor, MXFP4Tensor, combine_experts, expert_linear, expert_mlp, quantize_fp8, quantize_mxfp4,
                               route_experts)
from oracle import experts as ox
from oracle import fp8 as of

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "fp8", "mxfp4"]


def randn(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).bfloat16()


def weights(kind, seed, *shape, device, std=0.05):
    w = randn(seed, *shape, std=std).to(device)
    if kind == "fp8":
        return quantize_fp8(w, block_rows=128)
    return quantize_mxfp4(w) if kind == "mxfp4" else w


def values(w):
    if isinstance(w, FP8Tensor):
        return of.values(w.codes.view(torch.uint8).cpu().numpy(), w.scales.cpu().numpy())
    if isinstance(w, MXFP4Tensor):
        return ox.values(w.codes.cpu().numpy(), w.scales.cpu().numpy())
    return w.double().cpu().numpy()


def expected(x, logits, gate_up, down, top, renormalize=True, base=None, between=2.0**-8 + 2.0**-9):
    """Output and its bound in 64 bits; ``between``: how far, relative to it, what lies between the products may be off."""
    xv, gu, dn = x.double().cpu().numpy(), values(gate_up), values(down)
    share, chosen, *_ = ox.route(logits.double().cpu().numpy(), top, renormalize)
    y = np.zeros((len(xv), dn.shape[1])) if base is None else base.double().cpu().numpy()
    bound = 2.0**-23 * np.abs(y)
    for t in range(len(xv)):
        for j in range(top):
            e = chosen[t, j]
            if e < 0:
                continue
            h, h_bound = ox.product(xv[t : t + 1], gu[e], None, True)
            term, term_bound = ox.product(h, dn[e])
            y[t] += share[t, j] * term[0]
            bound[t] += share[t, j] * (term_bound + (between * np.abs(h) + h_bound) @ np.abs(dn[e]).T)[0]
            bound[t] += 2.0**-21 * share[t, j] * np.abs(term[0])
    return y, bound


def close(got, want):
    y, (v, bound) = got.double().cpu().numpy(), want
    assert y.shape == v.shape and np.array_equal(np.isnan(y), np.isnan(v))
    limit = bound + 2.0**-8 * (np.abs(v) + bound) + 2.0**-133
    worst = np.nanmax(np.abs(y - v) - limit, initial=-np.inf)
    assert worst <= 0, worst


def case(kind, tokens, experts, hidden, inter, device, seed=1):
    return (randn(seed, tokens, hidden).to(device), torch.randn(tokens, experts, generator=torch.Generator().manual_seed(seed + 1)).to(device) * 1.5,
            weights(kind, seed + 2, experts, 2 * inter, hidden, device=device), weights(kind, seed + 3, experts, hidden, inter, device=device))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 2, 3, 7, 15, 16, 17, 31, 32, 33, 48, 64, 65, 130])
def test_tokens(kind, tokens, device):
    x, logits, gate_up, down = case(kind, tokens, 24, 512, 256, device, seed=tokens)
    close(expert_mlp(x, logits, gate_up, down, 4), expected(x, logits, gate_up, down, 4))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize(
    "experts,top,hidden,inter",
    [(1, 1, 128, 128), (8, 8, 256, 128), (3, 2, 640, 384), (60, 6, 1152, 128), (300, 8, 128, 256), (9, 1, 4096, 640), (5, 3, 2176, 1408),
     (1024, 64, 128, 128)],
)
def test_sizes(kind, experts, top, hidden, inter, device):
    for tokens in (1, 6, 20):
        x, logits, gate_up, down = case(kind, tokens, experts, hidden, inter, device, seed=experts)
        base = randn(9, tokens, hidden).to(device)
        close(expert_mlp(x, logits.bfloat16(), gate_up, down, top, renormalize=False, base=base),
              expected(x, logits.bfloat16(), gate_up, down, top, False, base))


@pytest.mark.parametrize("kind,hidden,inter", [("bf16", 136, 72), ("bf16", 520, 264), ("fp8", 144, 128), ("fp8", 528, 256), ("mxfp4", 96, 32),
                                               ("mxfp4", 544, 288), ("bf16", 24, 8)])
def test_widths_that_are_no_multiple_of_128(kind, hidden, inter, device):
    for tokens in (1, 5, 40):
        x, logits, gate_up, down = case(kind, tokens, 10, hidden, inter, device, seed=hidden)
        close(expert_mlp(x, logits, gate_up, down, 3), expected(x, logits, gate_up, down, 3))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 16, 40])
def test_every_token_to_the_same_experts(kind, tokens, device):
    x, logits, gate_up, down = case(kind, tokens, 12, 384, 256, device)
    logits[:, 3] += 50.0
    logits[:, 11] += 40.0
    close(expert_mlp(x, logits, gate_up, down, 2), expected(x, logits, gate_up, down, 2))


@pytest.mark.parametrize("kind", KINDS)
def test_masked_experts_and_tokens_without_any(kind, device):
    """-inf marks an expert that a token may not choose: what fewer than top_k leave, and a token that has none."""
    x, logits, gate_up, down = case(kind, 12, 10, 256, 128, device)
    logits[torch.rand(12, 10, generator=torch.Generator().manual_seed(3)) < 0.7] = -np.inf
    logits[4] = -np.inf
    base = randn(5, 12, 256).to(device)
    for b in (None, base):
        y = expert_mlp(x, logits, gate_up, down, 3, base=b)
        close(y, expected(x, logits, gate_up, down, 3, base=b))
        assert torch.equal(y[4], torch.zeros_like(y[4]) if b is None else b[4])
    none = torch.full_like(logits, -np.inf)
    assert torch.equal(expert_mlp(x, none, gate_up, down, 3, base=base), base)
    assert not expert_mlp(x, none, gate_up, down, 3).any()


@pytest.mark.parametrize("kind", KINDS)
def test_ties_go_to_the_lowest_expert(kind, device):
    x, logits, gate_up, down = case(kind, 8, 16, 256, 128, device)
    logits = torch.round(logits)
    close(expert_mlp(x, logits, gate_up, down, 5), expected(x, logits, gate_up, down, 5))
    same = torch.zeros_like(logits)
    close(expert_mlp(x, same, gate_up, down, 4), expected(x, same, gate_up, down, 4))


@pytest.mark.parametrize("kind", KINDS)
def test_nan_and_infinity_stay_in_their_token(kind, device):
    """A token with NaN or infinity in x or NaN in its logits: its row, and no other one, also among those of the same expert."""
    x, logits, gate_up, down = case(kind, 14, 6, 256, 128, device)
    clean = expert_mlp(x, logits, gate_up, down, 2)
    x, logits = x.clone(), logits.clone()
    x[3, 17] = float("nan")
    x[6] = float("inf")
    logits[9, 1] = float("nan")
    logits[11, 2] = float("inf")
    y = expert_mlp(x, logits, gate_up, down, 2)
    rest = [t for t in range(14) if t not in (3, 6, 9, 11)]
    assert torch.isnan(y[[3, 9, 11]]).all()
    assert not torch.isfinite(y[6]).any()
    assert torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("kind", KINDS)
def test_bad_weights_of_an_expert_reach_only_its_tokens(kind, device):
    x, logits, gate_up, down = case(kind, 9, 8, 256, 128, device)
    clean = expert_mlp(x, logits, gate_up, down, 2)
    _, chosen, *_ = ox.route(logits.double().cpu().numpy(), 2)
    for w in (gate_up, down):
        held = w if kind == "bf16" else w.scales
        if kind == "mxfp4":
            held[5] = 255
        else:
            held[5] = float("nan")
        y = expert_mlp(x, logits, gate_up, down, 2)
        hit = (chosen == 5).any(1)
        assert hit.any() and not hit.all()
        assert torch.isnan(y[torch.from_numpy(hit)]).all() and torch.equal(y[torch.from_numpy(~hit)], clean[torch.from_numpy(~hit)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [5, 20, 70])
def test_strides_in_place_and_repeated(kind, tokens, device):
    x, logits, gate_up, down = case(kind, tokens, 16, 384, 128, device)
    want = expert_mlp(x, logits, gate_up, down, 4)
    store = torch.full((tokens, 408), float("nan"), dtype=torch.bfloat16, device=device)
    store[:, 8:392] = x
    wide = torch.full((tokens, 40), float("nan"), device=device)
    wide[:, 3:19] = logits
    out = torch.zeros(tokens, 400, dtype=torch.bfloat16, device=device)
    y = expert_mlp(store[:, 8:392], wide[:, 3:19], gate_up, down, 4, out=out[:, 5:389])
    assert y.data_ptr() == out[:, 5:].data_ptr() and torch.equal(y, want)
    assert not out[:, :5].any() and not out[:, 389:].any()
    base = randn(8, tokens, 384).to(device)
    want = expert_mlp(x, logits, gate_up, down, 4, base=base)
    for _ in range(3):
        assert torch.equal(expert_mlp(x, logits, gate_up, down, 4, base=base), want)
    onto = base.clone()
    assert expert_mlp(x, logits, gate_up, down, 4, base=onto, out=onto) is onto and torch.equal(onto, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,experts", [(1, 24), (8, 24), (9, 24), (33, 24), (130, 24), (192, 24), (70, 9), (20, 300)])
def test_keeps_16_bits_between_the_products(kind, tokens, experts, device):
    """32 choices an expert or fewer: a pair of bf16 is off by 2^-8 of 2^-8 of the value, the fp32 activation by 2^-20."""
    x, logits, gate_up, down = case(kind, tokens, experts, 512, 256, device, seed=tokens)
    want, bound = expected(x, logits, gate_up, down, 4, between=2.0**-16 + 2.0**-20)
    y = expert_mlp(x, logits, gate_up, down, 4)
    close(y, (want, bound))
    # y's rounding alone: an error uniform within half a step either way has 2^-7 / sqrt(12) of the power of two below the
    # value in the root mean square, which of normal values is 0.00166 of their deviation; with the intermediate
    # in bf16 there would be another 0.0017 or so, 0.0024 of both.
    off = (y.double().cpu().numpy() - want).std() / want.std()
    assert off <= 2.0**-9


@pytest.mark.parametrize("tokens", [8, 9])
def test_rows_of_x_far_apart(tokens, device):
    """The last rows of long sequences: 2 GiB and more between the first and the last."""
    x, logits, gate_up, down = case("bf16", tokens, 8, 256, 128, device)
    apart = torch.empty(tokens, 2**27 + 2**25, dtype=torch.bfloat16, device=device)
    far = apart[:, 64:320]
    far.copy_(x)
    assert torch.equal(expert_mlp(far[:2], logits[:2], gate_up, down, 2), expert_mlp(x[:2], logits[:2], gate_up, down, 2))
    close(expert_mlp(far, logits, gate_up, down, 2), expected(x, logits, gate_up, down, 2))


@pytest.mark.parametrize("tokens", [3, 20])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_weights_past_32_bits(kind, tokens, device):
    """Experts whose weights lie past 4 GiB: as in a tensor of those experts alone."""
    experts, hidden, inter = 80, 4096, 8192
    x, _, gate_up, down = case(kind, tokens, 2, hidden, inter, device)

    def spread(w):
        t = w if kind == "bf16" else w.codes
        big = torch.zeros(experts, *t.shape[1:], dtype=t.dtype, device=device)
        raw, part = (big, t) if kind == "bf16" else (big.view(torch.uint8), t.view(torch.uint8))
        raw[0], raw[experts - 1] = part[0], part[1]
        if kind == "bf16":
            return big
        scales = torch.zeros(experts, *w.scales.shape[1:], device=device)
        scales[0], scales[experts - 1] = w.scales[0], w.scales[1]
        return FP8Tensor(big, scales)

    few = torch.randn(tokens, 2, device=device)
    logits = torch.full((tokens, experts), -np.inf, device=device)
    logits[:, 0], logits[:, experts - 1] = few[:, 0], few[:, 1]
    y, alone = expert_mlp(x, logits, spread(gate_up), spread(down), 2), expert_mlp(x, few, gate_up, down, 2)
    if tokens <= 8:
        assert torch.equal(y, alone)
        return
    # (Of 80 experts the products may run in another kernel, whose sums have another order: the formula and the
    # bound of ``expected``, on the GPU in 64 bits.)
    def sums(a, w):
        return a @ w.T, (2.0 * a.shape[1] + 16.0) * 2.0**-24 * (a.abs() @ w.abs().T)

    share = few.double().softmax(1)
    want = torch.zeros(tokens, hidden, dtype=torch.float64, device=device)
    bound = torch.zeros_like(want)
    for e in range(2):
        gu, dn = (torch.from_numpy(values(w[e : e + 1] if kind == "bf16" else FP8Tensor(w.codes[e : e + 1], w.scales[e : e + 1]))[0]).to(device)
                  for w in (gate_up, down))
        (g, u), (dg, du) = (t.chunk(2, 1) for t in sums(x.double(), gu))
        act = g / (1.0 + (-g).exp())
        h = act * u
        h_bound = 1.1 * dg * (u.abs() + du) + (act.abs() + 1.1 * dg) * du + 2.0**-21 * h.abs()
        term, term_bound = sums(h, dn)
        want += share[:, e : e + 1] * term
        bound += share[:, e : e + 1] * (term_bound + ((2.0**-16 + 2.0**-20) * h.abs() + h_bound) @ dn.abs().T + 2.0**-21 * term.abs())
    for got in (y, alone):
        close(got, (want.cpu().numpy(), bound.cpu().numpy()))


def test_no_tokens(device):
    x, logits, gate_up, down = case("bf16", 2, 4, 128, 128, device)
    assert expert_mlp(x[:0], logits[:0], gate_up, down, 2).shape == (0, 128)


@pytest.mark.parametrize("tokens", [3, 24, 70])
@pytest.mark.parametrize("kind", KINDS)
def test_agrees_with_the_operators_in_a_chain(kind, tokens, device):
    """Against route, product, product and combine: the same bf16 rounding of the intermediate, but for the weight in it."""
    x, logits, gate_up, down = case(kind, tokens, 32, 640, 256, device)
    r = route_experts(logits, 4)
    h = expert_linear(x, gate_up, r.offsets, tokens=r.tokens, swiglu=True)
    chain = combine_experts(expert_linear(h, down, r.offsets), r.positions, r.weights)
    y = expert_mlp(x, logits, gate_up, down, 4)
    assert (y.float() - chain.float()).norm() <= 2.0**-7 * chain.float().norm()


@pytest.mark.parametrize("kind", KINDS)
def test_graphs_streams_and_shared_buffers(kind, device):
    """Two graphs captured on two streams and replayed in turn and side by side, beside eager calls."""
    x, logits, gate_up, down = case(kind, 8, 16, 512, 256, device)
    graphs = []
    for n in (8, 3):
        xi, li = x[:n].clone(), logits[:n].clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = expert_mlp(xi, li, gate_up, down, 2)
        graphs.append((graph, stream, xi, li, y))
    for seed in range(3):
        for graph, _, xi, li, y in graphs:
            xi.copy_(randn(50 + seed, *xi.shape).to(device))
            li.copy_(torch.randn(li.shape, device=device))
        torch.cuda.synchronize()
        eager = [expert_mlp(xi, li, gate_up, down, 2) for _, _, xi, li, _ in graphs]
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:  # side by side
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (*_, y), want in zip(graphs, eager):
            assert torch.equal(y, want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    want = expert_mlp(x, logits, gate_up, down, 2)
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(expert_mlp(x, logits, gate_up, down, 2))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in outs)


def test_refusals(device):
    x, logits, gate_up, down = case("bf16", 4, 8, 256, 128, device)
    f8 = weights("fp8", 1, 8, 256, 256, device=device)
    cases = [
        (lambda: expert_mlp(x, logits, gate_up[:7], down, 2), "gate_up must be"),
        (lambda: expert_mlp(x, logits, gate_up[:, :200], down, 2), "gate_up must be"),
        (lambda: expert_mlp(x, logits[:, :7], gate_up, down, 2), "logits must be"),
        (lambda: expert_mlp(x, logits[:3], gate_up, down, 2), "logits must be"),
        (lambda: expert_mlp(x, logits.half(), gate_up, down, 2), "logits must have dtype"),
        (lambda: expert_mlp(x[:, :128], logits, gate_up, down, 2), "x must be"),
        (lambda: expert_mlp(x.float(), logits, gate_up, down, 2), "x must be"),
        (lambda: expert_mlp(x, logits, gate_up, down, 0), "top_k"),
        (lambda: expert_mlp(x, logits, gate_up, down, 9), "top_k"),
        (lambda: expert_mlp(x, logits, gate_up, down, 2.0), "top_k"),
        (lambda: expert_mlp(x, logits, gate_up.transpose(1, 2), down, 2), "contiguous"),
        (lambda: expert_mlp(x, logits, gate_up, down, 2, base=x[:3]), "base must be"),
        (lambda: expert_mlp(x, logits, gate_up, down, 2, base=x.float()), "base must be"),
        (lambda: expert_mlp(x, logits, gate_up, down, 2, out=torch.empty(4, 255, dtype=torch.bfloat16, device=device)), "out must be"),
        (lambda: expert_mlp(x, logits, gate_up, down, 2, out=x), "share storage"),
        (lambda: expert_mlp(x.clone().requires_grad_(), logits, gate_up, down, 2), "inference-only"),
        (lambda: expert_mlp(x, logits, FP8Tensor(f8.codes, f8.scales[:, :1].contiguous()), down, 2), "one scale"),
    ]
    for call, match in cases:
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: expert_mlp(x, logits, gate_up, down, 2, renormalize=1), lambda: expert_mlp(x, None, gate_up, down, 2)):
        with pytest.raises(TypeError):
            call()
