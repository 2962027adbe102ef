"""The oracle of the MXFP4 and expert operators against closed forms and torch (CPU)."""

import numpy as np
import torch

from oracle import experts as ox


def test_levels_quantise_to_themselves():
    for exponent in (-127, -3, 0, 40, 120):
        x = np.zeros(32)
        x[:16] = np.concatenate([ox.LEVELS, -ox.LEVELS]) * 2.0**exponent
        codes, scales = ox.quantize(x)
        assert scales.tolist() == [max(exponent, -127) + 127]
        assert np.array_equal(ox.values(codes, scales), x)


def test_ties_go_to_even_codes_and_large_values_saturate():
    x = np.zeros(32)
    x[:10] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99]  # exponent 2, scale 1
    codes, scales = ox.quantize(x)
    assert scales.tolist() == [127]
    assert ox.values(codes, scales)[:10].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6]
    assert codes[0] == 0x06 and codes[1] == 0x22  # low nibble first: 4.0 then 0.25; 0.75 and 1.25 both go to 1.0


def test_zero_blocks_and_blocks_that_are_not_finite():
    x = np.zeros((3, 32))
    x[1, 5], x[2, 7] = np.inf, np.nan
    codes, scales = ox.quantize(x)
    assert scales.reshape(-1).tolist() == [0, 255, 255]
    v = ox.values(codes, scales)
    assert not v[0].any() and np.isnan(v[1:]).all()


def test_product_bound_holds_for_fp32_sums():
    g = torch.Generator().manual_seed(3)
    x, w, b = (torch.randn(*s, generator=g) for s in ((7, 513), (20, 513), (20,)))
    for swiglu in (False, True):
        y, bound = ox.product(x.double().numpy(), w.double().numpy(), b.double().numpy(), swiglu)
        z = x @ w.t() + b
        if swiglu:
            z = torch.nn.functional.silu(z[:, :10]) * z[:, 10:]
        assert (np.abs(z.double().numpy() - y) <= bound).all()


def test_routing_against_torch():
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(40, 12, generator=g, dtype=torch.float64)
    logits[torch.rand(40, 12, generator=g) < 0.6] = -np.inf
    logits[3] = -np.inf
    weights, experts, offsets, tokens, positions = ox.route(logits.numpy(), 4, False)
    p = torch.softmax(logits, 1).nan_to_num(0.0)
    value, index = p.topk(4, dim=1)
    assert np.allclose(weights, value.numpy())
    live = value.numpy() > 0
    assert np.array_equal(experts[live], index.numpy()[live]) and (experts[~live] == -1).all()
    assert (positions[~live] == -1).all() and offsets[-1] == live.sum()
    assert np.array_equal(tokens[positions[live]], np.nonzero(live)[0])
    for e in range(12):
        assert (np.diff(tokens[offsets[e] : offsets[e + 1]]) > 0).all()
        assert set(tokens[offsets[e] : offsets[e + 1]]) == set(np.nonzero((experts == e).any(1))[0])
    renormalised = ox.route(logits.numpy(), 4)[0]
    total = weights.sum(1, keepdims=True)
    assert np.allclose(renormalised, weights / np.where(total > 0, total, 1.0))
