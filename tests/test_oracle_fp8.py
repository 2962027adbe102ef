"""The FP8 oracle against closed forms, brute force and torch's e4m3 conversion."""

import numpy as np
import torch

from oracle import fp8 as of


def test_levels_are_e4m3():
    codes = torch.arange(256, dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double().numpy()
    own = of.values(codes.numpy().reshape(2, 128), np.ones((2, 1))).reshape(-1)
    assert np.array_equal(np.isnan(v), np.isnan(own)) and np.array_equal(np.nan_to_num(v), np.nan_to_num(own))
    assert np.array_equal(np.signbit(v[:255]), np.signbit(own[:255]))
    assert len(of.LEVELS) == 127 and of.LEVELS[-1] == 448.0


def test_nearest_by_brute_force():
    a = np.concatenate([of.LEVELS, (of.LEVELS[:-1] + of.LEVELS[1:]) / 2, np.random.default_rng(0).uniform(0, 448, 2000)])
    for value, code in zip(a, of.nearest(a)):
        d = np.abs(of.LEVELS - value)
        best = np.flatnonzero(d == d.min())
        assert code in best and (len(best) == 1 or code % 2 == 0)
    assert np.array_equal(of.nearest(a), torch.from_numpy(a).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_quantize_shapes_scales_and_error():
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((2, 130, 272))).bfloat16().double().numpy()
    for rows, held in ((1, (2, 130, 3)), (128, (2, 2, 3))):
        codes, scales = of.quantize(x, rows)
        assert codes.shape == x.shape and scales.shape == held and scales.dtype == np.float32
        back = of.values(codes, scales)
        top = np.repeat(np.repeat(scales.astype(np.float64), rows, 1)[:, :130], 128, 2)[..., :272] * 448
        assert (np.abs(back) <= top * (1 + 1e-7)).all()
        assert (np.abs(back - x) <= np.maximum(np.abs(x) * 2.0**-4, top / 448 * 2.0**-10) * (1 + 1e-6)).all()
    # The block of 128 x 128 has the scale of its largest value, here and in the short last row and column.
    assert scales[1, 1, 2] == np.float32(np.abs(x[1, 128:, 256:]).max() / 448)
    assert scales[0, 0, 1] == np.float32(np.abs(x[0, :128, 128:256]).max() / 448)


def test_quantize_zero_tiny_and_not_finite():
    x = np.zeros((4, 32))
    x[1, 3] = 2.0**-120
    x[2, 5] = np.inf
    x[3, 31] = np.nan
    codes, scales = of.quantize(x)
    assert (scales[:2] == np.float32(2.0**-100 / 448)).all() and not codes[0].any()
    assert np.isnan(of.values(codes, scales)[2:]).all() and not codes[2:].any()


def test_product_bounds():
    """Beside FP8 x the bound grows by what eight aligned products may lose, and covers a model of that loss."""
    rng = np.random.default_rng(3)
    x, w = (of.values(*of.quantize(rng.standard_normal((5, 48)) * np.exp2(rng.integers(-6, 7, (5, 48))))) for _ in range(2))
    y, bound = of.product(x, w)
    y8, bound8 = of.product(x, w, both=True)
    assert np.array_equal(y, y8) and (bound8 > bound).all()
    p = (x[:, None] * w[None]).reshape(5, 5, 6, 8)
    unit = np.exp2(np.floor(np.log2(np.abs(p).max(-1, keepdims=True))) - 13)
    kept = (np.trunc(p / unit) * unit).sum((-1, -2))
    assert (np.abs(kept - y) <= bound8 - bound).all() and (np.abs(kept - y) > bound).any()
