"""FP8 scales far from one, each range seen by itself, on every kernel.

The bound of ``oracle.fp8.product`` is made from each output's own terms, so outputs of blocks around 2^-100 are
held to their own size. Scales of x and of a weight are multiplied first: a product of two below 2^-126 may be flushed.
"""

import numpy as np
import pytest
import torch

from loraforge_amd.ops import FP8Tensor
from oracle import fp8 as of
from tests.test_fp8_gpu import PLANS, forced, operand, weight
from tests.test_mxfp4_gpu import close, randn, segments

pytestmark = pytest.mark.gpu

EXPONENTS = np.array([-100, -60, 0, 60, 100])


def scaled(t, exponents):
    """``t`` with its scales times 2^exponents, and its fp64 values."""
    t = FP8Tensor(t.codes, t.scales * torch.exp2(torch.from_numpy(np.array(exponents)).to(t.scales)))
    return t, of.values(t.codes.view(torch.uint8).cpu().numpy(), t.scales.cpu().numpy())


def every_plan(x, w, act, m, want, device):
    for plan in PLANS[act]:
        y = forced(x, FP8Tensor(w.codes[None], w.scales[None]), plan, experts=1, offsets=segments([m]).to(device))
        close(y, *want)


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_a_range_for_each_block_of_rows(act, device):
    """128 weight rows around 2^-100, 128 around 2^-60, ..., one step up or down from block to block of k."""
    m, n, k = 140, 600, 2128
    x, xv = operand(randn(7, m, k), act, device)
    w, _ = weight(8, n, k, device=device)
    w, wv = scaled(w, EXPONENTS[:, None] + np.arange(17)[None] % 3 - 1.0)
    want = of.product(xv, wv, both=act == "fp8")
    small = np.abs(want[0][:, :128])
    assert 0 < small.max() < 2.0**-90 and np.abs(want[0][:, 512:]).max() > 2.0**90
    every_plan(x, w, act, m, want, device)


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_ranges_of_x_and_weight_that_cancel(act, device):
    """Blocks of k whose x is around 2^e and whose weights are around 2^-e: all of them count alike in every output."""
    m, n, k = 140, 264, 2128
    powers = EXPONENTS[np.arange(17) % 5]
    xs = randn(9, m, k)
    if act == "fp8":
        x, _ = operand(xs, act, device)
        x, xv = scaled(x, np.broadcast_to(powers, (m, 17)))
    else:
        xs = (xs.double() * torch.from_numpy(np.exp2(np.repeat(powers, 128)[:k].astype(np.float64)))).bfloat16()
        x, xv = operand(xs, act, device)
    w, _ = weight(10, n, k, device=device)
    w, wv = scaled(w, np.broadcast_to(-powers, (3, 17)))
    want = of.product(xv, wv, both=act == "fp8")
    assert (np.abs(want[0]) > 2.0 * want[1]).mean() > 0.5
    every_plan(x, w, act, m, want, device)
