"""Products grouped over more experts than one wave looks up at once, in row tiles of every type of operand.

A workgroup finds its expert from bounds of up to 64, of up to 256 (four a lane) or, past those, 64 at
a time. Experts of many rows, of one and of none lie on both sides of each border.
"""

import numpy as np
import pytest
import torch

from loraforge_amd import _lib
from oracle import experts as ox
from oracle import fp8 as of
from tests import test_fp8_gpu as t8
from tests import test_mxfp4_gpu as tm
from tests.test_mxfp4_gpu import close, forced, randn, segments

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("bf16", "mxfp4"), ("mxfp4", "mxfp4"), ("bf16", "fp8"), ("fp8", "fp8")]
TILES = [(64, 64), (128, 256), (192, 128), (64, 192), (256, 64)]


def counts_of(experts):
    """Rows of each expert: none, a few, and many at the ends and on both sides of the borders."""
    counts = np.random.default_rng(experts).integers(0, 4, experts)
    for e, rows in ((0, 70), (63, 1), (64, 130), (65, 0), (127, 65), (128, 3), (129, 200), (191, 64), (192, 33), (255, 257), (256, 90)):
        if e < experts:
            counts[e] = rows
    counts[experts - 1] = 77
    return [int(c) for c in counts]


def operand(x, kind, device, block_rows):
    if kind == "fp8":
        return t8.operand(x, "fp8", device, block_rows)
    return tm.operand(x, kind, device)


@pytest.mark.parametrize("experts", [64, 65, 130, 256, 257])
@pytest.mark.parametrize("types", TYPES, ids="-".join)
def test_experts_of_row_tiles(types, experts, device):
    act, weight = types
    counts, n, k = counts_of(experts), 264, 544
    rows, behind = sum(counts), 9
    x, xv = operand(randn(1, rows + behind, k), act, device, 1)
    w, wv = operand(randn(2, experts, n, k, std=0.05), weight, device, 128)
    offsets = segments(counts).to(device)
    order = np.random.default_rng(3).permutation(rows + behind)
    tokens = torch.from_numpy(order.astype(np.int32)).to(device)
    product = (lambda a, b: of.product(a, b, both=True)) if act == "fp8" else ox.product
    want, bound = np.zeros((rows, n)), np.zeros((rows, n))
    for e, (first, count) in enumerate(zip(np.cumsum([0] + counts), counts)):
        if count:
            want[first : first + count], bound[first : first + count] = product(xv[order[first : first + count]], wv[e])
    for height, columns in TILES:
        if weight == "fp8" and (_lib.LF_EXPERT_TILE, height, columns) not in t8.tiles(act):
            continue
        out = torch.full((rows + behind, n), 7.0, dtype=torch.bfloat16, device=device)
        forced(x, w, (_lib.LF_EXPERT_TILE, height, columns), experts=experts, offsets=offsets, tokens=tokens, out=out)
        close(out[:rows], want, bound)
        assert (out[rows:] == 7.0).all()
