"""Products, quantisation and routing where their kernels can go wrong unseen: every kernel, forced.

- Long k with exact sums. Operands are small integers times 2^-2 at least, and the sum of all
  magnitudes of an output stays below 2^24 of the least product (asserted), so fp32 sums in
  any order are exact and the result is the fp64 one rounded once to bf16: equal, bit for bit.
- NaN, the scale byte 255 and scale bytes at both ends of the format, past the first unit of scales.
- Offsets past 32 bits, against the same rows in a small buffer.
- Routing of more tokens than 256 chunks of 32.
"""

import numpy as np
import pytest
import torch

from loraforge_amd import _lib
from loraforge_amd.ops import MXFP4Tensor, combine_experts, dequantize_mxfp4, mxfp4_linear, quantize_mxfp4
from oracle import experts as ox
from tests.test_experts_gpu import check_route, logits_of
from tests.test_mxfp4_gpu import PLANS, TYPES, check_codes, close, forced, operand, randn, segments

pytestmark = pytest.mark.gpu

EVERY = PLANS + [(_lib.LF_EXPERT_STREAM, part, columns) for part in (16, 32) for columns in (16, 32)]


def packed(rng, shape, scales, device):
    """Random codes with scale bytes out of ``scales``, and their fp64 values."""
    codes = rng.integers(0, 256, (*shape[:-1], shape[-1] // 2)).astype(np.uint8)
    bytes_ = rng.choice(np.array(scales, np.uint8), (*shape[:-1], shape[-1] // 32))
    return MXFP4Tensor(torch.from_numpy(codes).to(device), torch.from_numpy(bytes_).to(device)), ox.values(codes, bytes_)


def integers(rng, shape, device):
    v = rng.integers(-8, 9, shape).astype(np.float64)
    return torch.from_numpy(v).bfloat16().to(device), v


def rounded(v):
    return torch.from_numpy(v).float().bfloat16()


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("k", [8224, 12320])
def test_long_k_exact_on_every_kernel(types, k, device):
    act, weight = types
    k += 8 if weight == "bf16" else 0
    rng = np.random.default_rng(k)
    counts, n = [70, 0, 1, 130], 136
    make = {"bf16": lambda *shape: integers(rng, shape, device), "mxfp4": lambda *shape: packed(rng, shape, (126, 127, 128), device)}
    x, xv = make[act](sum(counts), k)
    w, wv = make[weight](len(counts), n, k)
    own = np.repeat(np.arange(len(counts)), counts)
    exact = np.concatenate([xv[own == e] @ wv[e].T for e in range(len(counts))])
    assert max((np.abs(xv[own == e]) @ np.abs(wv[e]).T).max() for e in (0, 2, 3)) * 16 < 2**24
    expected = rounded(exact)
    # The oracle without the last 32 k: most outputs would show it.
    short = rounded(exact - np.concatenate([xv[own == e][:, -32:] @ wv[e][:, -32:].T for e in range(len(counts))]))
    assert (short != expected).double().mean() > 0.5
    for plan in EVERY:
        y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device))
        assert torch.equal(y.cpu(), expected), plan


BLOCKS = (0, 15, 16, 47, 63, 64, 66)  # of 67: ends of units of 4, 16 and 64 scales, the last one


@pytest.mark.parametrize("types", TYPES[1:], ids="-".join)
def test_not_finite_blocks_on_every_kernel(types, device):
    """One block of a row or of a weight row is NaN: all of its row or column, and nothing else."""
    act, _ = types
    counts, n, k = [97, 53], 72, 2144
    rng = np.random.default_rng(1)
    x, xv = operand(randn(1, sum(counts), k), act, device)
    w, wv = packed(rng, (2, n, k), (120, 121, 122), device)
    for j, block in enumerate(BLOCKS):
        at = slice(32 * block, 32 * block + 32)
        xv[21 * j + 5, at] = np.nan
        wv[j % 2, 9 * j + 4, at] = np.nan
        w.scales[j % 2, 9 * j + 4, block] = 255
        if act == "mxfp4":
            x.scales[21 * j + 5, block] = 255
        else:
            x[21 * j + 5, 32 * block + j] = float("nan")
    for plan in EVERY:
        y = forced(x, w, plan, experts=2, offsets=segments(counts).to(device))
        close(y[:97], *ox.product(xv[:97], wv[0]))
        close(y[97:], *ox.product(xv[97:], wv[1]))


@pytest.mark.parametrize("types", TYPES[1:], ids="-".join)
def test_extreme_scales_on_every_kernel(types, device):
    """Scale bytes from 0 on: every output whose terms cannot overflow (below the normal range it may be flushed)."""
    act, _ = types
    m, n, k = 140, 72, 2144
    rng = np.random.default_rng(2)

    def rows(count, bytes_):
        t, _ = packed(rng, (count, k), (127,), "cpu")
        t.scales[:] = torch.tensor(bytes_, dtype=torch.uint8)[torch.arange(count) % len(bytes_)].unsqueeze(1)
        values = ox.values(t.codes.numpy(), t.scales.numpy())
        return MXFP4Tensor(t.codes.to(device), t.scales.to(device)), values

    if act == "mxfp4":
        x, xv = rows(m, (0, 1, 27, 127, 227, 253, 254))
    else:
        xv = rng.integers(-8, 9, (m, k)) * np.exp2(np.array((-120.0, -60.0, 0.0, 60.0, 119.0))[np.arange(m) % 5])[:, None]
        x = torch.from_numpy(xv).bfloat16().to(device)
    w, wv = rows(n, (0, 1, 27, 127, 227, 251, 252))  # (from 253 on a level may pass bf16's range beside bf16 x)
    w1 = MXFP4Tensor(w.codes.unsqueeze(0), w.scales.unsqueeze(0))
    expected, bound = ox.product(xv, wv)
    held = np.abs(xv) @ np.abs(wv).T < 2.0**127
    assert held.mean() > 0.5 and (np.abs(expected[held]) > 2.0**60).any()
    for plan in EVERY:
        y = forced(x, w1, plan, experts=1, offsets=segments([m]).to(device))
        close(y.cpu()[torch.from_numpy(held)], expected[held], bound[held] + 2.0**-126)


# --------------------------------------------------------------------------
# Offsets past 32 bits
# --------------------------------------------------------------------------

FEW = [(_lib.LF_EXPERT_STREAM, 0, 32), (_lib.LF_EXPERT_ROWS, 0, 128), (_lib.LF_EXPERT_TILE, 64, 64), (_lib.LF_EXPERT_TILE, 256, 256)]


@pytest.mark.parametrize("act", ["bf16", "mxfp4"])
def test_output_past_32_bits(act, device):
    """70000 x 32768 outputs (2.3 10^9): each row as in a product of the 50 different rows alone."""
    m, n, k = 70000, 32768, 512
    x, xv = operand(randn(60, 50, k), act, device)
    w, wv = operand(randn(61, n, k, std=0.05), "mxfp4", device)
    at = torch.arange(m, device=device) % 50
    many = x[at] if act == "bf16" else MXFP4Tensor(x.codes[at], x.scales[at])
    out = torch.empty(m, n, dtype=torch.bfloat16, device=device)
    for plan in FEW[:1] + FEW[3:]:
        one = forced(x, w, plan)
        columns = np.arange(0, n, 997)
        close(one[:, columns], *ox.product(xv, wv[columns]))
        out.fill_(7.0)
        forced(many, w, plan, out=out)
        for first in range(0, m, 10000):
            assert torch.equal(out[first : first + 10000], one[at[first : first + 10000]]), (plan, first)


def test_gathered_rows_past_32_bits(device):
    """x of 4.9 GB, only whose last rows are named."""
    n, k, total, rows = 96, 4096, 600000, 130
    x = torch.zeros(total, k, dtype=torch.bfloat16, device=device)
    last = randn(62, rows, k)
    x[-rows:] = last.to(device)
    w, wv = operand(randn(63, 1, n, k, std=0.05), "mxfp4", device)
    tokens = torch.arange(total - rows, total, dtype=torch.int32, device=device)
    for plan in FEW:
        close(forced(x, w, plan, experts=1, offsets=segments([rows]).to(device), tokens=tokens),
              *ox.product(last.double().numpy(), wv[0]))


@pytest.mark.parametrize("total", [2**20 - 1, 2**20 + 5])
def test_packed_rows_around_4_gib(total, device):
    """MXFP4 x whose codes end just below and above 4 GiB (the tiles' row offsets have 32 bits; above, none is offered)."""
    n, k, rows = 96, 8192, 130
    last, lv = operand(randn(64, rows, k), "mxfp4", device)
    x = MXFP4Tensor(torch.zeros(total, k // 2, dtype=torch.uint8, device=device),
                    torch.zeros(total, k // 32, dtype=torch.uint8, device=device))
    x.codes[-rows:], x.scales[-rows:] = last.codes, last.scales
    w, wv = operand(randn(65, 1, n, k, std=0.05), "mxfp4", device)
    tokens = torch.arange(total - rows, total, dtype=torch.int32, device=device)
    for plan in FEW:
        if plan[0] == _lib.LF_EXPERT_TILE and total > 2**20:
            continue
        close(forced(x, w, plan, experts=1, offsets=segments([rows]).to(device), tokens=tokens), *ox.product(lv, wv[0]))


def test_quantize_and_combine_past_32_bits(device):
    rows, k = 2**19 + 3, 4128  # 2.2 10^9 values
    last = randn(66, 70, k)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=device)
    x[-70:] = last.to(device)
    t = quantize_mxfp4(x)
    end = MXFP4Tensor(t.codes[-70:].clone(), t.scales[-70:].clone())
    check_codes(end, last)
    assert not t.codes[:-70].any() and not t.scales[:-70].any()
    back = dequantize_mxfp4(t)
    assert torch.equal(back[-70:], dequantize_mxfp4(end)) and not back[:-70].any()
    positions = torch.tensor([[rows - 1, rows - 70], [-1, rows - 2]], dtype=torch.int32, device=device)
    y = combine_experts(x, positions, torch.tensor([[0.5, 2.0], [1.0, 0.25]], device=device))
    v = last.double()
    expected = torch.stack([0.5 * v[69] + 2.0 * v[0], 0.25 * v[68]])
    assert ((y.double().cpu() - expected).abs() <= 2.0**-8 * expected.abs() + 2.0**-21 * (v[69].abs() + v[0].abs() * 2)).all()


# --------------------------------------------------------------------------
# Routing in chunks of more than 32 tokens
# --------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,experts,top,dtype", [(8193, 8, 2, torch.float32), (20011, 33, 3, torch.bfloat16), (70001, 5, 2, torch.float32)])
def test_route_many_tokens(tokens, experts, top, dtype, device):
    check_route(logits_of(tokens, tokens, experts, dtype, device), top, renormalize=tokens % 2 == 0)


def test_route_many_tokens_masked(device):
    logits = logits_of(3, 16411, 12, torch.float32, "cpu")
    logits[torch.rand(16411, 12, generator=torch.Generator().manual_seed(4)) < 0.8] = -np.inf
    check_route(logits.to(device), 4)


def test_short_k_of_many_rows(device):
    """MXFP4 on both sides with k below 512: the weight stream, whatever the rows."""
    for m, n, k in ((2000, 520, 480), (700, 72, 32)):
        x, xv = operand(randn(m, m, k), "mxfp4", device)
        w, wv = operand(randn(n, n, k, std=0.05), "mxfp4", device)
        close(mxfp4_linear(x, w), *ox.product(xv, wv))
