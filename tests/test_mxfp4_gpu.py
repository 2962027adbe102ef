"""MXFP4 quantisation and the products with MXFP4 and bf16 weights on gfx950, against the 64-bit oracle.

Quantisation and dequantisation have to give the oracle's bits. A product may
be off by the oracle's bound on fp32 sums and half a bf16 ulp of the result
(2^-8 of it), plus the smallest bf16 subnormal.
"""

import numpy as np
import pytest
import torch

from loraforge_amd import _lib
from loraforge_amd.ops import MXFP4Tensor, dequantize_mxfp4, expert_linear, mxfp4_linear, quantize_mxfp4
from loraforge_amd.ops.mxfp4 import product
from oracle import experts as ox

pytestmark = pytest.mark.gpu

EVERY_BF16 = np.arange(65536, dtype=np.uint32) << 16


def close(y, expected, bound):
    y = y.double().cpu().numpy()
    assert y.shape == expected.shape
    assert np.array_equal(np.isnan(y), np.isnan(expected))
    limit = bound + 2.0**-8 * (np.abs(expected) + bound) + 2.0**-133
    worst = np.nanmax(np.abs(y - expected) - limit, initial=-np.inf)
    assert worst <= 0, worst


def check_codes(t, x):
    codes, scales = ox.quantize(x.double().cpu().numpy())
    assert np.array_equal(t.scales.cpu().numpy(), scales)
    assert np.array_equal(t.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (7, 4096), (3, 2, 96), (160,), (513, 1056)])
def test_quantize_matches_oracle(shape, dtype, device):
    x = (torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape))) * 3).to(dtype).to(device)
    t = quantize_mxfp4(x)
    assert t.shape == tuple(shape)
    check_codes(t, x)
    back = dequantize_mxfp4(t)
    assert np.array_equal(back.double().cpu().numpy(), ox.values(t.codes.cpu().numpy(), t.scales.cpu().numpy()))


def test_quantize_every_bf16_value(device):
    # Each finite value beside block maxima of its own to 2^6 times its magnitude, subnormals and zeros among them.
    x = torch.from_numpy(EVERY_BF16.view(np.float32).copy())
    x = x[torch.isfinite(x)]
    x = x[: x.numel() // 31 * 31].reshape(-1, 31)
    for shift in range(0, 8):
        top = x.abs().amax(1, keepdim=True)
        lead = torch.ldexp(top, torch.tensor(shift)).clamp(max=3e38)
        block = torch.cat([lead, x], 1).bfloat16().to(device)
        check_codes(quantize_mxfp4(block), block)


def test_quantize_ties_zero_and_not_finite_blocks(device):
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.5])
    near = torch.cat([ties, torch.nextafter(ties, torch.zeros(9)), torch.nextafter(ties, torch.full((9,), 9.0))])
    x = torch.zeros(6, 32)
    x[0, :27] = near
    x[1, :27] = -near * 2.0**-60
    x[2, 3] = float("inf")
    x[3, 30] = float("nan")
    x[4, 0] = 3e38
    x[5, 1] = 1e-45  # the smallest fp32 subnormal
    x[0, 31] = x[1, 31] = 0.0
    t = quantize_mxfp4(x.to(device))
    check_codes(t, x)
    assert torch.isnan(dequantize_mxfp4(t)[2:4]).all()


def test_quantize_strided_rows_and_empty(device):
    store = torch.randn(9, 200, device=device).bfloat16()
    view = store[:, 8 : 8 + 160]
    check_codes(quantize_mxfp4(view), view)
    empty = quantize_mxfp4(store[:0, :64])
    assert empty.codes.shape == (0, 32) and dequantize_mxfp4(empty).shape == (0, 64)


def test_dequantize_every_scale_and_code(device):
    codes = torch.arange(256, dtype=torch.uint8).reshape(16, 16).repeat(16, 1)[:256]
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    out = dequantize_mxfp4(MXFP4Tensor(codes.to(device), scales.to(device)))
    expected = ox.values(codes.numpy(), scales.numpy())
    expected = torch.from_numpy(expected).bfloat16()  # (past bf16's range: infinity)
    assert torch.equal(torch.nan_to_num(out.cpu(), nan=7.0), torch.nan_to_num(expected, nan=7.0))
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(expected))


# --------------------------------------------------------------------------
# Products
# --------------------------------------------------------------------------


def randn(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).bfloat16()


def operand(x, act, device):
    """The operand handed over and its fp64 values."""
    if act == "mxfp4":
        codes, scales = ox.quantize(x.double().numpy())
        t = MXFP4Tensor(torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device))
        return t, ox.values(codes, scales)
    return x.to(device), x.double().numpy()


def check_linear(m, n, k, act, device, *, swiglu=False, bias=False, seed=1):
    x, xv = operand(randn(seed, m, k), act, device)
    w, wv = operand(randn(seed + 1, n, k, std=0.05), "mxfp4", device)
    b = randn(seed + 2, n) if bias else None
    y = mxfp4_linear(x, w, bias=None if b is None else b.to(device), swiglu=swiglu)
    close(y, *ox.product(xv, wv, None if b is None else b.double().numpy(), swiglu))


@pytest.mark.parametrize("act", ["bf16", "mxfp4"])
@pytest.mark.parametrize(
    "m,n,k",
    [(1, 64, 512), (1, 1000, 4096), (3, 16, 32), (15, 17, 96), (16, 300, 160), (17, 64, 2880), (33, 128, 1056), (63, 500, 640),
     (65, 96, 256), (128, 256, 512), (129, 520, 1184), (200, 1, 64), (300, 777, 352), (1, 2, 12320)],
)
def test_linear_sizes(m, n, k, act, device):
    check_linear(m, n, k, act, device, bias=m % 2 == 0)


@pytest.mark.parametrize("act", ["bf16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 2, 64), (2, 24, 512), (40, 520, 416), (70, 512, 256), (257, 1000, 544)])
def test_linear_swiglu(m, n, k, act, device):
    check_linear(m, n, k, act, device, swiglu=True, bias=m % 2 == 1)


@pytest.mark.parametrize("m", [5, 260])
def test_linear_strided_x_and_out(m, device):
    """Rows wider than K on both sides: what follows a row (NaN) is not read into it, what follows an output row stays."""
    n, k = 260, 416
    store = torch.full((m, k + 24), float("nan")).bfloat16()
    store[:, 8 : 8 + k] = randn(3, m, k)
    w, wv = operand(randn(4, n, k, std=0.05), "mxfp4", device)
    x = store.to(device)[:, 8 : 8 + k]
    out_store = torch.zeros(m, n + 5, dtype=torch.bfloat16, device=device)
    y = mxfp4_linear(x, w, out=out_store[:, 2 : 2 + n])
    assert y.data_ptr() == out_store[:, 2:].data_ptr()
    close(y, *ox.product(store[:, 8 : 8 + k].double().numpy(), wv))
    assert not out_store[:, :2].any() and not out_store[:, 2 + n :].any()


@pytest.mark.parametrize("act", ["bf16", "mxfp4"])
@pytest.mark.parametrize("m", [20, 150])
def test_linear_nan_stays_in_its_row_and_column(m, act, device):
    n, k = 96, 288
    x, w = randn(5, m, k), randn(6, n, k)
    x[7, 280], w[33, 3] = float("nan"), float("inf")
    x, xv = operand(x, act, device)
    w, wv = operand(w, "mxfp4", device)
    y = mxfp4_linear(x, w).cpu()
    assert torch.isnan(y[7]).all() and torch.isnan(y[:, 33]).all()
    rest_rows, rest_cols = [i for i in range(m) if i != 7], [j for j in range(n) if j != 33]
    close(y[rest_rows][:, rest_cols], *ox.product(xv[rest_rows], wv[rest_cols]))


@pytest.mark.parametrize("act", ["bf16", "mxfp4"])
def test_linear_extreme_scales(act, device):
    """Scale bytes at both ends of what products can hold; results that underflow to zero and large finite ones."""
    m, n, k = 9, 40, 128
    xv = randn(7, m, k).double()
    xv[::2] *= 2.0**-60
    wv = randn(8, n, k).double()
    wv[::3] *= 2.0**60
    wv[1::3] *= 2.0**-110
    x, xv = operand(xv.bfloat16(), act, device)
    w, wv = operand(wv.bfloat16(), "mxfp4", device)
    y, bound = ox.product(xv, wv)
    close(mxfp4_linear(x, w), y, bound + 2.0**-126)  # (sums below the normal range may be flushed)


def test_linear_no_rows_and_repeatable(device):
    w, _ = operand(randn(9, 512, 1024, std=0.05), "mxfp4", device)
    assert mxfp4_linear(torch.zeros(0, 1024, dtype=torch.bfloat16, device=device), w).shape == (0, 512)
    x = randn(10, 100, 1024).to(device)
    first = mxfp4_linear(x, w)
    for _ in range(3):
        assert torch.equal(mxfp4_linear(x, w), first)


def segments(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32)


RAGGED = [
    [1],
    [0, 3, 0],
    [5, 0, 16, 1, 33],
    [0, 0, 0, 70],
    [64, 65, 1, 0, 130, 7],
    [1] * 130,
    [300, 2, 0, 257, 64],
]


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("bf16", "mxfp4"), ("mxfp4", "mxfp4")])
@pytest.mark.parametrize("counts", RAGGED, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("gather", [False, True])
def test_expert_linear_ragged(counts, types, gather, device):
    act, weight = types
    n, k = (264, 320) if len(counts) < 100 else (40, 96)
    if weight == "bf16":
        k += 8
    experts, rows = len(counts), sum(counts)
    rng = np.random.default_rng(rows + experts)
    swiglu, bias = rows % 2 == 1, experts % 2 == 1
    source = max(1, rows // 2) if gather else rows
    tokens = rng.integers(0, source, rows).astype(np.int32)
    x, xv = operand(randn(11, source, k), act, device)
    w, wv = operand(randn(12, experts, n, k, std=0.05), weight, device)
    b = randn(13, experts, n) if bias else None
    y = expert_linear(x, w, segments(counts).to(device), tokens=torch.from_numpy(tokens).to(device) if gather else None,
                      bias=None if b is None else b.to(device), swiglu=swiglu)
    start = 0
    for e, count in enumerate(counts):
        own = np.arange(start, start + count)
        if count:
            close(y[start : start + count],
                  *ox.product(xv[tokens[own] if gather else own], wv[e], None if b is None else b[e].double().numpy(), swiglu))
        start += count


@pytest.mark.parametrize("counts", [[3, 0, 2], [100, 0, 90]])
def test_expert_linear_rows_without_expert_stay(counts, device):
    """Rows past the last segment are left as they are, tokens there (-1) are not read."""
    n, k, rows = 64, 256, sum(counts) + 40
    x, xv = operand(randn(14, 50, k), "bf16", device)
    w, wv = operand(randn(15, 3, n, k, std=0.05), "mxfp4", device)
    tokens = torch.full((rows,), -1, dtype=torch.int32)
    tokens[: sum(counts)] = torch.arange(sum(counts)) % 50
    out = torch.full((rows, n), 3.0, dtype=torch.bfloat16, device=device)
    expert_linear(x, w, segments(counts).to(device), tokens=tokens.to(device), out=out)
    assert (out[sum(counts) :] == 3.0).all()
    first = tokens[: counts[0]].numpy()
    close(out[: counts[0]], *ox.product(xv[first], wv[0]))


def test_expert_linear_many_experts(device):
    """More experts than a wave searches at once, most of them empty."""
    rng = np.random.default_rng(6)
    counts = np.zeros(500, np.int64)
    counts[rng.integers(0, 500, 40)] = rng.integers(1, 6, 40)
    n, k = 24, 64
    x, xv = operand(randn(16, int(counts.sum()), k), "bf16", device)
    w, wv = operand(randn(17, 500, n, k, std=0.05), "bf16", device)
    y = expert_linear(x, w, segments(counts).to(device))
    expected = np.concatenate([ox.product(xv[s : s + c], wv[e])[0] for e, (s, c) in enumerate(zip(np.cumsum(counts) - counts, counts))])
    bound = np.concatenate([ox.product(xv[s : s + c], wv[e])[1] for e, (s, c) in enumerate(zip(np.cumsum(counts) - counts, counts))])
    close(y, expected, bound)


def test_expert_linear_weights_past_4_gib(device):
    """Offsets into the weight that do not fit 32 bits: the last expert of 4.5 GiB."""
    n, k, experts = 4096, 4096, 144
    w = torch.zeros(experts, n, k, dtype=torch.bfloat16, device=device)
    w[-1] = randn(18, n, k, std=0.05).to(device)
    x = randn(19, 130, k).to(device)
    offsets = torch.zeros(experts + 1, dtype=torch.int32)
    offsets[-1] = 130
    for rows in (2, 130):
        offsets[-1] = rows
        y = expert_linear(x[:rows], w, offsets.to(device))
        columns = np.arange(0, n, 97)
        close(y[:, columns], *ox.product(x[:rows].double().cpu().numpy(), w[-1][columns].double().cpu().numpy()))


def test_products_on_a_side_stream_and_in_a_graph(device):
    w, wv = operand(randn(20, 512, 512, std=0.05), "mxfp4", device)
    x = randn(21, 24, 512).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = mxfp4_linear(quantize_mxfp4(x), w)
    side.synchronize()
    eager = mxfp4_linear(quantize_mxfp4(x), w)
    assert torch.equal(y, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mxfp4_linear(quantize_mxfp4(x), w)
    for seed in range(3):
        x.copy_(randn(30 + seed, 24, 512).to(device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mxfp4_linear(quantize_mxfp4(x), w))


# --------------------------------------------------------------------------
# Every kernel and tile, forced
# --------------------------------------------------------------------------

TYPES = [("bf16", "bf16"), ("bf16", "mxfp4"), ("mxfp4", "mxfp4")]
PLANS = [(_lib.LF_EXPERT_STREAM, 0, c) for c in (16, 32)] + [(_lib.LF_EXPERT_ROWS, 0, 128)] + [
    (_lib.LF_EXPERT_TILE, r, c) for r in (64, 128, 192, 256) for c in (64, 128, 192, 256)]


def forced(x, w, plan, **options):
    arguments = dict(experts=None, offsets=None, tokens=None, bias=None, swiglu=False, out=None)
    return product(x, w, **{**arguments, **options}, plan=_lib.ExpertPlan(*plan))


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("plan", PLANS, ids=lambda p: "-".join(map(str, p)))
@pytest.mark.parametrize("k", [128, 416, 2880])
def test_every_plan(types, plan, k, device):
    """Ragged experts on one kernel: tile heights of one to four 64-row steps, ends of k inside a stage, edge columns."""
    act, weight = types
    if k < 512 and ((act == "mxfp4" and plan[0] == _lib.LF_EXPERT_TILE) or (weight == "mxfp4" and plan[0] == _lib.LF_EXPERT_ROWS)):
        k += 512  # (what these kernels take begins there)
    counts = [130, 0, 1, 64, 257, 33, 190]
    n = 328
    rows = sum(counts)
    x, xv = operand(randn(k, rows, k), act, device)
    w, wv = operand(randn(k + 1, len(counts), n, k, std=0.05), weight, device)
    b = randn(k + 2, len(counts), n)
    y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device), bias=b.to(device))
    start = 0
    for e, count in enumerate(counts):
        if count:
            close(y[start : start + count], *ox.product(xv[start : start + count], wv[e], b[e].double().numpy()))
        start += count


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("plan", PLANS, ids=lambda p: "-".join(map(str, p)))
@pytest.mark.parametrize("n", [512, 776, 88])
def test_every_plan_swiglu(types, plan, n, device):
    act, weight = types
    k, counts = 544, [70, 3, 200]
    x, xv = operand(randn(n, sum(counts), k), act, device)
    w, wv = operand(randn(n + 1, len(counts), n, k, std=0.05), weight, device)
    b = randn(n + 2, len(counts), n)
    y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device), bias=b.to(device), swiglu=True)
    start = 0
    for e, count in enumerate(counts):
        close(y[start : start + count], *ox.product(xv[start : start + count], wv[e], b[e].double().numpy(), True))
        start += count


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("columns", [64, 128, 192, 256])
def test_tiles_of_one_dense_product(types, columns, device):
    """Several row and column tiles of one segment, on every workgroup order; results do not depend on the tile."""
    act, weight = types
    m, n, k = 1300, 700, 512
    x, xv = operand(randn(40, m, k), act, device)
    w, wv = operand(randn(41, 1, n, k, std=0.05), weight, device)
    whole = segments([m]).to(device)
    y = forced(x, w, (_lib.LF_EXPERT_TILE, 256, columns), experts=1, offsets=whole)
    close(y, *ox.product(xv, wv[0]))
    for rows in (64, 128, 192):
        assert torch.equal(forced(x, w, (_lib.LF_EXPERT_TILE, rows, columns), experts=1, offsets=whole), y)


@pytest.mark.parametrize("plan", [(_lib.LF_EXPERT_STREAM, 0, 32), (_lib.LF_EXPERT_ROWS, 0, 128), (_lib.LF_EXPERT_TILE, 256, 256)], ids=str)
def test_output_rows_of_any_alignment(plan, device):
    m, n, k = 200, 256, 576
    x, xv = operand(randn(42, m, k), "bf16", device)
    w, wv = operand(randn(43, n, k, std=0.05), "mxfp4", device)
    expected = ox.product(xv, wv)
    for pad, at in ((0, 0), (8, 8), (3, 1), (8, 4)):
        store = torch.zeros(m, n + pad, dtype=torch.bfloat16, device=device)
        out = store[:, at : at + n]
        forced(x, w, plan, out=out)
        close(out, *expected)
        assert not store[:, :at].any() and not store[:, at + n :].any()


@pytest.mark.parametrize("types", TYPES, ids="-".join)
def test_scales_and_rows_at_odd_addresses(types, device):
    """Scale bytes at any address; x rows gathered from a larger store, backwards."""
    act, weight = types
    m, n, k = 150, 192, 672
    x, xv = operand(randn(44, m, k), act, device)
    w, wv = operand(randn(45, 1, n, k, std=0.05), weight, device)

    def shifted(t):
        store = torch.zeros(t.numel() + 3, dtype=torch.uint8, device=device)
        store[3:] = t.reshape(-1)
        return store[3:].reshape(t.shape)

    if act == "mxfp4":
        x = MXFP4Tensor(x.codes, shifted(x.scales))
    if weight == "mxfp4":
        w = MXFP4Tensor(w.codes, shifted(w.scales))
    tokens = torch.arange(m - 1, -1, -1, dtype=torch.int32, device=device)
    for plan in PLANS[1], PLANS[2], PLANS[3], PLANS[-1]:
        y = forced(x, w, plan, experts=1, offsets=segments([m]).to(device), tokens=tokens)
        close(y, *ox.product(xv[::-1], wv[0]))


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("columns", [16, 32])
@pytest.mark.parametrize("part", [16, 32, 64])
def test_streamed_rows_in_passes(part, columns, types, device):
    """A workgroup for each pass of 16, 32 or 64 rows: whole and broken passes, of ragged experts and of a dense product."""
    act, weight = types
    plan = (_lib.LF_EXPERT_STREAM, part, columns)
    n, k = 104, 544
    counts = [16, 0, 33, 64, 1, 131, 0]
    x, xv = operand(randn(1, sum(counts), k), act, device)
    w, wv = operand(randn(2, len(counts), n, k, std=0.05), weight, device)
    y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device))
    start = 0
    for e, count in enumerate(counts):
        if count:
            close(y[start : start + count], *ox.product(xv[start : start + count], wv[e], None))
        start += count
    if weight == "mxfp4":
        for m in (15, 64, 97):
            x, xv = operand(randn(m, m, k), act, device)
            dense, dv = operand(randn(3, n, k, std=0.05), weight, device)
            close(forced(x, dense, plan), *ox.product(xv, dv, None))


def test_passes_past_the_second_grid_dimension(device):
    """65536 passes of 16 rows: more than a grid's second dimension holds."""
    m = 65536 * 16 - 3
    w, wv = operand(randn(4, 2, 32, std=0.5), "mxfp4", device)
    x, xv = operand(randn(5, 64, 32), "bf16", device)
    rows = torch.arange(m, device=device) % 64
    y = forced(x[rows], w, (_lib.LF_EXPERT_STREAM, 16, 16))
    first = forced(x, w, (_lib.LF_EXPERT_STREAM, 64, 16))
    close(first, *ox.product(xv, wv, None))
    assert torch.equal(y, first[rows])
