"""FP8 quantisation and the products with FP8 weights on gfx950, against the 64-bit oracle.

Codes and scales have to be the oracle's, bit for bit (a scale is one division, rounded
once). A product may be off by the oracle's bound on fp32 sums, whose count of roundings
covers those of the scales (a product of two and one a block, each 2^-24 of a block's
sum), beside FP8 x by what the 8-bit matrix instructions drop (``oracle.fp8.product``), and half a bf16
ulp of the result (2^-8 of it), plus the smallest bf16 subnormal.
"""

import numpy as np
import pytest
import torch

from loraforge_amd import _lib
from loraforge_amd.ops import FP8Tensor, dequantize_fp8, expert_linear, fp8_linear, quantize_fp8, quantize_mxfp4
from loraforge_amd.ops.mxfp4 import product
from oracle import fp8 as of
from tests.test_mxfp4_gpu import RAGGED, close, randn, segments

pytestmark = pytest.mark.gpu


def held(codes, scales, device):
    return FP8Tensor(torch.from_numpy(codes).to(device).view(torch.float8_e4m3fn), torch.from_numpy(scales).to(device))


def operand(x, act, device, rows=1):
    """The operand handed over and its fp64 values."""
    if act == "fp8":
        codes, scales = of.quantize(x.double().numpy(), rows)
        return held(codes, scales, device), of.values(codes, scales)
    return x.to(device), x.double().numpy()


def weight(seed, *shape, device, std=0.05):
    return operand(randn(seed, *shape, std=std), "fp8", device, 128)


def same(t, x, rows):
    codes, scales = of.quantize(x.double().cpu().numpy(), rows)
    assert np.array_equal(t.scales.cpu().numpy(), scales, equal_nan=True)
    assert np.array_equal(t.codes.view(torch.uint8).cpu().numpy(), codes)


# --------------------------------------------------------------------------
# Quantisation
# --------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 16), (7, 4096), (3, 2, 144), (130, 272), (513, 1056), (2, 257, 128), (1, 12320), (300, 16)])
def test_quantize_matches_oracle(shape, rows, device):
    x = (torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape))) * 3).bfloat16().to(device)
    t = quantize_fp8(x, block_rows=rows)
    assert t.shape == tuple(shape)
    same(t, x, rows)
    back = dequantize_fp8(t)
    expected = torch.from_numpy(of.values(t.codes.view(torch.uint8).cpu().numpy(), t.scales.cpu().numpy()))
    # (A product of a code and a 24-bit scale in fp32, off by 2^-24 of it, then to the 8 bits of bf16,
    # whose steps are 2^-7 from a power of two on: by half of that, 2^-8.)
    assert ((back.double().cpu() - expected).abs() <= expected.abs() * (2.0**-8 + 2.0**-23)).all()


def test_quantize_every_pair_of_magnitudes(device):
    """Each bf16 significand beside each as its block's largest, over the e4m3 range: all ties among them."""
    tops = torch.arange(128, 256, dtype=torch.float64) / 128
    small = torch.arange(128, 256, dtype=torch.float64) / 128
    for shift in range(0, 20):
        x = torch.where(torch.arange(128) % 2 == 0, 1.0, -1.0) * small * 2.0**-shift  # one block of 128
        x = x.repeat(128, 1)
        x = torch.minimum(x.abs(), tops.unsqueeze(1)) * torch.sign(x)
        x[:, 0] = tops
        for scale in (1.0, 2.0**-90, 2.0**119):
            v = (x * scale).bfloat16()
            assert torch.equal(v.double(), x * scale)
            same(quantize_fp8(v.to(device)), v, 1)
            same(quantize_fp8(v.to(device), block_rows=128), v, 128)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_zero_tiny_and_not_finite(rows, device):
    x = torch.zeros(300, 160)
    x[0, 3] = 1e-40  # a bf16 subnormal
    x[1, 5] = 2.0**-100
    x[130, 7] = float("inf")
    x[131, 140] = float("nan")
    x[257, 1] = -3e38
    x = x.bfloat16()
    t = quantize_fp8(x.to(device), block_rows=rows)
    same(t, x, rows)
    back = dequantize_fp8(t)
    assert torch.isnan(back[130, :128]).all() and torch.isnan(back[131, 128:]).all() and not torch.isnan(back[:128]).any()


def test_quantize_strided_rows_and_empty(device):
    store = torch.full((9, 208), float("nan"), device=device).bfloat16()
    store[:, 8:168] = torch.randn(9, 160, device=device).bfloat16()
    view = store[:, 8:168]
    for rows in (1, 128):
        same(quantize_fp8(view, block_rows=rows), view, rows)
        empty = quantize_fp8(store[:0, :64], block_rows=rows)
        assert empty.codes.shape == (0, 64) and empty.scales.shape == (0, 1) and dequantize_fp8(empty).shape == (0, 64)


def test_dequantize_every_code(device):
    codes = torch.arange(256, dtype=torch.uint8).reshape(2, 128)
    for scale in (1.0, 2.0**-100, 0.3, 2.0**110, 0.0, float("inf"), float("nan")):
        t = FP8Tensor(codes.to(device).view(torch.float8_e4m3fn), torch.full((2, 1), scale, device=device))
        with np.errstate(invalid="ignore"):
            expected = torch.from_numpy(of.values(codes.numpy(), t.scales.cpu().numpy())).float().bfloat16()
        out = dequantize_fp8(t, out=torch.empty(2, 128, dtype=torch.bfloat16, device=device)).cpu()
        assert torch.equal(torch.isnan(out), torch.isnan(expected))
        assert torch.equal(torch.nan_to_num(out, nan=7.0), torch.nan_to_num(expected, nan=7.0))


def test_quantize_and_back_past_32_bits(device):
    rows, k = 2**19 + 3, 4112  # 2.2 10^9 values
    last = randn(66, 70, k)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=device)
    x[-70:] = last.to(device)
    t = quantize_fp8(x)
    end = FP8Tensor(t.codes[-70:].clone(), t.scales[-70:].clone())
    same(end, last, 1)
    assert not t.codes[:-70].view(torch.uint8).any()
    back = dequantize_fp8(t)
    assert torch.equal(back[-70:], dequantize_fp8(end)) and not back[:-70].any()
    del back, t
    t = quantize_fp8(x, block_rows=128)
    first = (rows - 70) // 128 * 128
    whole = x[first:].contiguous()
    assert torch.equal(t.codes[first:].view(torch.uint8), quantize_fp8(whole, block_rows=128).codes.view(torch.uint8))


# --------------------------------------------------------------------------
# Products
# --------------------------------------------------------------------------


def check_linear(m, n, k, act, device, *, swiglu=False, bias=False, seed=1):
    x, xv = operand(randn(seed, m, k), act, device)
    w, wv = weight(seed + 1, n, k, device=device)
    b = randn(seed + 2, n) if bias else None
    y = fp8_linear(x, w, bias=None if b is None else b.to(device), swiglu=swiglu)
    close(y, *of.product(xv, wv, None if b is None else b.double().numpy(), swiglu, act == "fp8"))


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize(
    "m,n,k",
    [(1, 64, 512), (1, 1000, 4096), (3, 16, 16), (15, 17, 96), (16, 300, 144), (17, 64, 2880), (33, 128, 1040), (63, 500, 640),
     (65, 96, 256), (128, 256, 512), (129, 520, 1168), (200, 1, 64), (300, 777, 352), (1, 2, 12304)],
)
def test_linear_sizes(m, n, k, act, device):
    check_linear(m, n, k, act, device, bias=m % 2 == 0)


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", [(1, 256, 64), (2, 512, 512), (40, 768, 416), (70, 512, 256), (257, 1280, 528)])
def test_linear_swiglu(m, n, k, act, device):
    check_linear(m, n, k, act, device, swiglu=True, bias=m % 2 == 1)


@pytest.mark.parametrize("m", [5, 260])
def test_linear_strided_x_and_out(m, device):
    """Rows wider than K on both sides: what follows a row (NaN) is not read into it, what follows an output row stays."""
    n, k = 260, 400
    store = torch.full((m, k + 24), float("nan")).bfloat16()
    store[:, 8 : 8 + k] = randn(3, m, k)
    w, wv = weight(4, n, k, device=device)
    x = store.to(device)[:, 8 : 8 + k]
    out_store = torch.zeros(m, n + 5, dtype=torch.bfloat16, device=device)
    y = fp8_linear(x, w, out=out_store[:, 2 : 2 + n])
    assert y.data_ptr() == out_store[:, 2:].data_ptr()
    close(y, *of.product(store[:, 8 : 8 + k].double().numpy(), wv))
    assert not out_store[:, :2].any() and not out_store[:, 2 + n :].any()


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize("m", [20, 150])
def test_linear_nan_stays_in_its_row_and_block(m, act, device):
    """A NaN of x makes its row NaN, one code of a weight its column, one scale of a weight the columns of its block."""
    n, k = 300, 272
    xs, ws = randn(5, m, k), randn(6, n, k)
    xs[7, 260] = float("nan")
    x, xv = operand(xs, act, device)
    w, wv = operand(ws, "fp8", device, 128)
    w.codes.view(torch.uint8)[33, 3] = 0x7F
    w.scales[1, 2] = float("nan")
    y = fp8_linear(x, w).cpu()
    columns = [33, *range(128, 256)]
    assert torch.isnan(y[7]).all() and torch.isnan(y[:, columns]).all()
    rest_rows, rest_cols = [i for i in range(m) if i != 7], [j for j in range(n) if j not in columns]
    close(y[rest_rows][:, rest_cols], *of.product(xv[rest_rows], wv[rest_cols], both=act == "fp8"))


def test_linear_no_rows_and_repeatable(device):
    w, _ = weight(9, 512, 1024, device=device)
    assert fp8_linear(torch.zeros(0, 1024, dtype=torch.bfloat16, device=device), w).shape == (0, 512)
    x = randn(10, 100, 1024).to(device)
    for xi in (x, quantize_fp8(x)):
        first = fp8_linear(xi, w)
        for _ in range(3):
            assert torch.equal(fp8_linear(xi, w), first)


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize("counts", RAGGED, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("gather", [False, True])
def test_expert_linear_ragged(counts, act, gather, device):
    n, k = (264, 336) if len(counts) < 100 else (40, 96)
    experts, rows = len(counts), sum(counts)
    rng = np.random.default_rng(rows + experts)
    swiglu, bias = rows % 2 == 1, experts % 2 == 1
    n = 256 if swiglu else n
    source = max(1, rows // 2) if gather else rows
    tokens = rng.integers(0, source, rows).astype(np.int32)
    x, xv = operand(randn(11, source, k), act, device)
    w, wv = weight(12, experts, n, k, device=device)
    b = randn(13, experts, n) if bias else None
    y = expert_linear(x, w, segments(counts).to(device), tokens=torch.from_numpy(tokens).to(device) if gather else None,
                      bias=None if b is None else b.to(device), swiglu=swiglu)
    start = 0
    for e, count in enumerate(counts):
        own = np.arange(start, start + count)
        if count:
            close(y[start : start + count],
                  *of.product(xv[tokens[own] if gather else own], wv[e], None if b is None else b[e].double().numpy(), swiglu,
                              act == "fp8"))
        start += count


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize("counts", [[3, 0, 2], [100, 0, 90]])
def test_expert_linear_rows_without_expert_stay(counts, act, device):
    n, k, rows = 64, 256, sum(counts) + 40
    x, xv = operand(randn(14, 50, k), act, device)
    w, wv = weight(15, 3, n, k, device=device)
    tokens = torch.full((rows,), -1, dtype=torch.int32)
    tokens[: sum(counts)] = torch.arange(sum(counts)) % 50
    out = torch.full((rows, n), 3.0, dtype=torch.bfloat16, device=device)
    expert_linear(x, w, segments(counts).to(device), tokens=tokens.to(device), out=out)
    assert (out[sum(counts) :] == 3.0).all()
    close(out[: counts[0]], *of.product(xv[tokens[: counts[0]].numpy()], wv[0], both=act == "fp8"))


def test_products_on_a_side_stream_and_in_a_graph(device):
    w, _ = weight(20, 512, 512, device=device)
    x = randn(21, 24, 512).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = fp8_linear(quantize_fp8(x), w)
    side.synchronize()
    assert torch.equal(y, fp8_linear(quantize_fp8(x), w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp8_linear(quantize_fp8(x), w)
        back = dequantize_fp8(quantize_fp8(x, block_rows=128))
    for seed in range(3):
        x.copy_(randn(30 + seed, 24, 512).to(device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fp8_linear(quantize_fp8(x), w))
        assert torch.equal(back, dequantize_fp8(quantize_fp8(x, block_rows=128)))


def test_refusals(device):
    x = randn(1, 4, 256).to(device)
    w, w3 = quantize_fp8(x, block_rows=128), quantize_fp8(randn(2, 2, 256, 256).to(device), block_rows=128)
    many = quantize_fp8(randn(3, 256, 256).to(device), block_rows=128)
    rows = quantize_fp8(x)
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device=device)
    mx = quantize_mxfp4(x)
    cases = [
        (lambda: quantize_fp8(x[:, :24]), "multiple of 16"),
        (lambda: quantize_fp8(x[:, 1:17]), "16-byte aligned"),
        (lambda: quantize_fp8(randn(1, 2, 4, 64).to(device)[:, :, :32]), "contiguous"),
        (lambda: quantize_fp8(x.clone().requires_grad_()), "inference-only"),
        (lambda: dequantize_fp8(FP8Tensor(rows.codes, rows.scales[:, :1].contiguous())), "one scale"),
        (lambda: dequantize_fp8(FP8Tensor(rows.codes.view(torch.uint8), rows.scales)), "codes must be"),
        (lambda: dequantize_fp8(rows, out=x[:, :128]), "out must be"),
        (lambda: fp8_linear(x[:, :128], w), "inner dimension"),
        (lambda: fp8_linear(quantize_fp8(x[:, :128]), w), "inner dimension"),
        (lambda: fp8_linear(many, many), "of a row"),
        (lambda: fp8_linear(x, rows), "128 rows"),
        (lambda: fp8_linear(x, w, swiglu=True), "whole blocks"),
        (lambda: fp8_linear(mx, w), "MXFP4"),
        (lambda: expert_linear(rows, randn(1, 2, 8, 256).to(device), offsets), "needs an FP8 weight"),
        (lambda: fp8_linear(x, w, out=torch.empty(4, 3, dtype=torch.bfloat16, device=device)), "out must be"),
        (lambda: expert_linear(x, w3, offsets[:2]), "offsets must be contiguous"),
        (lambda: fp8_linear(x.clone().requires_grad_(), w), "inference-only"),
    ]
    for call, match in cases:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(TypeError, match="bool"):
        fp8_linear(x, w, swiglu=1)
    shared = torch.zeros(8, 256, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="share storage"):
        fp8_linear(shared[:4], w, out=shared[4:, :4])


# --------------------------------------------------------------------------
# Every kernel, forced
# --------------------------------------------------------------------------

STREAM = [(_lib.LF_EXPERT_STREAM, part, c) for part in (16, 32, 64) for c in (16, 32)]


def tiles(act):
    """Tile heights that there are beside a width: the sums leave no registers for more."""
    most = {"fp8": (256, 192), "bf16": (192, 128)}[act]
    return [(_lib.LF_EXPERT_TILE, r, c) for c in (64, 128, 192, 256) for r in (64, 128, 192, 256) if r <= most[c == 256]]


PLANS = {act: STREAM + [(_lib.LF_EXPERT_ROWS, 0, 128)] + tiles(act) for act in ("bf16", "fp8")}
BOTH = [(act, plan) for act in PLANS for plan in PLANS[act]]


def name(v):
    return "-".join(map(str, v)) if isinstance(v, tuple) else v


def forced(x, w, plan, **options):
    arguments = dict(experts=None, offsets=None, tokens=None, bias=None, swiglu=False, out=None)
    return product(x, w, **{**arguments, **options}, plan=_lib.ExpertPlan(*plan))


@pytest.mark.parametrize("act,plan", BOTH, ids=name)
@pytest.mark.parametrize("k", [16, 128, 416, 2896])
def test_every_plan(act, plan, k, device):
    counts = [130, 0, 1, 64, 257, 33, 190]
    n, rows = 328, sum(counts)
    x, xv = operand(randn(k, rows, k), act, device)
    w, wv = weight(k + 1, len(counts), n, k, device=device)
    b = randn(k + 2, len(counts), n)
    y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device), bias=b.to(device))
    start = 0
    for e, count in enumerate(counts):
        if count:
            close(y[start : start + count], *of.product(xv[start : start + count], wv[e], b[e].double().numpy(), False, act == "fp8"))
        start += count


@pytest.mark.parametrize("act,plan", BOTH, ids=name)
@pytest.mark.parametrize("n", [256, 768])
def test_every_plan_swiglu(act, plan, n, device):
    k, counts = 544, [70, 3, 200]
    x, xv = operand(randn(n, sum(counts), k), act, device)
    w, wv = weight(n + 1, len(counts), n, k, device=device)
    b = randn(n + 2, len(counts), n)
    y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device), bias=b.to(device), swiglu=True)
    start = 0
    for e, count in enumerate(counts):
        close(y[start : start + count], *of.product(xv[start : start + count], wv[e], b[e].double().numpy(), True, act == "fp8"))
        start += count


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize("k", [8208, 12304])
def test_long_k_exact_on_every_kernel(act, k, device):
    """Small integers with scales that are powers of two: fp32 sums in any order are exact (and products of
    integers to 8 within 13 bits of one another), so results are equal."""
    rng = np.random.default_rng(k)
    counts, n = [70, 0, 1, 130], 136
    blocks = -(-k // 128)

    def small(shape, rows):
        v = rng.integers(-8, 9, shape)
        codes = torch.from_numpy(v).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        lead = (*shape[:-2], -(-shape[-2] // rows), blocks)
        scales = np.exp2(rng.integers(-1, 2, lead)).astype(np.float32)
        return held(codes, scales, device), of.values(codes, scales)

    if act == "fp8":
        x, xv = small((sum(counts), k), 1)
    else:
        xv = rng.integers(-8, 9, (sum(counts), k)).astype(np.float64)
        x = torch.from_numpy(xv).bfloat16().to(device)
    w, wv = small((len(counts), n, k), 128)
    own = np.repeat(np.arange(len(counts)), counts)
    exact = np.concatenate([xv[own == e] @ wv[e].T for e in range(len(counts))])
    assert max((np.abs(xv[own == e]) @ np.abs(wv[e]).T).max() for e in (0, 2, 3)) * 4 < 2**24
    expected = torch.from_numpy(exact).float().bfloat16()
    for plan in PLANS[act]:
        y = forced(x, w, plan, experts=len(counts), offsets=segments(counts).to(device))
        assert torch.equal(y.cpu(), expected), plan


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_extreme_scales_on_every_kernel(act, device):
    """Scales from 0 and subnormals to 2^100, weights beside them that bring the sums back into range."""
    m, n, k = 140, 264, 2128
    xs = randn(7, m, k)
    w, _ = weight(8, n, k, device=device)
    exponents = torch.tensor([-100.0, 0.0, 60.0, 100.0, -60.0])
    w.scales.copy_(torch.exp2(exponents[torch.arange(w.scales.numel()) % 5]).reshape(w.scales.shape).to(device))
    w.scales[0, 3] = 0.0
    wv = of.values(w.codes.view(torch.uint8).cpu().numpy(), w.scales.cpu().numpy())
    x, xv = operand(xs, act, device)
    if act == "fp8":
        x.scales[::3] = 1e-41
        x.scales[1::3] *= 2.0**-70
        xv = of.values(x.codes.view(torch.uint8).cpu().numpy(), x.scales.cpu().numpy())
    y, bound = of.product(xv, wv, both=act == "fp8")
    # (A product of two scales below the normal range may be flushed: at most 2^-126 of a block's code sum of 448^2 128.)
    bound = bound + 2.0**-126 * 448**2 * 128 * 17
    for plan in PLANS[act]:
        close(forced(x, FP8Tensor(w.codes[None], w.scales[None]), plan, experts=1, offsets=segments([m]).to(device)), y, bound)


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_tiles_of_one_dense_product(act, device):
    """Several row and column tiles of one segment; results do not depend on the tile."""
    m, n, k = 1300, 712, 528
    x, xv = operand(randn(40, m, k), act, device)
    w, wv = weight(41, 1, n, k, device=device)
    first = None
    for plan in tiles(act):
        y = forced(x, w, plan, experts=1, offsets=segments([m]).to(device))
        if first is None:
            first = y
            close(y, *of.product(xv, wv[0], both=act == "fp8"))
        assert torch.equal(y, first), plan


@pytest.mark.parametrize("act", ["bf16", "fp8"])
def test_gathered_rows_and_output_of_any_alignment(act, device):
    m, n, k = 200, 264, 592
    x, xv = operand(randn(42, m, k), act, device)
    w, wv = weight(43, 1, n, k, device=device)
    tokens = torch.arange(m - 1, -1, -1, dtype=torch.int32, device=device)
    want = of.product(xv[::-1], wv[0], both=act == "fp8")
    for plan in PLANS[act]:
        for pad, at in ((0, 0), (8, 8), (3, 1)):
            store = torch.zeros(m, n + pad, dtype=torch.bfloat16, device=device)
            out = store[:, at : at + n]
            forced(x, w, plan, experts=1, offsets=segments([m]).to(device), tokens=tokens, out=out)
            close(out, *want)
            assert not store[:, :at].any() and not store[:, at + n :].any()


@pytest.mark.parametrize("act", ["bf16", "fp8"])
@pytest.mark.parametrize("over", [False, True])
def test_rows_around_2_gib(act, over, device):
    """x whose rows end just below and above 2 GiB (the tiles' offsets): only its last rows are named."""
    n, k, rows = 96, 4096, 130
    total = 2**31 // (k if act == "fp8" else 2 * k) + (5 if over else -1)
    last, lv = operand(randn(64, rows, k), act, device)
    w, wv = weight(65, 1, n, k, device=device)
    tokens = torch.arange(total - rows, total, dtype=torch.int32, device=device)
    if act == "fp8":
        x = FP8Tensor(torch.zeros(total, k, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                      torch.zeros(total, k // 128, device=device))
        x.codes.view(torch.uint8)[-rows:], x.scales[-rows:] = last.codes.view(torch.uint8), last.scales
    else:
        x = torch.zeros(total, k, dtype=torch.bfloat16, device=device)
        x[-rows:] = last
    close(expert_linear(x, w, segments([rows]).to(device), tokens=tokens), *of.product(lv, wv[0], both=act == "fp8"))
    for plan in PLANS[act]:
        if over and plan[0] == _lib.LF_EXPERT_TILE:
            with pytest.raises(ValueError, match="tiles"):
                forced(x, w, plan, experts=1, offsets=segments([rows]).to(device), tokens=tokens)
        else:
            close(forced(x, w, plan, experts=1, offsets=segments([rows]).to(device), tokens=tokens), *of.product(lv, wv[0], both=act == "fp8"))


def test_weights_past_4_gib(device):
    """Offsets into the weight that do not fit 32 bits: the last expert of 4.5 GiB."""
    n, k, experts = 4096, 4096, 288
    last, wv = weight(18, n, k, device=device)
    w = FP8Tensor(torch.zeros(experts, n, k, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                  torch.zeros(experts, 32, 32, device=device))
    w.codes.view(torch.uint8)[-1] = last.codes.view(torch.uint8)
    w.scales[-1] = last.scales
    x, offsets = randn(19, 130, k).to(device), torch.zeros(experts + 1, dtype=torch.int32)
    columns = np.arange(0, n, 97)
    for rows in (2, 130):
        offsets[-1] = rows
        for act in ("bf16", "fp8"):
            xi, xv = operand(x[:rows].cpu(), act, device)
            close(expert_linear(xi, w, offsets.to(device))[:, columns], *of.product(xv, wv[columns], both=act == "fp8"))
