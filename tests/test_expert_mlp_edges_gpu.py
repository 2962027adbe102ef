"""Edges of the whole expert MLP (``expert_mlp``): weights that are not finite, what the layout of its inputs may not change, and
the sizes at which each variant of its kernels runs.

Infinite values follow the formula: a product of an infinite weight and a value that is not
zero is infinite with their sign, so a sum that holds one is, and every other output keeps its bits.
"""

import numpy as np
import pytest
import torch

from loraforge_amd.ops import expert_mlp
from oracle import experts as ox
from oracle import fp8 as of
from tests.test_expert_mlp_gpu import KINDS, case, close, expected, values
from tests.test_native_calls_gpu import both

pytestmark = pytest.mark.gpu

# Two launches (16 and 8 waves in the second), the first one ahead of the operators, the operators alone; of
# the down product the weight stream, a wave for 16 weight rows and row tiles.
FORMS = [(1, 8, 8, 512, 256), (3, 8, 2, 512, 256), (8, 8, 2, 2688, 128), (9, 24, 4, 512, 256), (30, 8, 2, 2176, 256), (40, 8, 2, 512, 256),
         (64, 24, 4, 1024, 1024), (128, 24, 4, 640, 512)]


def activations(x, gate_up, expert):
    """silu(gate) up of every token for one expert, in 64 bits."""
    gu = values(gate_up if isinstance(gate_up, torch.Tensor) else type(gate_up)(gate_up.codes[expert : expert + 1], gate_up.scales[expert : expert + 1]))
    return ox.product(x.double().cpu().numpy(), gu[expert if isinstance(gate_up, torch.Tensor) else 0], None, True)[0]


def chosen_case(kind, tokens, experts, *sizes, device):
    """``case`` with expert 1 among the first token's choices."""
    x, logits, gate_up, down = case(kind, tokens, experts, *sizes, device, seed=tokens)
    logits[0, 1] = 9.0
    return x, logits, gate_up, down


def hit_by(logits, top, expert):
    _, chosen, *_ = ox.route(logits.double().cpu().numpy(), top)
    return torch.from_numpy((chosen == expert).any(1))


@pytest.mark.parametrize("tokens,experts,top,hidden,inter", FORMS)
def test_infinite_down_weights(tokens, experts, top, hidden, inter, device):
    x, logits, gate_up, down = chosen_case("bf16", tokens, experts, hidden, inter, device=device)
    clean = expert_mlp(x, logits, gate_up, down, top)
    down[1, 3, 5], down[1, 140, inter - 1] = float("inf"), float("-inf")
    y = expert_mlp(x, logits, gate_up, down, top).cpu()
    h, hit = activations(x, gate_up, 1), hit_by(logits, top, 1)
    want = clean.cpu().clone()
    want[:, 3] = torch.where(hit, torch.from_numpy(h[:, 5] * np.inf).bfloat16(), want[:, 3])
    want[:, 140] = torch.where(hit, torch.from_numpy(h[:, inter - 1] * -np.inf).bfloat16(), want[:, 140])
    assert (np.abs(h[:, [5, inter - 1]]) > 1e-5).all()  # (a sign that fp32 sums do not change)
    assert torch.equal(y, want)


@pytest.mark.parametrize("tokens,experts,top,hidden,inter", FORMS)
def test_infinite_scale_of_a_down_block(tokens, experts, top, hidden, inter, device):
    """A block's products are summed, then scaled: infinite with the sum's sign."""
    x, logits, gate_up, down = chosen_case("fp8", tokens, experts, hidden, inter, device=device)
    clean = expert_mlp(x, logits, gate_up, down, top).cpu()
    down.scales[1, 1, 0] = float("inf")
    y = expert_mlp(x, logits, gate_up, down, top).cpu()
    h, hit = activations(x, gate_up, 1), hit_by(logits, top, 1)
    codes = of.values(down.codes[1].view(torch.uint8).cpu().numpy(), np.ones(down.scales.shape[1:], np.float32))
    part = codes[128:256, :128]
    sums, size = h[:, :128] @ part.T, np.abs(h[:, :128]) @ np.abs(part).T
    clear = torch.from_numpy(np.abs(sums) > 2.0**-12 * size) & hit[:, None]
    assert clear.sum() >= 0.9 * 128 * hit.sum()
    want = clean.clone()
    want[:, 128:256] = torch.where(hit[:, None], torch.from_numpy(sums * np.inf).bfloat16(), want[:, 128:256])
    got = y.clone()
    got[:, 128:256] = torch.where(hit[:, None] & ~clear, want[:, 128:256], got[:, 128:256])
    assert torch.equal(got, want)
    assert not torch.isfinite(y[hit][:, 128:256]).any()


@pytest.mark.parametrize("tokens,experts,top,hidden,inter", FORMS)
def test_infinite_gate_and_up_weights(tokens, experts, top, hidden, inter, device):
    """silu(gate) times an infinite up is infinite, so are all outputs of its token with the signs of the down weights."""
    x, logits, gate_up, down = chosen_case("bf16", tokens, experts, hidden, inter, device=device)
    clean = expert_mlp(x, logits, gate_up, down, top)
    h, hit = activations(x, gate_up, 1), hit_by(logits, top, 1)
    gate_up[1, inter + 7, 11] = float("inf")
    y = expert_mlp(x, logits, gate_up, down, top).cpu()
    gate = x.double().cpu().numpy() @ gate_up[1, 7].double().cpu().numpy()
    sign = np.sign(gate) * np.sign(x[:, 11].double().cpu().numpy())
    want = clean.cpu().clone()
    with np.errstate(invalid="ignore"):  # (infinity times a weight of zero)
        want[hit] = torch.from_numpy((sign[:, None] * np.inf) * down[1, :, 7].double().cpu().numpy()[None])[hit].bfloat16()
    assert (np.abs(gate) > 1e-4).all() and (sign != 0).all()
    assert torch.equal(y[~hit], want[~hit]) and np.array_equal(y.float().numpy(), want.float().numpy(), equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,experts", [(2, 8), (3, 8), (8, 8), (8, 300), (9, 8)])
def test_rows_of_x_that_span_2_gib(kind, tokens, experts, device, monkeypatch):
    """Bit for bit the result of the same rows beside each other, on the native path and in Python."""
    x, logits, gate_up, down = case(kind, tokens, experts, 256, 128, device)
    base = x.flip(0)
    want = expert_mlp(x, logits, gate_up, down, 2, base=base)
    span = 2**30 // (tokens - 1) // 8 * 8 + 64
    far = torch.empty((tokens - 1) * span + 256, dtype=torch.bfloat16, device=device).as_strided((tokens, 256), (span, 1))
    far.copy_(x)
    taken, python = both(monkeypatch, lambda: expert_mlp(far, logits, gate_up, down, 2, base=base))
    assert torch.equal(taken, want) and torch.equal(python, want)


# --------------------------------------------------------------------------
# Sizes at which another variant of a kernel runs, at 16 bits between the products
# --------------------------------------------------------------------------

PAIRS = 2.0**-16 + 2.0**-20  # a pair of bf16 is off by 2^-8 of 2^-8 of the value, the fp32 activation by 2^-20


def check(y, x, logits, gate_up, down, top, **options):
    """Within the bound of pairs; of many outputs the deviation is that of their own rounding.

    An error uniform within half a step has 2^-7 / sqrt(12) of the power of two below the value in the root
    mean square, 0.00166 of values that are spread smoothly; rounding the intermediate to bf16 would make it 0.0024.
    """
    want, bound = expected(x, logits, gate_up, down, top, between=PAIRS, **options)
    close(y, (want, bound))
    if want.size >= 4096:
        assert (y.double().cpu().numpy() - want).std() <= 2.0**-9 * want.std()


def few(x, logits, tokens):
    return x[:tokens], logits[:tokens]


@pytest.mark.parametrize("kind,hidden", [("bf16", 4104), ("bf16", 8192), ("fp8", 4112), ("fp8", 8192), ("mxfp4", 4224), ("mxfp4", 8192)])
def test_wide_hidden(kind, hidden, device):
    """All registers of x: through LDS while it fits, else by loads (MXFP4, FP8: exchanged between the quarters of a wave)."""
    x, logits, gate_up, down = case(kind, 16, 6, hidden, 128, device, seed=hidden)
    for tokens in (1, 2, 6, 7, 8, 9, 16):
        xs, ls = few(x, logits, tokens)
        check(expert_mlp(xs, ls, gate_up, down, 2), xs, ls, gate_up, down, 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hidden", [2176, 3200, 4096])
def test_x_past_what_lds_holds(kind, hidden, device):
    """9 to 16 tokens whose x does not fit LDS beside two workgroups of a CU."""
    x, logits, gate_up, down = case(kind, 16, 6, hidden, 128, device, seed=hidden)
    for tokens in (9, 12, 16):
        xs, ls = few(x, logits, tokens)
        check(expert_mlp(xs, ls, gate_up, down, 2), xs, ls, gate_up, down, 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("experts,top", [(65, 1), (100, 8), (128, 16), (129, 16), (130, 8), (200, 1), (256, 16), (257, 3)])
def test_many_experts(kind, experts, top, device):
    """Routing in the first launch by ranks (1 and 2 tokens) and in rounds, of up to 128 and up to 256 experts."""
    x, logits, gate_up, down = case(kind, 20, experts, 256, 128, device, seed=experts)
    tied = torch.round(logits)
    masked = logits.clone()
    masked[torch.rand(masked.shape, generator=torch.Generator().manual_seed(top)) < 0.95] = -np.inf
    masked[1], masked[:, experts - 1] = -np.inf, 0.5
    masked[3] = -np.inf
    for tokens in (1, 2, 5, 20):
        for all_logits, renormalize in ((logits, True), (tied, False), (masked, True), (tied.bfloat16(), True)):
            xs, ls = few(x, all_logits, tokens)
            y = expert_mlp(xs, ls, gate_up, down, top, renormalize=renormalize)
            check(y, xs, ls, gate_up, down, top, renormalize=renormalize)


@pytest.mark.parametrize("kind,hidden,inter", [("bf16", 136, 72), ("bf16", 520, 264), ("bf16", 24, 8), ("bf16", 1032, 328), ("fp8", 144, 128),
                                               ("fp8", 528, 256), ("fp8", 1040, 384), ("mxfp4", 96, 32), ("mxfp4", 544, 288), ("mxfp4", 384, 640)])
def test_widths_with_a_remainder(kind, hidden, inter, device):
    """Remainders of every loop and tile, with a base, of 1 to 160 tokens (routed by ranks, in rounds, in a chain; in row tiles)."""
    x, logits, gate_up, down = case(kind, 160, 15, hidden, inter, device, seed=hidden)
    base = x.flip(0)
    for tokens in (1, 2, 5, 8, 16, 20, 40, 160):
        (xs, ls), bs = few(x, logits, tokens), base[:tokens]
        for b in (None, bs):
            check(expert_mlp(xs, ls, gate_up, down, 3, base=b), xs, ls, gate_up, down, 3, base=b)


@pytest.mark.parametrize("kind", KINDS)
def test_pairs_in_row_tiles(kind, device):
    """The down product of many rows: tiles of up to 256 rows, experts past the 64th among them."""
    for tokens, experts, top, hidden, inter in ((128, 24, 4, 640, 512), (200, 70, 8, 512, 256), (256, 130, 8, 264 if kind == "bf16" else 640, 256)):
        x, logits, gate_up, down = case(kind, tokens, experts, hidden, inter, device, seed=experts)
        check(expert_mlp(x, logits, gate_up, down, top), x, logits, gate_up, down, top)
