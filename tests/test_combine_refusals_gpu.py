"""``combine_experts`` with a base beside an output that the native call path cannot take.

A wrong output is refused with the operator's own error, one that only the Python path takes is
served, whether or not the native path has been enabled by an earlier call.
"""

import pytest
import torch

from loraforge_amd.ops import combine_experts
from tests.test_native_calls_gpu import both

pytestmark = pytest.mark.gpu

TOKENS, TOP, N = 6, 2, 64


class Subclass(torch.Tensor):
    pass


def arguments(device):
    rows = torch.randn(TOKENS * TOP, N, device=device).bfloat16()
    positions = torch.arange(TOKENS * TOP, dtype=torch.int32, device=device).reshape(TOKENS, TOP)
    weights = torch.rand(TOKENS, TOP, device=device)
    base = torch.randn(TOKENS, N, device=device).bfloat16()
    return (rows, positions, weights), base


def empty(device, *shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=device)


@pytest.mark.parametrize("with_base", [True, False])
@pytest.mark.parametrize(
    "make,match",
    [
        (lambda device: empty(device, TOKENS, N + 1), "out must be"),
        (lambda device: empty(device, TOKENS - 1, N), "out must be"),
        (lambda device: empty(device, TOKENS * N), "out must be 2D"),
        (lambda device: empty(device, TOKENS, N, dtype=torch.float32), "out must be 2D"),
        (lambda device: empty("cpu", TOKENS, N), "same CUDA"),
        (lambda device: empty(device, N, TOKENS).t(), "unit column stride"),
        (lambda device: empty(device, TOKENS, N).requires_grad_(), "inference-only"),
    ],
    ids=["columns", "rows", "vector", "dtype", "cpu", "columns-apart", "gradient"],
)
def test_wrong_outputs_are_refused(make, match, with_base, device):
    given, base = arguments(device)
    combine_experts(*given, base=base)  # (the native path is on from here)
    with pytest.raises(ValueError, match=match):
        combine_experts(*given, base=base if with_base else None, out=make(device))


def test_an_output_of_no_tensor_is_refused(device):
    given, base = arguments(device)
    combine_experts(*given, base=base)
    with pytest.raises(TypeError, match="torch.Tensor"):
        combine_experts(*given, base=base, out=[0.0])


@pytest.mark.parametrize("with_base", [True, False])
def test_a_subclass_is_served_in_python(monkeypatch, with_base, device):
    given, base = arguments(device)
    base = base if with_base else None
    expected = combine_experts(*given, base=base)
    out = empty(device, TOKENS, N).as_subclass(Subclass)
    for y in both(monkeypatch, lambda: combine_experts(*given, base=base, out=out), native=False):
        assert y is out and torch.equal(y.as_subclass(torch.Tensor), expected)
