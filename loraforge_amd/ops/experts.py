"""Mixture-of-experts operators on gfx950: routing, the product grouped by expert, the weighted sum back.

A block of experts runs as

    r = route_experts(router_logits, top_k)
    h = expert_linear(x, gate_up, r.offsets, tokens=r.tokens, swiglu=True)
    y = combine_experts(expert_linear(h, down, r.offsets), r.positions, r.weights, base=shared)

with no host synchronisation: segment bounds stay on the device, buffers are
sized for every choice (``tokens * top_k`` rows), and the calls can be captured
in a HIP graph. Expert weights are bf16 or MXFP4 ``[E, N, K]``. The operators are
for inference: tensors that require gradients are refused.
"""

from __future__ import annotations

from dataclasses import dataclass

from .. import _lib
from ..annotations import ExperimentalAPI
from ._checks import distinct_output, require_arch, tensor
from .mxfp4 import MXFP4Tensor, product

MAX_EXPERTS = 1024
MAX_TOP = 64


@dataclass
class ExpertRouting:
    """The choices of ``T`` tokens among ``E`` experts, and their order by expert.

    ``weights`` fp32 and ``experts`` int32 ``[T, k]`` (-1 with weight 0 where a
    token may not choose that many); ``offsets`` int32 ``[E + 1]``: expert
    ``e`` owns the places ``offsets[e]`` to ``offsets[e + 1]``; ``tokens`` int32
    ``[T * k]``: the token at each place (-1 from ``offsets[E]`` on);
    ``positions`` int32 ``[T, k]``: the place of each choice (-1 for none).
    Within an expert the places are in order of token, then choice.
    """

    weights: object
    experts: object
    offsets: object
    tokens: object
    positions: object


@ExperimentalAPI(reason="Mixture-of-experts routing; gfx950 HIP kernel.")
def route_experts(logits, top_k: int, *, renormalize: bool = True) -> ExpertRouting:
    """Top-k of the softmax of ``logits`` (bf16 or fp32 ``[T, E]``, E up to 1024, k up to 64).

    The ``top_k`` largest logits of a token are chosen, of equal ones the
    lowest expert first; -inf marks an expert that the token may not choose. A
    weight is the softmax probability over all experts, with ``renormalize``
    divided by the sum of the token's chosen ones. A token whose logits hold NaN or
    +inf gets NaN weights for its choices (NaN ranks below every number and is not
    chosen: of NaN and -inf alone, none is).
    """
    import torch

    if getattr(logits, "is_cuda", False):
        done = _lib.binding().route(logits, top_k, renormalize)
        if done is not None:
            return ExpertRouting(*done)
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must have dtype torch.bfloat16 or torch.float32")
    tensor(logits, "logits", 2, logits.dtype)
    count, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"logits must have 1..{MAX_EXPERTS} experts")
    if type(top_k) is not int or not 1 <= top_k <= min(experts, MAX_TOP):
        raise ValueError(f"top_k must be in 1..min(experts, {MAX_TOP})")
    if type(renormalize) is not bool:
        raise TypeError("renormalize must be a bool")
    stride = logits.stride(0) if count > 1 else experts
    if logits.stride(1) != 1 or stride < experts:
        raise ValueError("logits must have unit column stride and rows apart")
    if count * top_k >= 2**31 - 2**16:
        raise ValueError("tokens * top_k must fit signed int32 indexing")
    require_arch(logits.device)
    lib = _lib.library()
    integers = dict(dtype=torch.int32, device=logits.device)
    r = ExpertRouting(
        torch.empty(count, top_k, dtype=torch.float32, device=logits.device),
        torch.empty(count, top_k, **integers),
        torch.empty(experts + 1, **integers),
        torch.empty(count * top_k, **integers),
        torch.empty(count, top_k, **integers),
    )
    size = lib.lf_route_experts_workspace_size(count, experts)
    scratch = torch.empty(size, dtype=torch.uint8, device=logits.device) if size else None
    with torch.cuda.device(logits.device):
        _lib.check(
            lib.lf_route_experts(
                logits.data_ptr(), logits.dtype == torch.float32, count, experts, stride, top_k, renormalize,
                r.weights.data_ptr(), r.experts.data_ptr(), r.offsets.data_ptr(), r.tokens.data_ptr(),
                r.positions.data_ptr(), _lib.ptr(scratch), size, _lib.stream_of(logits.device)))
    return r


@ExperimentalAPI(reason="Product grouped by expert; gfx950 HIP kernel.")
def expert_linear(x, weight, offsets, *, tokens=None, bias=None, swiglu: bool = False, out=None):
    """Rows ``offsets[e]`` to ``offsets[e + 1]`` times the transpose of ``weight[e]``, for every expert.

    ``weight`` is bf16 ``[E, N, K]`` (K a multiple of 8) or an ``MXFP4Tensor``
    of that shape; ``x`` bf16 ``[rows, K]`` with 16-byte aligned rows, or an
    ``MXFP4Tensor`` beside an MXFP4 weight. With ``tokens`` (int32, one entry per
    row of the result) row ``p`` is ``x[tokens[p]]``, so the rows are gathered by the
    product itself; without, ``x`` is in expert order already. ``bias`` is bf16
    ``[E, N]``, ``swiglu`` as in ``mxfp4_linear``. fp32 sums, rounded once to bf16.
    Rows past ``offsets[E]`` belong to no expert and are left as they are.
    """
    import torch

    if not isinstance(weight, (torch.Tensor, MXFP4Tensor)):
        raise TypeError("weight must be a torch.Tensor or an MXFP4Tensor")
    if weight.ndim != 3:
        raise ValueError("weight must be 3D, [experts, n, k]")
    return product(x, weight, experts=weight.shape[0], offsets=offsets, tokens=tokens, bias=bias, swiglu=swiglu, out=out)


@ExperimentalAPI(reason="Weighted sum of the experts' rows; gfx950 HIP kernel.")
def combine_experts(rows, positions, weights, *, base=None, out=None):
    """``out[t] = base[t] + sum_j weights[t, j] * rows[positions[t, j]]`` in bf16, fp32 sums in order of ``j``.

    ``rows`` bf16 ``[R, N]``, ``positions`` int32 and ``weights`` fp32 ``[T, k]``
    (``ExpertRouting``; -1 adds nothing), ``base`` bf16 ``[T, N]`` (a shared
    expert's output or the residual). ``out`` may be ``base``.
    """
    import torch

    if getattr(rows, "is_cuda", False):
        done = _lib.binding().combine(rows, positions, weights, base, out)
        if done is not None:
            return done
    tensor(rows, "rows", 2, torch.bfloat16)
    tensor(positions, "positions", 2, torch.int32, rows.device)
    tensor(weights, "weights", 2, torch.float32, rows.device)
    if positions.shape != weights.shape or positions.shape[1] < 1 or not positions.is_contiguous() or not weights.is_contiguous():
        raise ValueError("positions and weights must be contiguous [tokens, k]")
    count, n = positions.shape[0], rows.shape[1]
    if n < 1:
        raise ValueError("rows must have columns")

    def stride(t, name):
        step = t.stride(0) if t.shape[0] > 1 else n
        if t.numel() and (t.stride(1) != 1 or step < n):
            raise ValueError(f"{name} must have unit column stride and rows apart")
        return step

    if base is not None:
        tensor(base, "base", 2, torch.bfloat16, rows.device)
        if base.shape != (count, n):
            raise ValueError("base must be [tokens, columns]")
    if out is None:
        out = torch.empty(count, n, dtype=torch.bfloat16, device=rows.device)
    tensor(out, "out", 2, torch.bfloat16, rows.device)
    if out.shape != (count, n):
        raise ValueError("out must be [tokens, columns]")
    same = base is not None and out.data_ptr() == base.data_ptr() and out.stride() == base.stride()
    distinct_output(out, (rows, positions, weights, None if same else base))
    require_arch(rows.device)
    if count == 0:
        return out
    with torch.cuda.device(rows.device):
        _lib.check(
            _lib.library().lf_combine_experts(
                rows.data_ptr(), rows.shape[0], stride(rows, "rows"), positions.data_ptr(), weights.data_ptr(), count,
                positions.shape[1], n, _lib.ptr(base), 0 if base is None else stride(base, "base"), out.data_ptr(),
                stride(out, "out"), _lib.stream_of(rows.device)))
    return out
