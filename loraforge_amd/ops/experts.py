"""Mixture-of-experts operators on gfx950: routing, the product grouped by expert, the weighted sum back.

A block of experts runs as

    r = route_experts(router_logits, top_k)
    h = expert_linear(x, gate_up, r.offsets, tokens=r.tokens, swiglu=True)
    y = combine_experts(expert_linear(h, down, r.offsets), r.positions, r.weights, base=shared)

with no host synchronisation: segment bounds stay on the device, buffers are
sized for every choice (``tokens * top_k`` rows), and the calls can be captured
in a HIP graph. ``expert_mlp`` is the whole block in one call. Expert weights are bf16, MXFP4 or
FP8 ``[E, N, K]``. The operators are for inference: tensors that require gradients are refused.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

from .. import _lib
from ..annotations import ExperimentalAPI
from ._checks import distinct_output, require_arch, tensor
from .fp8 import BLOCK, FP8Tensor, scaled
from .mxfp4 import MXFP4Tensor, packed, product

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

    ``weight`` is bf16 ``[E, N, K]`` (K a multiple of 8), or an ``MXFP4Tensor`` or
    ``FP8Tensor`` (a scale for each 128 x 128 block) of that shape; ``x`` bf16 ``[rows, K]``
    with 16-byte aligned rows, or an ``MXFP4Tensor`` beside an MXFP4 weight, an ``FP8Tensor``
    (a scale for each 128 values of a row) beside an FP8 one. With ``tokens`` (int32, one entry per
    row of the result) row ``p`` is ``x[tokens[p]]``, so the rows are gathered by the
    product itself; without, ``x`` is in expert order already. ``bias`` is bf16
    ``[E, N]``, ``swiglu`` as in ``mxfp4_linear`` and ``fp8_linear``. fp32 sums, rounded once to bf16.
    Rows past ``offsets[E]`` belong to no expert and are left as they are.
    """
    import torch

    if not isinstance(weight, (torch.Tensor, MXFP4Tensor, FP8Tensor)):
        raise TypeError("weight must be a torch.Tensor, an MXFP4Tensor or an FP8Tensor")
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


@ExperimentalAPI(reason="Whole mixture-of-experts MLP; gfx950 HIP kernels.")
def expert_mlp(x, logits, gate_up, down, top_k: int, *, renormalize: bool = True, base=None, out=None):
    """``out[t] = base[t] + sum_j weight_tj down_e (silu(gate_e x[t]) * (up_e x[t]))`` over the ``top_k`` experts of each token.

    ``x`` bf16 ``[T, H]`` with 16-byte aligned rows; ``logits`` bf16 or fp32 ``[T, E]``, choices and
    weights as ``route_experts`` makes them; ``gate_up`` ``[E, 2 I, H]`` (gate rows, then up rows) and
    ``down`` ``[E, H, I]``, each bf16, an ``MXFP4Tensor`` or an ``FP8Tensor`` (a scale for
    each 128 x 128 block); ``base`` bf16 ``[T, H]`` (a shared expert's output or the residual).
    ``out`` may be ``base``. A token that may choose no expert is left with ``base`` (or zeros).
    fp32 sums, rounded once to bf16; what lies between the products is held in 16 bits of mantissa where an expert
    has 32 choices or fewer on average and both weights are of one type, else in bf16, as ``expert_linear`` gives it
    (so also where the address of MXFP4 scales is no multiple of 4). Rows of ``x`` of up to 8 tokens that span 2 GiB are
    gathered first.
    """
    import torch

    if getattr(x, "is_cuda", False):
        done = _lib.binding().mlp(x, logits, gate_up, down, top_k, renormalize, base, out)
        if done is not None:
            return done
    for name, w in (("gate_up", gate_up), ("down", down)):
        if not isinstance(w, (torch.Tensor, MXFP4Tensor, FP8Tensor)):
            raise TypeError(f"{name} must be a torch.Tensor, an MXFP4Tensor or an FP8Tensor")
        if w.ndim != 3:
            raise ValueError(f"{name} must be 3D, [experts, n, k]")
    tensor(x, "x", 2, torch.bfloat16)
    for name, w in (("gate_up", gate_up), ("down", down)):
        _expert_weight(w, name, x.device)
    experts, hidden, inter = down.shape
    if tuple(gate_up.shape) != (experts, 2 * inter, hidden):
        raise ValueError("gate_up must be [experts, 2 * inter, hidden] beside down [experts, hidden, inter]")
    if isinstance(gate_up, FP8Tensor) and inter % BLOCK:
        raise ValueError("gate_up must hold whole blocks of 128 FP8 gate and up rows")
    count = x.shape[0]
    if x.shape[1] != hidden:
        raise ValueError("x must be [tokens, hidden]")
    if x.numel() and (x.stride(1) != 1 or x.data_ptr() % 16 or (count > 1 and (x.stride(0) < hidden or x.stride(0) % 8))):
        raise ValueError("x rows must be 16-byte aligned with unit stride")
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must have dtype torch.bfloat16 or torch.float32")
    tensor(logits, "logits", 2, logits.dtype, x.device)
    if tuple(logits.shape) != (count, experts):
        raise ValueError("logits must be [tokens, experts]")
    if type(renormalize) is not bool:
        raise TypeError("renormalize must be a bool")
    if base is not None:
        tensor(base, "base", 2, torch.bfloat16, x.device)
        if tuple(base.shape) != (count, hidden):
            raise ValueError("base must be [tokens, columns]")
    if out is None:
        out = torch.empty(count, hidden, dtype=torch.bfloat16, device=x.device)
    tensor(out, "out", 2, torch.bfloat16, x.device)
    if tuple(out.shape) != (count, hidden):
        raise ValueError("out must be [tokens, columns]")
    same = base is not None and out.data_ptr() == base.data_ptr() and out.stride() == base.stride()
    distinct_output(out, (x, logits, *_parts(gate_up), *_parts(down), None if same else base))
    if type(top_k) is not int or not 1 <= top_k <= min(experts, MAX_TOP):
        raise ValueError(f"top_k must be in 1..min(experts, {MAX_TOP})")
    if logits.numel() and (logits.stride(1) != 1 or (count > 1 and logits.stride(0) < experts)):
        raise ValueError("logits must have unit column stride and rows apart")
    for t, name in ((base, "base"), (out, "out")):
        if t is not None and t.numel() and (t.stride(1) != 1 or (count > 1 and t.stride(0) < hidden)):
            raise ValueError(f"{name} must have unit column stride and rows apart")
    require_arch(x.device)
    if count == 0:
        return out
    if type(gate_up) is type(down) and _expert_mlp(x, logits, gate_up, down, top_k, renormalize, base, out):
        return out
    r = route_experts(logits, top_k, renormalize=renormalize)
    h = expert_linear(x, gate_up, r.offsets, tokens=r.tokens, swiglu=True)
    rows = expert_linear(h, down, r.offsets)
    return combine_experts(rows, r.positions, r.weights, base=base, out=out)


def _expert_mlp(x, logits, gate_up, down, top_k, renormalize, base, out) -> bool:
    """The MLP of a few tokens in one call of the library; False where it does not take it."""
    import torch

    (count, hidden), (experts, _, inter) = x.shape, down.shape
    kind = (_lib.LF_EXPERT_MXFP4 if isinstance(down, MXFP4Tensor) else _lib.LF_EXPERT_FP8 if isinstance(down, FP8Tensor)
            else _lib.LF_EXPERT_BF16)
    lib = _lib.library()
    size = lib.lf_expert_mlp_workspace_size(count, experts, top_k, hidden, inter, kind)
    parts = _parts(gate_up), _parts(down)
    if size < 0 or any(t.data_ptr() % 4 for part in parts for t in part[1:]):
        return False
    if 1 < count <= 8 and x.stride(0) >= (2**30 - hidden) // (count - 1):
        x = x.contiguous()  # (the two launches take offsets of 31 bits)
    a = _lib.ExpertMlp()
    a.x, a.logits, a.y = x.data_ptr(), logits.data_ptr(), out.data_ptr()
    a.x_stride, a.logits_stride, a.y_stride = (t.stride(0) if count > 1 else t.shape[1] for t in (x, logits, out))
    a.fp32, a.renormalize, a.type = logits.dtype == torch.float32, renormalize, kind
    a.tokens, a.hidden, a.inter, a.experts, a.top = count, hidden, inter, experts, top_k
    a.gate_up, a.down = parts[0][0].data_ptr(), parts[1][0].data_ptr()
    if kind != _lib.LF_EXPERT_BF16:
        a.gate_up_scales, a.down_scales = parts[0][1].data_ptr(), parts[1][1].data_ptr()
    if base is not None:
        a.base, a.base_stride = base.data_ptr(), base.stride(0) if count > 1 else hidden
    scratch = torch.empty(size, dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(lib.lf_expert_mlp(ctypes.byref(a), scratch.data_ptr(), size, _lib.stream_of(x.device)))
    return True


def _parts(w):
    return (w.codes, w.scales) if isinstance(w, (MXFP4Tensor, FP8Tensor)) else (w,)


def _expert_weight(w, name, device):
    import torch

    if isinstance(w, FP8Tensor):
        scaled(w, name, 3, device, block_rows=BLOCK)
    elif isinstance(w, MXFP4Tensor):
        packed(w, name, 3, device)
    else:
        tensor(w, name, 3, torch.bfloat16, device)
        if not w.is_contiguous() or w.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous and 16-byte aligned")
        if w.shape[2] % 8:
            raise ValueError(f"{name}'s last dimension must be a multiple of 8")
    if 0 in tuple(w.shape):
        raise ValueError(f"{name} must not be empty")
