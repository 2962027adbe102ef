"""Timed cases of the MXFP4 and mixture-of-experts operators.

A case is one pass through one operator as a serving program calls it: MXFP4
quantisation and back, the dense MXFP4 linear, expert routing, the product
grouped by expert, and the weighted sum of the experts' rows. ``run`` computes
it in elementary fp32 torch operations where ``own`` is false and with
``loraforge_amd.ops`` where it is true.

Weights are ``N(0, 0.02)``, activations ``N(0, 1)`` with one channel in 64 eight
times as large, router logits ``N(0, 1.5)`` around a popularity ``N(0, 0.5)`` of
each expert, so that the experts' shares are ragged and some are empty.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------


def _quant(m, k, what):
    return dict(kind="quant", m=m, k=k, what=what)


def _linear(m, n, k, act, *, swiglu=False, bias=False):
    return dict(kind="linear", m=m, n=n, k=k, act=act, swiglu=swiglu, bias=bias)


def _route(tokens, experts, top, dtype, *, renormalize=True, masked=False):
    return dict(kind="route", tokens=tokens, experts=experts, top=top, dtype=dtype, renormalize=renormalize, masked=masked)


def _experts(tokens, experts, top, n, k, act, weight, *, swiglu=False, bias=False, gather=True):
    return dict(kind="experts", tokens=tokens, experts=experts, top=top, n=n, k=k, act=act, weight=weight, swiglu=swiglu,
                bias=bias, gather=gather)


def _combine(tokens, top, n, *, base=False, masked=False):
    return dict(kind="combine", tokens=tokens, top=top, n=n, base=base, masked=masked)


def listed():
    return [
        # The smallest call: the activations of a decode batch of odd size, to MXFP4 and back.
        dict(_quant(7, 4096, "act"), name="quant_7"),
        # A whole merged gate/up weight as it is prepared for serving.
        dict(_quant(24576, 4096, "weight"), name="quant_gate_up"),
        # One user's token through a square projection.
        dict(_linear(1, 4096, 4096, "bf16"), name="linear_1"),
        # A short prompt chunk through a merged gate/up projection, activations kept in bf16.
        dict(_linear(300, 24576, 4096, "bf16", swiglu=True), name="linear_swiglu_300"),
        # A prefill batch through an up projection with both operands in MXFP4.
        dict(_linear(4096, 12288, 4096, "mxfp4", bias=True), name="linear_mxfp4_4096"),
        # The router of one decode step, and of a long ragged prefill batch.
        dict(_route(16, 128, 8, "fp32"), name="route_16"),
        dict(_route(8191, 128, 8, "bf16"), name="route_8191"),
        # A decode batch through the merged gate/up of its experts: every expert has a few rows or none.
        dict(_experts(24, 64, 4, 4096, 4096, "bf16", "mxfp4", swiglu=True), name="experts_24"),
        # Prefill through unquantised down projections, rows already in expert order, ragged.
        dict(_experts(2047, 32, 4, 4096, 2048, "bf16", "bf16", gather=False), name="experts_bf16_2047"),
        # The largest: a prefill batch through the experts' merged gate/up with both operands in MXFP4.
        dict(_experts(8192, 64, 4, 4096, 4096, "mxfp4", "mxfp4", swiglu=True), name="experts_mxfp4_8192"),
        # The experts' rows back to tokens: a decode batch onto the shared expert's output, and a prefill batch.
        dict(_combine(24, 4, 4096, base=True), name="combine_24"),
        dict(_combine(8191, 8, 4096), name="combine_8191"),
    ]


def _between(rng, lo, hi):
    """An integer spread over the logarithm of its range, both ends included."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _width(rng, lo, hi, unit):
    """A width in units of ``unit``; half of the time in units of 256, as most projections are (3072 is none of them here)."""
    if rng.random() < 0.5:
        unit = 256
    width = max(unit, round(_between(rng, lo, hi) / unit) * unit)
    return width + unit if width == 3072 else width


def draw(rng):
    kind = rng.choice(("quant", "linear", "linear", "linear", "route", "experts", "experts", "experts", "combine"))
    if kind == "quant":
        k = _width(rng, 512, 12288, BLOCK)
        return _quant(_between(rng, 1, 24576 * 4096 // k), k, rng.choice(("act", "weight")))
    if kind == "route":
        experts = rng.choice((8, 16, 60, 64, 128, 256))
        return _route(_between(rng, 1, 16384), experts, rng.randint(1, min(8, experts)), rng.choice(("fp32", "bf16")),
                      renormalize=rng.random() < 0.7, masked=rng.random() < 0.3)
    if kind == "combine":
        top = rng.randint(1, 8)
        return _combine(_between(rng, 1, 8191), top, _width(rng, 512, 4096, 8), base=rng.random() < 0.5, masked=rng.random() < 0.3)
    swiglu, bias = rng.random() < 0.4, rng.random() < 0.3
    n, k = _width(rng, 512, 16384, 24), _width(rng, 512, 12288, BLOCK)
    if kind == "linear":
        m = min(_between(rng, 1, 8192), 4096 * 12288 * 4096 // (n * k))
        return _linear(m, n, k, rng.choice(("bf16", "mxfp4")), swiglu=swiglu, bias=bias)
    act, weight = rng.choice((("bf16", "mxfp4"), ("bf16", "bf16"), ("mxfp4", "mxfp4")))
    experts = rng.choice((8, 32, 60, 64, 128))
    top = rng.randint(1, min(8, experts))
    n = min(n, 8192)
    # No more weight bytes than the largest listed case, and no more operations at the operands' rate.
    k = min(k, 8192, max(512, (2**28 if weight == "bf16" else 2**30) // (experts * n) // 256 * 256))
    if k == 3072:
        k -= 256
    most = 8192 * 4 * 4096 * 4096 // (1 if act == "mxfp4" else 4)
    tokens = min(_between(rng, 1, 8192), max(1, most // (n * k * top)))
    return _experts(tokens, experts, top, n, k, act, weight, swiglu=swiglu, bias=bias, gather=rng.random() < 0.7)


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------


def _dev():
    return torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _activations(g, m, k):
    x = torch.randn(m, k, generator=g, device=_dev())
    x[:, ::64] *= 8.0
    return x.bfloat16()


def _weights(g, *shape):
    return (torch.randn(*shape, generator=g, device=_dev()) * 0.02).bfloat16()


def _logits(g, tokens, experts, masked):
    logits = torch.randn(tokens, experts, generator=g, device=_dev()) * 1.5
    logits += torch.randn(experts, generator=g, device=_dev()) * 0.5
    if masked:  # three experts in four not allowed; now and then none is
        logits[torch.rand(tokens, experts, generator=g, device=_dev()) < 0.75] = -math.inf
    return logits


def _quantize(x):
    """Packed codes and scale bytes of ``x`` (``[..., K]``) by the format's rule, for inputs held in MXFP4."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    exponent = torch.frexp(b.abs().amax(-1)).exponent - 3  # floor(log2 max) - 2
    exponent = exponent.clamp(-127, 127)
    a = torch.ldexp(b.abs(), -exponent.unsqueeze(-1))
    code = (a > 0.25).to(torch.uint8)
    for bound, tie_up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= bound) if tie_up else (a > bound)
    code += torch.signbit(b) * torch.tensor(8, dtype=torch.uint8, device=x.device)
    code = code.flatten(-2)
    scales = torch.where(b.abs().amax(-1) == 0, 0, exponent + 127).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def _packed_weights(g, *shape):
    """A random weight in MXFP4, made in slices of its first axis."""
    parts = [_quantize(_weights(g, *shape[1:])) for _ in range(shape[0])] if len(shape) == 3 else [
        _quantize(part) for part in _weights(g, *shape).split(4096)]
    join = torch.stack if len(shape) == 3 else torch.cat
    return join([p[0] for p in parts]), join([p[1] for p in parts])


def _order(experts, count):
    """Expert order of the flat choices: offsets, token of each position, position of each choice."""
    tokens, top = experts.shape
    flat = experts.reshape(-1).long()
    live = flat >= 0
    order = torch.argsort(torch.where(live, flat, count), stable=True)
    counts = (flat.unsqueeze(0) == torch.arange(count, device=flat.device).unsqueeze(1)).sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    total = offsets[-1]
    rank = torch.arange(flat.numel(), device=flat.device)
    token = torch.where(rank < total, order // top, -1)
    positions = torch.empty_like(flat)
    positions[order] = torch.where(rank < total, rank, -1)
    return offsets.int(), token.int(), positions.reshape(tokens, top).int()


def _inputs(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    kind = case["kind"]
    if kind == "quant":
        s["x"] = _activations(g, case["m"], case["k"]) if case["what"] == "act" else _weights(g, case["m"], case["k"])
    elif kind == "linear":
        s["x"] = _activations(g, case["m"], case["k"])
        s["w"] = _packed_weights(g, case["n"], case["k"])
        s["bias"] = (torch.randn(case["n"], generator=g, device=_dev()) * 0.5).bfloat16() if case["bias"] else None
    elif kind == "route":
        logits = _logits(g, case["tokens"], case["experts"], case["masked"])
        s["logits"] = logits.bfloat16() if case["dtype"] == "bf16" else logits
    elif kind == "experts":
        tokens, count, n, k = case["tokens"], case["experts"], case["n"], case["k"]
        chosen = _logits(g, tokens, count, False).topk(case["top"], dim=1).indices
        s["offsets"], s["tokens"], _ = _order(chosen, count)
        s["bounds"] = s["offsets"].tolist()
        rows = tokens if case["gather"] else tokens * case["top"]
        s["x"] = _activations(g, rows, k)
        s["w"] = _packed_weights(g, count, n, k) if case["weight"] == "mxfp4" else _weights(g, count, n, k)
        s["bias"] = (torch.randn(count, n, generator=g, device=_dev()) * 0.5).bfloat16() if case["bias"] else None
    else:
        tokens, top, n = case["tokens"], case["top"], case["n"]
        count = max(8, top)
        logits = _logits(g, tokens, count, case["masked"])
        value, chosen = logits.topk(top, dim=1)
        chosen = torch.where(value > -math.inf, chosen, -1)
        _, _, s["positions"] = _order(chosen, count)
        weights = torch.where(chosen >= 0, torch.exp(value - value[:, :1]), 0.0)
        s["weights"] = weights / weights.sum(1, keepdim=True).clamp_min(1e-20)
        s["rows"] = torch.randn(tokens * top, n, generator=g, device=_dev()).bfloat16()
        s["base"] = torch.randn(tokens, n, generator=g, device=_dev()).bfloat16() if case["base"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] in ("linear", "experts") and isinstance(s["w"], tuple):
        from loraforge_amd.ops import MXFP4Tensor

        s["w"] = MXFP4Tensor(*s["w"])
    return s


# --------------------------------------------------------------------------
# The pass
# --------------------------------------------------------------------------


def _values(codes, scales):
    """The fp32 values of packed codes with their scale bytes."""
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    levels = torch.cat([levels, -levels])
    v = levels[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    scale = torch.exp2(scales.float() - 127.0)
    return (v.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def _product(x, w, bias, swiglu):
    y = x @ w.t()
    if bias is not None:
        y = y + bias.float()
    if swiglu:
        g, u = y.chunk(2, dim=1)
        y = g / (1.0 + torch.exp(-g)) * u
    return y.bfloat16()


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "quant":
        return _values(*_quantize(s["x"])).bfloat16()
    if kind == "route":
        logits = s["logits"].float()
        top = case["top"]
        value, order = torch.sort(logits, dim=1, descending=True, stable=True)
        value, chosen = value[:, :top], order[:, :top]
        live = value > -math.inf
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        p = torch.where(live, e.gather(1, chosen), 0.0)
        total = p.sum(1, keepdim=True) if case["renormalize"] else e.sum(1, keepdim=True)
        weights = torch.where(live, p / total, 0.0)
        experts = torch.where(live, chosen, -1)
        return (weights, experts.int(), *_order(experts, case["experts"]))
    if kind == "combine":
        positions = s["positions"].long()
        y = torch.zeros(case["tokens"], case["n"], device=positions.device) if s["base"] is None else s["base"].float()
        for j in range(case["top"]):
            p = positions[:, j]
            row = s["rows"][p.clamp_min(0)].float() * s["weights"][:, j : j + 1]
            y = y + torch.where(p.unsqueeze(1) >= 0, row, 0.0)
        return y.bfloat16()
    x = _values(*_quantize(s["x"])) if case["act"] == "mxfp4" else s["x"].float()
    if kind == "linear":
        return _product(x, _values(*s["w"]), s["bias"], case["swiglu"])
    if case["gather"]:
        x = x[s["tokens"].long()]
    parts = []
    for e in range(case["experts"]):
        lo, hi = s["bounds"][e], s["bounds"][e + 1]
        if lo < hi:
            w = _values(s["w"][0][e], s["w"][1][e]) if case["weight"] == "mxfp4" else s["w"][e].float()
            parts.append(_product(x[lo:hi], w, None if s["bias"] is None else s["bias"][e], case["swiglu"]))
    return torch.cat(parts)


def run(s):
    if not own:
        return _plain(s)
    from loraforge_amd import ops

    case = s["case"]
    kind = case["kind"]
    if kind == "quant":
        return ops.dequantize_mxfp4(ops.quantize_mxfp4(s["x"]))
    if kind == "route":
        r = ops.route_experts(s["logits"], case["top"], renormalize=case["renormalize"])
        return r.weights, r.experts, r.offsets, r.tokens, r.positions
    if kind == "combine":
        return ops.combine_experts(s["rows"], s["positions"], s["weights"], base=s["base"])
    x = ops.quantize_mxfp4(s["x"]) if case["act"] == "mxfp4" else s["x"]
    if kind == "linear":
        return ops.mxfp4_linear(x, s["w"], bias=s["bias"], swiglu=case["swiglu"])
    return ops.expert_linear(x, s["w"], s["offsets"], tokens=s["tokens"] if case["gather"] else None, bias=s["bias"],
                             swiglu=case["swiglu"])


# --------------------------------------------------------------------------
# Work, and the values in 64 bits
# --------------------------------------------------------------------------


def _packed_bytes(count):
    return count // 2 + count // BLOCK


def work(case):
    kind = case["kind"]
    if kind == "quant":  # the input and the values, both bf16
        return {"bytes": 4 * case["m"] * case["k"], "flops": 0}
    if kind == "route":
        tokens, top = case["tokens"], case["top"]
        logit = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": logit * tokens * case["experts"] + 16 * tokens * top + 4 * (case["experts"] + 1), "flops": 0}
    if kind == "combine":
        tokens, top, n = case["tokens"], case["top"], case["n"]
        live = tokens * top
        if case["masked"]:  # the expected number of choices left of a quarter of the experts
            count = max(8, top)
            live = tokens * sum(min(i, top) * math.comb(count, i) * 0.25**i * 0.75 ** (count - i) for i in range(count + 1))
        return {"bytes": int(2 * live * n + 2 * tokens * n * (2 if case["base"] else 1) + 8 * tokens * top), "flops": int(2 * live * n)}
    n, k = case["n"], case["k"]
    width = n // 2 if case["swiglu"] else n
    if kind == "linear":
        m = case["m"]
        return {"bytes": _packed_bytes(n * k) + 2 * m * k + 2 * m * width + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    tokens, count, top = case["tokens"], case["experts"], case["top"]
    rows = tokens * top
    used = count * (1 - (1 - top / count) ** tokens)  # experts with a row, if all were equally popular
    weight = _packed_bytes(n * k) if case["weight"] == "mxfp4" else 2 * n * k
    read = 2 * (tokens if case["gather"] else rows) * k
    return {"bytes": int(used * weight) + read + 2 * rows * width + 4 * (rows if case["gather"] else 0), "flops": 2 * rows * n * k}


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(x):
    """The fp64 values that the format gives ``x``: the nearest level, of two equally near the one of even code."""
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=x.device)
    odd = torch.arange(8, device=x.device) % 2
    out = []
    for rows in x.split(max(1, 2**24 // x.shape[1])):
        b = rows.double().reshape(rows.shape[0], -1, BLOCK)
        top = b.abs().amax(2, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2).clamp(2.0**-127, 2.0**127)
        distance = (b.abs().div(scale).unsqueeze(3) - levels).abs()
        best = distance.amin(3, keepdim=True)
        code = torch.where(distance == best, odd * 8 + torch.arange(8, device=x.device), 99).amin(3) % 8
        out.append((levels[code] * torch.where(b < 0, -scale, scale)).reshape(rows.shape))
    return torch.cat(out)


def _unpacked(codes, scales):
    """fp64 values of one packed matrix."""
    k = codes.shape[1] * 2
    v = torch.empty(codes.shape[0], k, dtype=torch.float64, device=codes.device)
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=codes.device)
    for i, nibble in enumerate((codes % 16, codes // 16)):
        nibble = nibble.long()
        v[:, i::2] = levels[nibble % 8] * (1 - 2 * (nibble // 8))
    return v * torch.pow(2.0, scales.double() - 127).repeat_interleave(BLOCK, 1)


def _affine(x, w, bias, swiglu):
    y = torch.cat([x @ part.t() for part in w.split(4096)], 1)
    if bias is not None:
        y += bias.double()
    if not swiglu:
        return y
    half = y.shape[1] // 2
    return y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]


def _route_exact(s):
    case = s["case"]
    logits = s["logits"].double()
    tokens, count = logits.shape
    left = logits.clone()
    p = torch.softmax(torch.where(torch.isinf(logits), -1e300, logits), 1)
    columns = torch.arange(count, device=logits.device)
    experts, weights = [], []
    for _ in range(case["top"]):
        best = left.amax(1, keepdim=True)
        first = torch.where(left == best, columns, count).amin(1, keepdim=True)
        live = best > -math.inf
        experts.append(torch.where(live, first, -1))
        weights.append(torch.where(live, p.gather(1, first), 0.0))
        left.scatter_(1, first, -math.inf)
    experts, weights = torch.cat(experts, 1), torch.cat(weights, 1)
    if case["renormalize"]:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
    flat = experts.reshape(-1).cpu().tolist()
    segments = [[] for _ in range(count)]
    for i, e in enumerate(flat):
        if e >= 0:
            segments[e].append(i)
    offsets, order = [0], []
    for segment in segments:
        order += segment
        offsets.append(len(order))
    token = [i // case["top"] for i in order] + [-1] * (len(flat) - len(order))
    positions = [-1] * len(flat)
    for place, i in enumerate(order):
        positions[i] = place
    as_int = dict(dtype=torch.int32, device=logits.device)
    return (weights, experts.int(), torch.tensor(offsets, **as_int), torch.tensor(token, **as_int),
            torch.tensor(positions, **as_int).reshape(tokens, -1))


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _nearest(s["x"])
    if kind == "route":
        return _route_exact(s)
    if kind == "combine":
        rows, positions, weights = s["rows"], s["positions"].long(), s["weights"].double()
        y = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=rows.device)
        if s["base"] is not None:
            y += s["base"].double()
        for j in range(case["top"]):
            t = torch.nonzero(positions[:, j] >= 0).squeeze(1)
            y[t] += weights[t, j : j + 1] * rows[positions[t, j]].double()
        return y
    x = _nearest(s["x"]) if case["act"] == "mxfp4" else s["x"].double()
    if kind == "linear":
        return _affine(x, _unpacked(*s["w"]), s["bias"], case["swiglu"])
    source = s["tokens"].long() if case["gather"] else torch.arange(case["tokens"] * case["top"], device=x.device)
    parts = []
    for e in range(case["experts"]):
        rows = source[s["bounds"][e] : s["bounds"][e + 1]]
        if rows.numel():
            w = _unpacked(s["w"][0][e], s["w"][1][e]) if case["weight"] == "mxfp4" else s["w"][e].double()
            parts.append(_affine(x[rows], w, None if s["bias"] is None else s["bias"][e], case["swiglu"]))
    return torch.cat(parts)
