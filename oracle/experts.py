"""MXFP4 and mixture-of-experts operators in numpy, 64 bits. TEST INFRASTRUCTURE ONLY.

The reference has neither: the definitions are those of the OCP microscaling
format (MXFP4: blocks of 32 e2m1 codes, e8m0 scales) and of top-k routing over a
softmax, restated here without the product's code. ``tests/test_oracle_experts.py``
checks them against closed forms and brute force.
"""

from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def quantize(x):
    """Codes (uint8, two a byte, even index low) and scale bytes of fp64-representable ``x`` ``[..., K]``."""
    x = np.asarray(x, dtype=np.float64)
    blocks = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = np.abs(blocks).max(-1)
    finite = np.isfinite(top)
    safe = np.where(finite & (top > 0), top, 1.0)
    exponent = np.floor(np.log2(safe)).astype(np.int64)
    exponent -= (np.ldexp(1.0, exponent) > safe).astype(np.int64)  # log2 may round up below a power of two
    scale = np.maximum(exponent - 2 + 127, 0)
    scale = np.where(finite, np.where(top > 0, scale, 0), 255)
    a = np.abs(np.where(finite[..., None], blocks, 0.0)) / np.ldexp(1.0, np.where(finite, scale, 127) - 127)[..., None]
    distance = np.abs(a[..., None] - LEVELS)
    best = distance == distance.min(-1, keepdims=True)
    order = np.arange(8) % 2 * 8 + np.arange(8)  # of two equally near codes the even one
    code = np.where(best, order, 99).min(-1) % 8
    code = np.where(finite[..., None], code + 8 * np.signbit(blocks), 0).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.astype(np.uint8)


def values(codes, scales):
    """fp64 values of packed codes (NaN for scale 255)."""
    codes = np.asarray(codes)
    nibbles = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)
    v = LEVELS[nibbles & 7] * np.where(nibbles >> 3, -1.0, 1.0)
    scale = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(scale, BLOCK, axis=-1)


def product(x, w, bias=None, swiglu=False):
    """``(y, bound)``: ``x @ w.T (+ bias)`` in fp64, and how far fp32 sums of it may be off.

    The bound: each of the K products and sums may lose 2^-24 of the sum of
    magnitudes, twice for matrix instructions that round inside a step. Through
    silu (slope at most 1.1) and the product with up it grows as they do; the
    activation itself is within 2^-21.
    """
    k = x.shape[-1]
    y = x @ w.T
    bound = (2.0 * k + 16.0) * 2.0**-24 * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias
        bound = bound + 2.0**-23 * (np.abs(y) + np.abs(bias))
    if swiglu:
        half = w.shape[0] // 2
        g, u, dg, du = y[:, :half], y[:, half:], bound[:, :half], bound[:, half:]
        act = g / (1.0 + np.exp(-g))
        y = act * u
        bound = 1.1 * dg * (np.abs(u) + du) + (np.abs(act) + 1.1 * dg) * du + 2.0**-21 * np.abs(y)
    return y, bound


def route(logits, top, renormalize=True):
    """weights, experts, offsets, tokens, positions of fp64 ``logits`` ``[T, E]`` by brute force."""
    tokens, count = logits.shape
    weights = np.zeros((tokens, top))
    experts = np.full((tokens, top), -1, np.int32)
    for t in range(tokens):
        row = logits[t]
        allowed = [e for e in range(count) if row[e] > -np.inf]
        chosen = sorted(allowed, key=lambda e: (-row[e], e))[:top]
        experts[t, : len(chosen)] = chosen
        if not chosen:
            continue
        if np.isnan(row).any() or np.isposinf(row).any():
            weights[t, : len(chosen)] = np.nan
            continue
        p = np.exp(row[chosen] - row[chosen[0]])
        weights[t, : len(chosen)] = p / (p.sum() if renormalize else np.exp(row[allowed] - row[chosen[0]]).sum())
    offsets, order = [0], []
    flat = experts.reshape(-1)
    for e in range(count):
        order += [i for i in range(flat.size) if flat[i] == e]
        offsets.append(len(order))
    positions = np.full(flat.size, -1, np.int32)
    positions[order] = np.arange(len(order))
    token = np.full(flat.size, -1, np.int32)
    token[: len(order)] = np.array(order, dtype=np.int64) // top
    return weights, experts, np.array(offsets, np.int32), token, positions.reshape(tokens, top)
