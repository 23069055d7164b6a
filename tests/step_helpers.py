"""Shared helpers of the attention-step tests: 16-bit values in numpy."""

from __future__ import annotations

import numpy as np

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # of a rounding, relative to the value
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}      # half the smallest subnormal


def to_half(x, dtype):
    """float array -> the uint16 patterns of the nearest fp16 / bf16 values (ties to even)."""
    x = np.asarray(x, np.float32)
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u >> 16) + ((u & 0xFFFF) + ((u >> 16) & 1) > 0x8000)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def to_float(u, dtype):
    """uint16 patterns -> float32."""
    u = np.ascontiguousarray(u, np.uint16)
    if dtype == "f16":
        return u.view(np.float16).astype(np.float32)
    return (u.astype(np.uint32) << 16).view(np.float32)


def normal(rng, shape, dtype, std=1.0):
    return to_half(rng.standard_normal(shape).astype(np.float32) * std, dtype)


NAN16 = np.uint16(0x7FFF)    # a NaN in either type


def scored_bound(q, kc, vc, bt, ctx, off, dtype, parts, want, **score):
    """How far an output may be from `want`, the oracle's in float64 (q, kc and
    vc as floats): half a step of the value for the one rounding, and for the
    weights, as shares of the weighted sum of |v|:
      - 32-bit products and sums: D + 8 roundings of scale |q| |k|, a few of the
        cap and of the bias, each moving a weight by its error in the exponent;
      - the exp2, the sum of the weights and of the products: (L + 8) roundings
        of 2^-24 at most, L / 16 of them where sums are tiled (taken whole);
      - weights in two 16-bit parts: 2^-20 of a weight in fp16, 2^-14 in
        bfloat16, or in one part, half a step; and fp16's subnormal weights,
        2^-32 of the row's largest for each key."""
    import oracle

    size = np.abs(vc)
    mean = oracle.scored_attention(q, kc, np.where(np.isfinite(size), size, 0), bt, ctx, off, **score)
    norms = np.sqrt(np.nansum(np.square(np.where(np.isfinite(kc), kc, 0), dtype=np.float64), axis=2)).max()
    D, L = q.shape[2], max(int(np.max(ctx, initial=1)), 1)
    top = abs(score["scale"]) * np.sqrt(np.square(q, dtype=np.float64).sum(axis=2, keepdims=True)) * norms
    exponent = (D + 8) * 2.0 ** -24 * top + 8 * 2.0 ** -24 * score.get("softcap", 0.0)
    if score.get("slopes") is not None:
        exponent = exponent + 4 * 2.0 ** -24 * L * np.abs(np.asarray(score["slopes"], np.float64))[None, :, None]
    share = 2 * exponent + (L + 8) * 2.0 ** -23 + L * 2.0 ** -31 + weights_share(dtype, parts)
    return HALF_STEP[dtype] * np.abs(want) + TINY[dtype] + share * mean


def weights_share(dtype, parts):
    """Relative error of a weight kept in `parts` 16-bit parts."""
    return {("f16", 2): 2.0 ** -20, ("bf16", 2): 2.0 ** -14}.get((dtype, parts), 2 * HALF_STEP[dtype])
