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
