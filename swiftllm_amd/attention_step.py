"""One attention step around the paged cache, all of it on the device.

    plan_step           block tables, slot maps and positions from request lengths
    rotary_and_cache    rotary positions of q and k, and the cache write of k and v
    scored_decode       paged attention of one new token, its scores shaped: soft cap,
                        distance bias (ALiBi), sliding window, prefix
    scored_prefill      the same of packed prompts or chunks of them

Reference (paths relative to the swiftllm repository): the host routines and
options these stand for are
  crates/swiftllm-core/src/memory/block_manager.rs, kv_cache.rs:186-216
                                               block allocation, get_slot_mapping
  crates/swiftllm-models/src/layers/attention.rs:297-353
                                               RoPE and its long-context scaling
  crates/swiftllm-core/src/memory/paged_attention.rs:39-43, 111-135
                                               sliding window and ALiBi options
Device tensors are DeviceArrays or raw device pointers (ints); values are fp16
("f16") or bfloat16 ("bf16"). Nothing here synchronises or allocates, so every
call may be captured in a graph.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _lib
from ._hip import DeviceArray, Stream
from .paged_attention import (CudaError, InvalidParameter, NotSupported, Ptr, _p, _s,
                              check_status)

DTYPES = {"f16": 0, "bf16": 1}   # SWIFTLLM_HIP_F16, SWIFTLLM_HIP_BF16


def _dtype(name: str) -> int:
    if name not in DTYPES:
        raise NotSupported(f"dtype {name!r} (supported: {', '.join(DTYPES)})")
    return DTYPES[name]


# ---------------------------------------------------------------------------
# Plan
# ---------------------------------------------------------------------------
def plan_step(block_tables: Ptr, cached_lens: Ptr, new_lens: Ptr, free_blocks: Ptr,
              num_free: Ptr, free_capacity: int, num_seqs: int, max_num_blocks_per_seq: int,
              block_size: int, num_tokens: int, context_lens: Ptr, query_offsets: Ptr,
              positions: Ptr, slot_mapping: Ptr, counts: Ptr, num_blocks: int = 0,
              stream: Optional[Stream] = None) -> None:
    """Block tables and slot maps of one step from the requests' lengths
    (swiftllm_hip_plan_step): takes the missing blocks of every sequence from
    free_blocks in order, and writes context_lens [S], query_offsets [S + 1],
    positions and slot_mapping [num_tokens] (-1 behind the last token) and
    counts [3] = (blocks taken, tokens placed, sequences refused)."""
    check_status(_lib.lib().swiftllm_hip_plan_step(
        _p(block_tables), _p(cached_lens), _p(new_lens), _p(free_blocks), _p(num_free),
        free_capacity, num_seqs, max_num_blocks_per_seq, block_size, num_tokens, num_blocks,
        _p(context_lens), _p(query_offsets), _p(positions), _p(slot_mapping), _p(counts),
        _s(stream)))


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
def rotary_inv_freq(rotary_dim: int, base: float = 10000.0, scaling: str = "none",
                    factor: float = 1.0, original_context: int = 8192, beta_fast: float = 32.0,
                    beta_slow: float = 1.0, low_factor: float = 1.0,
                    high_factor: float = 4.0) -> tuple[np.ndarray, float]:
    """(inv_freq, attn_factor) of rotary_and_cache: the float64 radians per
    position of the rotary_dim / 2 pairs, and the factor of the rotated values.

    scaling, for contexts `factor` times the `original_context` trained on:
      "none"     base^(-2 i / rotary_dim)
      "linear"   positions interpolated: every frequency / factor
      "ntk"      a larger base, base * factor^(d / (d - 2)), d = rotary_dim: the
                 slowest pair is interpolated, the fastest stays
      "yarn"     by wavelength: pairs that turn more than beta_fast times in
                 the original context stay, those of less than beta_slow are
                 interpolated, a ramp over the pair's index between; values
                 times 0.1 ln(factor) + 1
      "banded"   pairs of more than high_factor turns stay, those of less than
                 low_factor are interpolated, a ramp in turns between
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise InvalidParameter(f"rotary_dim {rotary_dim} (even)")
    if not all(0 < x < math.inf for x in (base, factor, original_context)):
        raise InvalidParameter(f"base {base} factor {factor} original_context {original_context}")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    freq = float(base) ** (-2.0 * i / max(rotary_dim, 1))
    if scaling == "none":
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "ntk":
        if rotary_dim <= 2:
            return freq, 1.0
        wide = base * factor ** (rotary_dim / (rotary_dim - 2.0))
        return wide ** (-2.0 * i / rotary_dim), 1.0
    turns = original_context * freq / (2.0 * math.pi)
    if scaling == "yarn":
        if not math.inf > beta_fast > beta_slow > 0 or not base > 1:
            raise InvalidParameter(f"beta_fast {beta_fast} beta_slow {beta_slow} base {base} (above 1)")

        def pair_of(n: float) -> float:   # the (fractional) pair that turns n times
            return (rotary_dim * math.log(original_context / (2.0 * math.pi * n))
                    / (2.0 * math.log(base)))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        keep = 1.0 - np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        return freq / factor * (1.0 - keep) + freq * keep, 0.1 * math.log(max(factor, 1.0)) + 1.0
    if scaling == "banded":
        if not math.inf > high_factor > low_factor > -math.inf:
            raise InvalidParameter(f"low_factor {low_factor} high_factor {high_factor}")
        keep = np.clip((turns - low_factor) / (high_factor - low_factor), 0.0, 1.0)
        return freq / factor * (1.0 - keep) + freq * keep, 1.0
    raise NotSupported(f"rotary scaling {scaling!r}")


def rotary_and_cache(query_out: Ptr, query: Ptr, key: Ptr, value: Ptr, key_cache: Ptr,
                     value_cache: Ptr, positions: Ptr, slot_mapping: Ptr, inv_freq: Ptr,
                     num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int,
                     rotary_dim: int, block_size: int, dtype: str = "f16",
                     attn_factor: float = 1.0, interleaved: bool = False,
                     query_stride: Optional[int] = None, key_stride: Optional[int] = None,
                     value_stride: Optional[int] = None, num_blocks: int = 0,
                     stream: Optional[Stream] = None) -> None:
    """Rotates the queries into query_out and the keys into the cache, and
    writes the values there (swiftllm_hip_rotary_and_cache). Strides are
    elements between tokens, packed rows by default; inv_freq is float64
    [rotary_dim / 2] on the device (rotary_inv_freq). Tokens with a negative
    position are padding."""
    check_status(_lib.lib().swiftllm_hip_rotary_and_cache(
        _p(query_out), _p(query), _p(key), _p(value), _p(key_cache), _p(value_cache),
        _p(positions), _p(slot_mapping), _p(inv_freq), attn_factor, int(interleaved),
        _dtype(dtype), num_tokens, num_heads, num_kv_heads, head_dim, rotary_dim, block_size,
        num_heads * head_dim if query_stride is None else query_stride,
        num_kv_heads * head_dim if key_stride is None else key_stride,
        num_kv_heads * head_dim if value_stride is None else value_stride, num_blocks,
        _s(stream)))


# ---------------------------------------------------------------------------
# Attention with shaped scores
# ---------------------------------------------------------------------------
@dataclass
class ScoreParams:
    """How raw products become scores, and what a query at position p sees.

    score of key j = softcap * tanh(scale q.k / softcap), scale q.k where
    softcap is 0, minus alibi_slopes[h] * |p - j|; seen where j <= p and
    (window 0 or p - j < window), or j < prefix_lens[s]. alibi_slopes is
    float32 [num_heads], prefix_lens int32 [num_seqs], both on the device."""
    scale: float
    softcap: float = 0.0
    window: int = 0
    alibi_slopes: Ptr = None
    prefix_lens: Ptr = None


def alibi_slopes(num_heads: int) -> np.ndarray:
    """The usual slopes of a distance bias, float32 [num_heads]: the powers
    2^(-8 i / n), i = 1 .. n, for n heads a power of two; for other counts
    those of the next lower power of two, then every other one of twice as
    many."""
    if num_heads < 1:
        raise InvalidParameter(f"num_heads {num_heads}")
    n = 1 << (num_heads.bit_length() - 1)
    first = 2.0 ** (-8.0 * np.arange(1, n + 1) / n)
    more = 2.0 ** (-4.0 * np.arange(1, 2 * n, 2) / n)
    return np.concatenate([first, more])[:num_heads].astype(np.float32)


def scored_decode_workspace_size(num_seqs: int, num_heads: int, num_kv_heads: int, head_dim: int,
                                 block_size: int, max_num_blocks_per_seq: int) -> int:
    n = _lib.lib().swiftllm_hip_scored_decode_workspace_size(
        num_seqs, num_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq)
    if n == 0:
        check_status(_lib.lib().swiftllm_hip_last_error() or CudaError.code)
    return int(n)


def scored_decode(output: Ptr, workspace: Ptr, workspace_bytes: int, query: Ptr, key_cache: Ptr,
                  value_cache: Ptr, block_tables: Ptr, context_lens: Ptr, score: ScoreParams,
                  num_seqs: int, num_heads: int, num_kv_heads: int, head_dim: int,
                  block_size: int, max_num_blocks_per_seq: int, dtype: str = "f16",
                  num_blocks: int = 0, query_offsets: Ptr = None, num_tokens: int = 0,
                  stream: Optional[Stream] = None) -> None:
    """Paged attention of the last token of every sequence with shaped scores
    (swiftllm_hip_scored_decode): row s of query and output, or with
    query_offsets the last of the sequence's rows of num_tokens. `workspace` is
    plain scratch of scored_decode_workspace_size(...) bytes; calls that share
    one are ordered on one stream."""
    check_status(_lib.lib().swiftllm_hip_scored_decode(
        _p(output), _p(workspace), workspace_bytes, _p(query), _p(key_cache), _p(value_cache),
        _p(block_tables), _p(context_lens), _p(query_offsets), _p(score.alibi_slopes),
        _p(score.prefix_lens), score.scale, score.softcap, score.window, _dtype(dtype),
        num_tokens, num_seqs, num_heads, num_kv_heads, head_dim, block_size,
        max_num_blocks_per_seq, num_blocks, _s(stream)))


def scored_prefill(output: Ptr, query: Ptr, key_cache: Ptr, value_cache: Ptr, block_tables: Ptr,
                   context_lens: Ptr, query_offsets: Ptr, score: ScoreParams, num_tokens: int,
                   num_seqs: int, num_heads: int, num_kv_heads: int, head_dim: int,
                   block_size: int, max_num_blocks_per_seq: int, dtype: str = "f16",
                   num_blocks: int = 0, stream: Optional[Stream] = None) -> None:
    """Paged attention of packed query tokens with shaped scores
    (swiftllm_hip_scored_prefill): rows query_offsets[s] .. query_offsets[s + 1]
    - 1 are the last tokens of sequence s, whose keys are in the cache."""
    check_status(_lib.lib().swiftllm_hip_scored_prefill(
        _p(output), _p(query), _p(key_cache), _p(value_cache), _p(block_tables),
        _p(context_lens), _p(query_offsets), _p(score.alibi_slopes), _p(score.prefix_lens),
        score.scale, score.softcap, score.window, _dtype(dtype), num_tokens, num_seqs, num_heads,
        num_kv_heads, head_dim, block_size, max_num_blocks_per_seq, num_blocks, _s(stream)))


class AttentionStep:
    """A layer's share of a serving step: rotary positions and the cache write,
    then attention with shaped scores, over the arrays that plan() makes once
    per step for all layers. Calls are asynchronous on `stream`, and the arrays
    are the object's own, so a step of fixed capacities can be captured in a
    graph; steps that overlap take an object each.

        step = AttentionStep(num_seqs, num_tokens, max_blocks, H, Hkv, D, score, inv_freq)
        step.plan(tables, cached, new, free, num_free, free_capacity)   # once per step
        step.layer(q, k, v, key_cache, value_cache, out)                # every layer

    num_seqs and num_tokens are capacities: sequences past a batch have
    cached and new lengths of 0, rows past its tokens are left as they are.
    The rows of a step whose every sequence brings at most one token go through
    scored_decode (decode=True), all others through scored_prefill."""

    def __init__(self, num_seqs: int, num_tokens: int, max_num_blocks_per_seq: int,
                 num_heads: int, num_kv_heads: int, head_dim: int, score: ScoreParams,
                 inv_freq: np.ndarray, attn_factor: float = 1.0, interleaved: bool = False,
                 dtype: str = "f16", block_size: int = 16):
        _dtype(dtype)
        inv = np.ascontiguousarray(inv_freq, dtype=np.float64)
        if inv.ndim != 1 or 2 * inv.size > head_dim:
            raise InvalidParameter(f"inv_freq of shape {inv.shape} for head_dim {head_dim}")
        self.num_seqs, self.num_tokens = num_seqs, num_tokens
        self.max_num_blocks_per_seq, self.block_size = max_num_blocks_per_seq, block_size
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.score, self.dtype = score, dtype
        self.rotary_dim, self.attn_factor, self.interleaved = 2 * inv.size, attn_factor, interleaved
        self.inv_freq = DeviceArray.from_numpy(inv if inv.size else np.zeros(1))
        n = scored_decode_workspace_size(num_seqs, num_heads, num_kv_heads, head_dim, block_size,
                                         max_num_blocks_per_seq)
        self.workspace = DeviceArray((n,), np.uint8)
        self.context_lens = DeviceArray((max(num_seqs, 1),), np.int32)
        self.query_offsets = DeviceArray((num_seqs + 1,), np.int32)
        self.positions = DeviceArray((max(num_tokens, 1),), np.int32)
        self.slot_mapping = DeviceArray((max(num_tokens, 1),), np.int32)
        self.counts = DeviceArray((3,), np.int32)
        self.query = DeviceArray((max(num_tokens, 1), num_heads, head_dim), np.uint16)
        self._tables: Ptr = None

    def plan(self, block_tables: Ptr, cached_lens: Ptr, new_lens: Ptr, free_blocks: Ptr,
             num_free: Ptr, free_capacity: int, num_blocks: int = 0,
             stream: Optional[Stream] = None) -> None:
        """plan_step into this object's arrays; block_tables is completed in place."""
        plan_step(block_tables, cached_lens, new_lens, free_blocks, num_free, free_capacity,
                  self.num_seqs, self.max_num_blocks_per_seq, self.block_size, self.num_tokens,
                  self.context_lens, self.query_offsets, self.positions, self.slot_mapping,
                  self.counts, num_blocks=num_blocks, stream=stream)
        self._tables = block_tables

    def layer(self, query: Ptr, key: Ptr, value: Ptr, key_cache: Ptr, value_cache: Ptr,
              output: Ptr, query_stride: Optional[int] = None, key_stride: Optional[int] = None,
              value_stride: Optional[int] = None, num_blocks: int = 0, decode: bool = False,
              stream: Optional[Stream] = None) -> None:
        """Rotates the step's queries and keys, writes keys and values to this
        layer's cache and attends over it. query, key and value hold num_tokens
        rows; output is [num_tokens, num_heads, head_dim]. decode: the caller
        knows that no sequence brings more than one token (of more, only the
        last would be attended)."""
        if self._tables is None:
            raise InvalidParameter("layer() before plan()")
        H, Hkv, D = self.num_heads, self.num_kv_heads, self.head_dim
        rotary_and_cache(self.query, query, key, value, key_cache, value_cache, self.positions,
                         self.slot_mapping, self.inv_freq, self.num_tokens, H, Hkv, D,
                         self.rotary_dim, self.block_size, dtype=self.dtype,
                         attn_factor=self.attn_factor, interleaved=self.interleaved,
                         query_stride=query_stride, key_stride=key_stride,
                         value_stride=value_stride, num_blocks=num_blocks, stream=stream)
        if decode:
            scored_decode(output, self.workspace, self.workspace.nbytes, self.query, key_cache,
                          value_cache, self._tables, self.context_lens, self.score, self.num_seqs,
                          H, Hkv, D, self.block_size, self.max_num_blocks_per_seq,
                          dtype=self.dtype, num_blocks=num_blocks,
                          query_offsets=self.query_offsets, num_tokens=self.num_tokens,
                          stream=stream)
        else:
            scored_prefill(output, self.query, key_cache, value_cache, self._tables,
                           self.context_lens, self.query_offsets, self.score, self.num_tokens,
                           self.num_seqs, H, Hkv, D, self.block_size,
                           self.max_num_blocks_per_seq, dtype=self.dtype, num_blocks=num_blocks,
                           stream=stream)
