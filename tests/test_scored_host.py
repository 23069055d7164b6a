"""The scored attention's entry points without a GPU: argument checks and the
distance bias's slopes."""

import math

import numpy as np
import pytest

import oracle
from swiftllm_amd import _lib
from swiftllm_amd import attention_step as step
from swiftllm_amd import paged_attention as pa

INVALID, UNSUP = -4, -6
P = 1 << 20   # never dereferenced: validation fails first


def _decode(**kw):
    a = dict(output=P, workspace=P, workspace_bytes=1 << 40, query=P, key_cache=P, value_cache=P,
             block_tables=P, context_lens=P, query_offsets=0, alibi_slopes=0, prefix_lens=0, scale=0.1,
             softcap=0.0, window=0, dtype=0, num_tokens=-1, num_seqs=3, num_heads=8, num_kv_heads=2, head_dim=64, block_size=16,
             max_num_blocks_per_seq=4, num_blocks=0)
    a.update(kw)
    return _lib.lib().swiftllm_hip_scored_decode(*a.values(), None)


SHARED = [
    (dict(num_seqs=-1), INVALID),
    (dict(num_heads=0), INVALID),
    (dict(num_heads=9), INVALID),
    (dict(head_dim=96), UNSUP),
    (dict(head_dim=0), INVALID),
    (dict(block_size=32), UNSUP),
    (dict(max_num_blocks_per_seq=-1), INVALID),
    (dict(max_num_blocks_per_seq=1 << 27), UNSUP),
    (dict(num_seqs=65536), UNSUP),
    (dict(num_seqs=65535, max_num_blocks_per_seq=1 << 20), UNSUP),
    (dict(dtype=2), UNSUP),
    (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID),
    (dict(softcap=-1.0), INVALID),
    (dict(softcap=math.nan), INVALID),
    (dict(softcap=math.inf), INVALID),
    (dict(softcap=1e-30, scale=1e30), INVALID),     # scale / softcap is no finite number
    (dict(window=-1), INVALID),
    (dict(query=0), INVALID),
    (dict(context_lens=0), INVALID),
    (dict(block_tables=0), INVALID),
    (dict(query=P + 4), INVALID),
    (dict(key_cache=P + 2), INVALID),
    (dict(output=P + 1), INVALID),
    (dict(alibi_slopes=P + 2), INVALID),
    (dict(prefix_lens=P + 2), INVALID),
]


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(workspace=P + 128), INVALID),
    (dict(workspace=0), INVALID),
    (dict(workspace_bytes=1000), INVALID),
    (dict(query_offsets=P), INVALID),               # and num_tokens below 0
    (dict(query_offsets=P + 2, num_tokens=5), INVALID),
])
def test_decode_refuses(kw, code):
    assert _decode(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


def _prefill(**kw):
    a = dict(output=P, query=P, key_cache=P, value_cache=P, block_tables=P, context_lens=P,
             query_offsets=P, alibi_slopes=0, prefix_lens=0, scale=0.1, softcap=0.0, window=0,
             dtype=0, num_tokens=10, num_seqs=3, num_heads=8, num_kv_heads=2, head_dim=64,
             block_size=16, max_num_blocks_per_seq=4, num_blocks=0)
    a.update(kw)
    return _lib.lib().swiftllm_hip_scored_prefill(*a.values(), None)


@pytest.mark.parametrize("kw,code", [c for c in SHARED if c[0].get("max_num_blocks_per_seq") != 1 << 20] + [
    (dict(num_tokens=-1), INVALID),
    (dict(num_tokens=1 << 30), UNSUP),
    (dict(max_num_blocks_per_seq=1 << 26), UNSUP),
    (dict(query_offsets=0), INVALID),
    (dict(query_offsets=P + 1), INVALID),
    (dict(key_cache=P + 8), INVALID),
    (dict(value_cache=P + 8), INVALID),
    (dict(output=P + 4), INVALID),
    (dict(num_tokens=(1 << 30) - 1, num_heads=1024, num_kv_heads=1024), UNSUP),
])
def test_prefill_refuses(kw, code):
    assert _prefill(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_a_cap_has_an_upper_bound(call):
    """The capped score is off by 2^-24 of its cap."""
    assert call(softcap=1024.5) == UNSUP
    assert "at most 1024" in _lib.last_error()[1]


def test_outputs_that_overlap_are_refused():
    far = 1 << 40   # of the other arguments
    for d in (-64, 64, 3 * 8 * 64 * 2 - 16):        # of 3 rows of 8 heads x 64 values
        assert _decode(workspace=far, output=P + d) == INVALID
        assert "overlaps" in _lib.last_error()[1]
    assert _decode(workspace=far, output=P + 64, query_offsets=P, num_tokens=1) == INVALID
    assert _decode(output=far) == INVALID            # workspace on the queries
    assert _decode(query=far) == INVALID             # and on the output
    for d in (-64, 64, 10 * 8 * 64 * 2 - 16):
        assert _prefill(output=P + d) == INVALID
        assert "overlaps" in _lib.last_error()[1]


def test_decode_workspace_size():
    n = step.scored_decode_workspace_size(8, 64, 8, 128, 16, 2048)
    # two fragments of 16-byte aligned heads for each of the ranges
    assert 512 * 2 * 8 * (128 + 2) * 4 <= n < 64 << 20
    with pytest.raises(pa.NotSupported):
        step.scored_decode_workspace_size(8, 64, 8, 96, 16, 2048)
    with pytest.raises(pa.InvalidParameter):
        step.scored_decode_workspace_size(8, 9, 8, 64, 16, 2048)


def test_alibi_slopes():
    assert step.alibi_slopes(8).tolist() == [2.0 ** -i for i in range(1, 9)]
    s = step.alibi_slopes(12)
    assert s[:8].tolist() == step.alibi_slopes(8).tolist()
    assert np.allclose(s[8:], [2.0 ** -(i / 2) for i in (1, 3, 5, 7)], rtol=1e-7)
    assert step.alibi_slopes(1).tolist() == [2.0 ** -8]
    for n in (1, 3, 16, 40, 64):
        assert step.alibi_slopes(n).shape == (n,) and step.alibi_slopes(n).dtype == np.float32
    with pytest.raises(pa.InvalidParameter):
        step.alibi_slopes(0)


def test_oracle_without_shaping_is_plain_attention():
    """The shaped oracle at cap 0, no bias and no window gives the decode and
    prefill oracles' values."""
    rng = np.random.default_rng(1)
    kc, vc = rng.standard_normal((2, 9, 2, 64, 16)).astype(np.float16)
    bt = rng.permutation(9)[:8].reshape(2, 4).astype(np.int32)
    q = rng.standard_normal((2, 8, 64)).astype(np.float16)
    ctx = np.array([50, 17], np.int32)
    got = oracle.scored_attention(q, kc, vc, bt, ctx, [0, 1, 2], 0.125)
    assert np.allclose(got, oracle.decode_numpy(q, kc, vc, bt, ctx, 0.125), rtol=1e-12, atol=1e-14)
    qp = rng.standard_normal((67, 8, 64)).astype(np.float16)
    slots = np.concatenate([pa.get_slot_mapping(bt[0], 16, 0, 50), pa.get_slot_mapping(bt[1], 16, 0, 17)])
    got = oracle.scored_attention(qp, kc, vc, bt, ctx, [0, 50, 67], 0.125)
    assert np.allclose(got, oracle.prefill_numpy(qp, kc, vc, slots, ctx, 0.125), rtol=1e-12, atol=1e-14)


_SIZES = dict(num_seqs=3, num_heads=8, num_kv_heads=2, head_dim=64, max_num_blocks_per_seq=4, num_blocks=5)


@pytest.mark.parametrize("name,nbytes", [
    ("key_cache", 5 * 2 * 64 * 16 * 2), ("value_cache", 5 * 2 * 64 * 16 * 2), ("block_tables", 3 * 4 * 4),
    ("context_lens", 3 * 4), ("query_offsets", 4 * 4), ("alibi_slopes", 8 * 4), ("prefix_lens", 3 * 4)])
def test_outputs_on_any_other_argument_are_refused(name, nbytes):
    """The output, and the decode's workspace, from the argument's first byte to its last."""
    M = 1 << 32
    names = ["query", "key_cache", "value_cache", "block_tables", "context_lens", "query_offsets", "alibi_slopes",
             "prefix_lens"]
    at = {n: (i + 2) * M for i, n in enumerate(names)}
    ws = step.scored_decode_workspace_size(3, 8, 2, 64, 16, 4)
    out = 10 * 8 * 64 * 2
    last = at[name] + (nbytes - 1) // 16 * 16
    for where in (at[name] - out + 16, at[name], last):
        assert _prefill(output=where, **at, **_SIZES) == INVALID
        assert "overlaps" in _lib.last_error()[1]
        assert _decode(output=where, workspace=M, num_tokens=10, **at, **_SIZES) == INVALID
        assert "overlaps" in _lib.last_error()[1]
    for where in (at[name] - (ws - 1) // 256 * 256, at[name]):
        assert _decode(output=1 << 20, workspace=where, workspace_bytes=1 << 40, num_tokens=10, **at,
                       **_SIZES) == INVALID
        assert "overlaps" in _lib.last_error()[1]
