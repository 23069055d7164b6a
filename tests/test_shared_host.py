"""Attention over shared blocks without a GPU: argument checks of the plan and the
attention, and the oracle's rule of what a group shares on cases done by hand."""

import math

import numpy as np
import pytest

import oracle
from swiftllm_amd import _lib
from swiftllm_amd import attention_step as step
from swiftllm_amd import paged_attention as pa

INVALID, UNSUP = -4, -6
P = 1 << 32   # never dereferenced: validation fails first


def _plan(**kw):
    a = dict(plan=P, plan_bytes=1 << 40, shared_blocks=2 * P, block_tables=3 * P, context_lens=4 * P,
             group_offsets=5 * P, num_groups=2, num_seqs=6, num_heads=8, num_kv_heads=2, head_dim=64,
             block_size=16, max_num_blocks_per_seq=4, min_saved=-1)
    a.update(kw)
    return _lib.lib().swiftllm_hip_plan_shared(*a.values(), None)


def _decode(**kw):
    a = dict(output=P, workspace=2 * P, workspace_bytes=1 << 40, plan=3 * P, plan_bytes=1 << 40, query=4 * P,
             key_cache=5 * P, value_cache=6 * P, block_tables=7 * P, query_offsets=0, alibi_slopes=0,
             scale=0.1, softcap=0.0, dtype=0, num_tokens=-1, num_seqs=6, num_heads=8, num_kv_heads=2,
             head_dim=64, block_size=16, max_num_blocks_per_seq=4, num_blocks=100)
    a.update(kw)
    return _lib.lib().swiftllm_hip_shared_decode(*a.values(), None)


SIZES = [
    (dict(num_seqs=-1), INVALID),
    (dict(num_seqs=65536), UNSUP),
    (dict(num_heads=0), INVALID),
    (dict(num_heads=9), INVALID),
    (dict(num_kv_heads=0), INVALID),
    (dict(head_dim=0), INVALID),
    (dict(head_dim=96), UNSUP),
    (dict(block_size=0), INVALID),
    (dict(block_size=32), UNSUP),
    (dict(max_num_blocks_per_seq=-1), INVALID),
    (dict(max_num_blocks_per_seq=1 << 27), UNSUP),
    (dict(num_seqs=65535, max_num_blocks_per_seq=1 << 14), UNSUP),
    (dict(plan=0), INVALID),
    (dict(block_tables=0), INVALID),
    (dict(plan_bytes=300), INVALID),
]


@pytest.mark.parametrize("kw,code", SIZES + [
    (dict(num_groups=-1), INVALID),
    (dict(num_groups=65536), UNSUP),
    (dict(shared_blocks=0), INVALID),
    (dict(context_lens=0), INVALID),
    (dict(group_offsets=0), INVALID),
    (dict(plan=P + 128), INVALID),
    (dict(group_offsets=5 * P + 2), INVALID),
    (dict(shared_blocks=5 * P + 8), INVALID),
    (dict(plan=4 * P), INVALID),
])
def test_plan_refuses(kw, code):
    assert _plan(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


@pytest.mark.parametrize("kw,code", SIZES + [
    *[({k: 0}, INVALID) for k in ("output", "workspace", "query", "key_cache", "value_cache")],
    (dict(workspace_bytes=1000), INVALID),
    (dict(dtype=2), UNSUP),
    (dict(scale=math.nan), INVALID),
    (dict(softcap=-1.0), INVALID),
    (dict(softcap=math.inf), INVALID),
    (dict(softcap=1025.0), UNSUP),
    (dict(query_offsets=8 * P), INVALID),               # and num_tokens below 0
    (dict(query_offsets=8 * P + 2, num_tokens=6), INVALID),
    (dict(key_cache=5 * P + 8), INVALID),
    (dict(query=4 * P + 4), INVALID),
    (dict(output=P + 1), INVALID),
    (dict(workspace=2 * P + 128), INVALID),
    (dict(plan=3 * P + 4), INVALID),
    (dict(alibi_slopes=8 * P + 2), INVALID),
    (dict(output=4 * P), INVALID),                      # not in the query's place
    (dict(output=6 * P + 64), INVALID),
    (dict(workspace=3 * P), INVALID),
    (dict(output=7 * P + 8), INVALID),
])
def test_decode_refuses(kw, code):
    assert _decode(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


def test_python_refusals():
    with pytest.raises(pa.NotSupported):
        step.shared_decode(P, P, 0, P, 0, P, P, P, P, step.ScoreParams(0.1, window=5), 1, 8, 8, 64, 16, 1)
    with pytest.raises(pa.NotSupported):
        step.shared_decode(P, P, 0, P, 0, P, P, P, P, step.ScoreParams(0.1), 1, 8, 8, 64, 16, 1, dtype="f32")
    with pytest.raises(pa.InvalidParameter):
        step.plan_shared_size(-1, 8, 8, 64, 16, 1)
    with pytest.raises(pa.NotSupported):
        step.shared_decode_workspace_size(1, 8, 8, 80, 16, 1)


def test_oracle_shared_blocks_by_hand():
    bt = np.array([[1, 2, 3], [1, 2, 4], [1, 9, 3], [7, 7, 7], [7, 7, 8], [5, 6, 0]])
    assert oracle.shared_blocks(bt, [48, 33, 0, 32, 16, 20], [0, 3, 3, 5, 6]).tolist() == [2, 0, 1, 2]
    assert oracle.shared_blocks(bt, [48, 48, 17, 99, 99, -1], [0, 3, 5, 6]).tolist() == [1, 2, 0]
    assert oracle.shared_blocks(bt, [48] * 6, [0, 4, 2]).tolist() == [0, 0]
