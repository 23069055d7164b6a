"""The attention step's plan and rotary entry points without a GPU: argument
checks, the rotary frequencies, and the oracle's plan against the host routine
that it generalises."""

import ast
import inspect
import math
import re

import numpy as np
import pytest

import oracle
from swiftllm_amd import _lib
from swiftllm_amd import attention_step as step
from swiftllm_amd import paged_attention as pa

OK, INVALID, NODEV, UNSUP = 0, -4, -5, -6
P = 0x100000   # never dereferenced: validation fails first


def _plan(**kw):
    a = dict(block_tables=P, cached_lens=2 * P, new_lens=3 * P, free_blocks=4 * P, num_free=5 * P,
             free_capacity=8, num_seqs=4, max_num_blocks_per_seq=4, block_size=16, num_tokens=9,
             num_blocks=0, context_lens=6 * P, query_offsets=7 * P, positions=8 * P,
             slot_mapping=9 * P, counts=10 * P)
    a.update(kw)
    return _lib.lib().swiftllm_hip_plan_step(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(num_seqs=-1), INVALID),
    (dict(num_tokens=-1), INVALID),
    (dict(max_num_blocks_per_seq=-1), INVALID),
    (dict(free_capacity=-1), INVALID),
    (dict(block_size=0), INVALID),
    (dict(block_size=32), UNSUP),
    (dict(num_seqs=65536), UNSUP),
    (dict(max_num_blocks_per_seq=1 << 27), UNSUP),
    (dict(num_tokens=(1 << 30) - 1), UNSUP),
    (dict(counts=0), INVALID),
    (dict(num_free=0), INVALID),
    (dict(query_offsets=0), INVALID),
    (dict(free_blocks=0), INVALID),
    (dict(positions=0), INVALID),
    (dict(block_tables=0), INVALID),
    (dict(counts=10 * P + 2), INVALID),
    (dict(context_lens=2 * P), INVALID),           # on cached_lens
    (dict(context_lens=3 * P + 12), INVALID),      # on the end of new_lens
    (dict(slot_mapping=8 * P + 32), INVALID),      # on positions
    (dict(counts=7 * P + 16), INVALID),            # on query_offsets' last entry
])
def test_plan_refuses(kw, code):
    assert _plan(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


def _rotary(**kw):
    a = dict(query_out=P, query=2 * P, key=3 * P, value=4 * P, key_cache=5 * P, value_cache=6 * P,
             positions=7 * P, slot_mapping=8 * P, inv_freq=9 * P, attn_factor=1.0, interleaved=0,
             dtype=0, num_tokens=5, num_heads=8, num_kv_heads=2, head_dim=64, rotary_dim=64,
             block_size=16, query_stride=512, key_stride=128, value_stride=128, num_blocks=0)
    a.update(kw)
    return _lib.lib().swiftllm_hip_rotary_and_cache(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(num_tokens=-1), INVALID),
    (dict(num_heads=0), INVALID),
    (dict(attn_factor=math.nan), INVALID),
    (dict(attn_factor=math.inf), INVALID),
    (dict(rotary_dim=66), INVALID),
    (dict(rotary_dim=31), INVALID),
    (dict(rotary_dim=-2), INVALID),
    (dict(head_dim=96, rotary_dim=96), UNSUP),
    (dict(block_size=8), UNSUP),
    (dict(dtype=2), UNSUP),
    (dict(dtype=-1), UNSUP),
    (dict(query_stride=511), INVALID),
    (dict(key_stride=127), INVALID),
    (dict(value_stride=(1 << 40) + 1), INVALID),
    (dict(key=0), INVALID),
    (dict(inv_freq=0), INVALID),
    (dict(key_cache=5 * P + 4), INVALID),
    (dict(inv_freq=9 * P + 4), INVALID),
    (dict(query=2 * P + 1), INVALID),
    (dict(query=P, query_stride=1024), INVALID),   # in place, but rows elsewhere
    (dict(query=P + 16), INVALID),
    (dict(key=P + 1024), INVALID),
    (dict(value=P + 4 * 1024 + 512), INVALID),
    (dict(num_tokens=2_000_000_000, query_out=1 << 44, query=2 << 44, key=3 << 44, value=4 << 44), UNSUP),
])
def test_rotary_refuses(kw, code):
    assert _rotary(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


def test_python_refuses_unknown_types():
    with pytest.raises(pa.NotSupported):
        step.rotary_and_cache(P, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P, 7 * P, 8 * P, 9 * P, 5, 8, 2,
                              64, 64, 16, dtype="float32")


def test_oracle_plan_matches_the_host_slot_mapping():
    """The slots of each sequence are get_slot_mapping of its completed table."""
    rng = np.random.default_rng(3)
    S, MB = 11, 9
    cached, new = rng.integers(0, 80, S), rng.integers(0, 60, S)
    bt = np.zeros((S, MB), np.int32)
    ids = rng.permutation(400)
    at = 0
    for s in range(S):
        n = -(-int(cached[s]) // 16)
        bt[s, :n] = ids[at:at + n]
        at += n
    T = int(new.sum()) + 5
    out, ctx, off, pos, slots, counts = oracle.plan_step(bt, cached, new, ids[at:], T)
    assert counts.tolist() == [sum(-(-int(c + n) // 16) + -(int(c) // -16) * -1 for c, n in zip(cached, new)),
                               new.sum(), 0]
    for s in range(S):
        got = slots[off[s]:off[s + 1]]
        want = pa.get_slot_mapping(out[s], 16, int(cached[s]), int(new[s]))
        assert got.tolist() == want.tolist()
        assert pos[off[s]:off[s + 1]].tolist() == list(range(cached[s], cached[s] + new[s]))
    assert (slots[off[-1]:] == -1).all() and (pos[off[-1]:] == -1).all()
    assert len(set(slots[:off[-1]].tolist())) == off[-1]


def test_inv_freq_kinds():
    """Each scaling against its definition at the ends: what stays and what is
    interpolated by the factor, and monotone in between."""
    plain, f = step.rotary_inv_freq(128, 500000.0)
    assert f == 1.0 and plain.dtype == np.float64 and plain[0] == 1.0
    assert np.allclose(plain, 500000.0 ** (-np.arange(64) / 64), rtol=1e-14)
    linear, f = step.rotary_inv_freq(128, 500000.0, "linear", factor=4.0)
    assert f == 1.0 and np.allclose(linear * 4.0, plain, rtol=1e-14)
    ntk, _ = step.rotary_inv_freq(128, 500000.0, "ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1] * 4.0, plain[-1], rel_tol=1e-12)
    yarn, f = step.rotary_inv_freq(128, 10000.0, "yarn", factor=16.0, original_context=4096)
    base, _ = step.rotary_inv_freq(128, 10000.0)
    assert math.isclose(f, 0.1 * math.log(16.0) + 1.0)
    turns = 4096 * base / (2 * math.pi)
    assert np.allclose(yarn[turns > 40], base[turns > 40], rtol=1e-14)
    assert np.allclose(yarn[turns < 0.9] * 16, base[turns < 0.9], rtol=1e-14)
    assert (np.diff(yarn) < 0).all()
    banded, f = step.rotary_inv_freq(128, 500000.0, "banded", factor=8.0, original_context=8192)
    turns = 8192 * plain / (2 * math.pi)
    assert f == 1.0
    assert np.allclose(banded[turns >= 4], plain[turns >= 4], rtol=1e-14)
    assert np.allclose(banded[turns <= 1] * 8, plain[turns <= 1], rtol=1e-14)
    assert (np.diff(banded) < 0).all()
    assert step.rotary_inv_freq(0)[0].size == 0
    for kind in ("none", "linear", "ntk", "yarn", "banded"):
        assert step.rotary_inv_freq(2, scaling=kind, factor=2.0)[0].shape == (1,)
    with pytest.raises(pa.NotSupported):
        step.rotary_inv_freq(128, scaling="cubic")
    with pytest.raises(pa.InvalidParameter):
        step.rotary_inv_freq(3)
    with pytest.raises(pa.InvalidParameter):
        step.rotary_inv_freq(64, factor=0.0)


@pytest.mark.parametrize("name", ["query_stride", "key_stride", "value_stride"])
def test_rotary_refuses_strides_past_any_memory(name):
    """Each within its bound, but not the last token's offset."""
    far = dict(query_out=1 << 44, query=2 << 44, key=3 << 44, value=4 << 44)
    for T, stride in ((1 << 24, 1 << 40), ((1 << 23) + 1, 1 << 40), (66, 1 << 40), ((1 << 20) + 2, 1 << 26)):
        assert _rotary(num_tokens=T, **far, **{name: stride}) == INVALID, (T, stride, _lib.last_error())
        assert f"num_tokens={T}" in _lib.last_error()[1]


@pytest.mark.parametrize("name,nbytes", [
    ("positions", 5 * 4), ("slot_mapping", 5 * 4), ("inv_freq", 32 * 8), ("key_cache", 3 * 2 * 64 * 16 * 2),
    ("value_cache", 3 * 2 * 64 * 16 * 2), ("key", 5 * 128 * 2), ("value", 5 * 128 * 2)])
def test_rotary_refuses_queries_out_on_any_other_argument(name, nbytes):
    at = {"positions": 7 * P, "slot_mapping": 8 * P, "inv_freq": 9 * P, "key_cache": 5 * P, "value_cache": 6 * P,
          "key": 3 * P, "value": 4 * P}[name]
    out = 5 * 512 * 2
    for where in (at - out + 8, at, at + nbytes - 2):
        assert _rotary(query_out=where, num_blocks=3) == INVALID
        assert "overlaps" in _lib.last_error()[1]


def test_documented_calls_of_a_step_are_calls():
    """The example of AttentionStep's docstring: every call fits its signature."""
    doc = inspect.getdoc(step.AttentionStep)
    lines = re.findall(r"^ +(?:step = AttentionStep|step\.\w+)\(.*?\)(?= *(?:#|$))", doc, flags=re.M)
    assert len(lines) == 3
    for line in lines:
        call = ast.walk(ast.parse(line.strip()))
        call = next(n for n in call if isinstance(n, ast.Call))
        f = step.AttentionStep if isinstance(call.func, ast.Name) else getattr(step.AttentionStep, call.func.attr)
        args = [None] * (len(call.args) + (f is not step.AttentionStep))
        inspect.signature(f).bind(*args, **{k.arg: None for k in call.keywords})


@pytest.mark.parametrize("kw", [
    dict(scaling="yarn", base=1.0), dict(scaling="yarn", base=0.5), dict(scaling="yarn", beta_fast=math.inf),
    dict(scaling="yarn", beta_fast=math.nan), dict(scaling="yarn", beta_slow=0.0),
    dict(scaling="yarn", original_context=math.inf), dict(base=math.inf), dict(base=math.nan), dict(base=0.0),
    dict(scaling="linear", factor=math.inf), dict(scaling="ntk", factor=math.nan),
    dict(scaling="banded", low_factor=4.0), dict(scaling="banded", high_factor=math.inf),
    dict(scaling="banded", low_factor=-math.inf)])
def test_inv_freq_refuses(kw):
    """Numbers that leave no frequencies are refused, not divided by."""
    with pytest.raises(pa.InvalidParameter):
        step.rotary_inv_freq(64, **kw)


@pytest.mark.parametrize("base", [0.5, 1.0])
@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "banded"])
def test_inv_freq_of_small_bases(kind, base):
    """Only the ramp over pairs needs frequencies that fall."""
    f, _ = step.rotary_inv_freq(64, base, kind, factor=2.0)
    assert f.shape == (32,) and np.isfinite(f).all()
