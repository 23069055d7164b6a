"""A search's calls out of turn: what they would spoil is refused before anything
changes, and the search goes on."""

import numpy as np
import pytest

from swiftllm_amd import paged_attention as pa
from swiftllm_amd._hip import DeviceArray, synchronize
from test_gpu_beam_search import start

pytestmark = pytest.mark.gpu

ARRAYS = ("scores", "next_rows", "next_tokens", "ref_counts", "num_free", "free_blocks", "counts", "new_lens", "block_tables",
          "context_lens")


def _search(seed=1, lens=(20, 37)):
    return start(np.random.default_rng(seed), list(lens), 4, 32, 8, 80, 4, 2, 64, "f16")


def _state(s):
    synchronize()
    return {k: getattr(s.search, k).numpy() for k in ARRAYS}


def test_two_searches_on_one_step(dev):
    """In turns from fork() on; a plan between the other's plan() and fork() is refused by that one."""
    a, b = _search(1), _search(2, (100, 3))
    b.step = a.step
    taken = {}
    for s in (a, b):
        s.inputs()
        s.forked()
        s.layers()
        synchronize()
        taken[s] = int(s.check(0)[0][0])
        if s is a:
            before = {k: getattr(a.search, k).numpy() for k in ARRAYS if k != "context_lens"}
    a.inputs()
    for call in (lambda: a.search.select(a.d_logits), lambda: a.search.context_lens, a.forked,
                 lambda: a.search.fork([], [], 2, 64)):
        with pytest.raises(pa.InvalidParameter):
            call()
    synchronize()
    for k, v in before.items():
        assert np.array_equal(getattr(a.search, k).numpy(), v), k
    b.steps(2, taken=taken[b])


@pytest.mark.parametrize("bad", ["lists", "null", "heads", "head_dim"])
def test_caches_that_are_refused(dev, bad):
    """By fork() and by compact(), with the tables as they were: the same call with the right caches goes on from them."""
    s = _search()
    k, v = [c[0] for c in s.caches], [c[1] for c in s.caches]
    args = dict(lists=(k, v[:1], 2, 64), null=([k[0], None], v, 2, 64), heads=(k, v, 0, 64), head_dim=(k, v, 2, -64))[bad]
    taken = s.steps(1)
    s.inputs()
    s.search.select(s.d_logits)
    before = _state(s)
    with pytest.raises(pa.InvalidParameter):
        s.search.fork(*args)
    for key, x in _state(s).items():
        assert np.array_equal(x, before[key]), key
    s.search.fork(k, v, 2, 64)
    before = _state(s)
    with pytest.raises(pa.InvalidParameter):
        s.search.compact(*args, DeviceArray((80,), np.int32), 80)
    for key, x in _state(s).items():
        assert np.array_equal(x, before[key]), key
    s.layers()
    synchronize()
    s.check(taken)


def test_compact_keeps_the_counts_of_the_fork(dev):
    """How many rows fork() cut is there after compact() too, which counts by itself."""
    s = start(np.random.default_rng(5), [30, 30], 4, 32, 8, 7, 4, 2, 64, "f16")
    s.inputs()
    s.forked()
    synchronize()
    counts, refs = s.search.counts.numpy(), s.search.ref_counts.numpy()
    assert counts[1] > 0
    s.search.compact([c[0] for c in s.caches], [c[1] for c in s.caches], 2, 64, DeviceArray((7,), np.int32), 7)
    synchronize()
    assert np.array_equal(s.search.counts.numpy(), counts)
    used = np.flatnonzero(refs)
    assert s.search.compact_counts.numpy().tolist() == [(used >= len(used)).sum(), len(used)]


def test_ids_and_lengths_past_32_bits_are_refused(dev):
    """Numbers that a cast to 32 bits would bring back into range."""
    s = _search()
    s.search.start(np.array([[3, 4], [5, 6]]), np.array([20, 32]))
    for tables, lens in (([[3, 4], [2 ** 32 + 5, 6]], [20, 32]), ([[3, 4], [5, -2 ** 32]], [20, 32]),
                         ([[3, 4], [5, 6]], [2 ** 32 + 4, 32]), ([[3, 4], [5, 6]], [20, 16 - 2 ** 32])):
        with pytest.raises(pa.InvalidParameter):
            s.search.start(np.array(tables), np.array(lens))
    # (entries behind a prompt may hold anything)
    s.search.start(np.array([[3, 2 ** 40], [5, 6]]), np.array([16, 32]))
    assert s.search.ref_counts.numpy()[[3, 5, 6]].tolist() == [1, 1, 1] and int(s.search.num_free.numpy()[0]) == 77
