"""A search's calls out of turn: what they would spoil is refused before anything
changes, and the search goes on."""

import numpy as np
import pytest

from swiftllm_amd import paged_attention as pa
from swiftllm_amd._hip import synchronize
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
