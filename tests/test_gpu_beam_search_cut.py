"""Rows of a search that bring no token, because fork() cut them or plan() found no
block: what stands in their logits is nobody's, and select() passes over them, in
a graph too, where no caller comes between the steps."""

import numpy as np
import pytest

from swiftllm_amd import _lib
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize
from test_beam_pages_host import INVALID, P
from test_gpu_beam_search import start
from test_gpu_beam_select import Select, _logits


def _rows(**kw):
    a = dict(logits=P, beam_scores=2 * P, query_offsets=10 * P, cand_scores=3 * P, cand_rows=4 * P, cand_tokens=5 * P,
             next_scores=6 * P, next_rows=7 * P, next_tokens=8 * P, workspace=9 * P,
             workspace_bytes=1 << 40, dtype=2, num_requests=3, beam_width=4, vocab=1000,
             num_candidates=8, logits_stride=1000, eos_id=-1)
    a.update(kw)
    return _lib.lib().swiftllm_hip_beam_select_rows(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(query_offsets=10 * P + 2), dict(query_offsets=7 * P), dict(query_offsets=3 * P - 48),
                                dict(query_offsets=9 * P + 512), dict(logits=0), dict(num_candidates=3)])
def test_select_of_rows_refuses(kw):
    assert _rows(**kw) == INVALID
    assert _lib.last_error()[0] == INVALID and _lib.last_error()[1]


@pytest.mark.gpu
@pytest.mark.parametrize("R,W,V,C", [(3, 4, 9000, 8), (2, 16, 50000, 32)])
def test_rows_without_a_token_have_no_logits(dev, R, W, V, C):
    """At random, a whole request's, and with offsets that fall."""
    rng = np.random.default_rng(W)
    s = Select(_logits(rng, R, W, V), -rng.random((R, W)), C)
    brings = rng.random(R * W) < 0.6
    brings[:W] = False
    off = np.concatenate([[0], np.cumsum(brings)]).astype(np.int32)
    off[-1] = off[-2] - 3
    brings[-1] = False
    d_off = DeviceArray.from_numpy(off)
    from swiftllm_amd import beam_search as bs
    bs.beam_select(s.at, s.d_s, *s.out.values(), s.ws, s.ws.nbytes, R, W, V, C, query_offsets=d_off)
    s.scores[~brings.reshape(R, W)] = -np.inf      # what it comes to
    got, _ = s.check()
    assert (got[1][0] == -1).all() and brings[got[1][got[1] >= 0]].all()


def _lone(s):
    """Rows with a score that brought no token."""
    off = s.step.query_offsets.numpy()
    return (off[1:] == off[:-1]) & np.isfinite(s.search.scores.numpy().reshape(-1))


@pytest.mark.gpu
def test_row_that_was_cut_ends(dev):
    s = start(np.random.default_rng(5), [30, 30], 4, 32, 8, 7, 4, 2, 64, "f16")
    s.inputs()
    s.forked()
    s.layers()
    took, counts, _ = s.check(0)
    lone = _lone(s)
    assert counts[1] > 0 and lone.any() and not lone.all()
    s.scores = s.scores.copy()
    s.scores.reshape(-1)[lone] = -np.inf       # for the oracle alone
    s.inputs()
    s.x[lone] += 50.0
    s.d_logits.upload(s.x)
    s.forked()
    s.layers()
    s.check(int(took[0]))


@pytest.mark.gpu
def test_rows_cut_and_refused_within_a_graph(dev):
    """Two steps captured, of a pool that runs out in the first of them, against eager
    steps between which the caller sets the scores of rows without a token."""
    a, b = (start(np.random.default_rng(7), [30, 30], 4, 32, 8, 12, 4, 2, 64, "f16") for _ in range(2))
    stream = Stream()

    def step(s, stream=None):
        s.forked(stream)
        s.layers(stream)

    def ended(s):
        synchronize()
        lone = _lone(s)
        scores = s.search.scores.numpy()
        scores.reshape(-1)[lone] = -np.inf
        s.search.scores.upload(scores)
        return lone.sum()

    for s in (a, b):
        s.rng = np.random.default_rng(8)
        s.inputs()
        step(s)
        step(s)
    g = Graph(stream, lambda: (step(a, stream), step(a, stream)))
    within = 0
    for _ in range(12):
        for s in (a, b):
            s.inputs()
        g.launch(stream)
        ended(b)
        step(b)
        within += ended(b)
        step(b)
        synchronize()
        for k in ("scores", "cand_scores", "cand_rows", "cand_tokens", "next_rows", "next_tokens", "ref_counts", "num_free",
                  "copy_pairs", "counts", "new_lens", "block_tables", "context_lens"):
            assert np.array_equal(getattr(a.search, k).numpy(), getattr(b.search, k).numpy()), k
    assert within > 0
