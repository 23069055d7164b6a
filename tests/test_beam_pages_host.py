"""Beam selection and the pages' forks and compaction without a GPU: argument
checks of the entry points, and the oracle's rules on cases done by hand."""

import numpy as np
import pytest

import oracle
from swiftllm_amd import _lib, beam_search, pages
from swiftllm_amd import paged_attention as pa

INVALID, UNSUP = -4, -6
P = 1 << 32   # never dereferenced: validation fails first


def _select(**kw):
    a = dict(logits=P, beam_scores=2 * P, cand_scores=3 * P, cand_rows=4 * P, cand_tokens=5 * P,
             next_scores=6 * P, next_rows=7 * P, next_tokens=8 * P, workspace=9 * P,
             workspace_bytes=1 << 40, dtype=2, num_requests=3, beam_width=4, vocab=1000,
             num_candidates=8, logits_stride=1000, eos_id=-1)
    a.update(kw)
    return _lib.lib().swiftllm_hip_beam_select(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(num_requests=-1), INVALID),
    (dict(beam_width=0), INVALID),
    (dict(vocab=0), INVALID),
    (dict(num_candidates=3), INVALID),
    (dict(num_candidates=65), UNSUP),
    (dict(vocab=(1 << 27) + 1, logits_stride=1 << 28), UNSUP),
    (dict(num_requests=1 << 19, vocab=200000, logits_stride=200000), UNSUP),
    (dict(dtype=3), UNSUP),
    (dict(logits_stride=999), INVALID),
    (dict(logits_stride=(1 << 40) + 1), INVALID),
    *[({k: 0}, INVALID) for k in ("logits", "beam_scores", "cand_scores", "cand_rows", "cand_tokens",
                                  "next_scores", "next_rows", "next_tokens", "workspace")],
    (dict(logits=P + 2), INVALID),
    (dict(logits=P + 1, dtype=0), INVALID),
    (dict(cand_rows=4 * P + 2), INVALID),
    (dict(workspace=9 * P + 128), INVALID),
    (dict(workspace_bytes=1000), INVALID),
    (dict(cand_tokens=3 * P + 4), INVALID),             # outputs that overlap
    (dict(next_scores=2 * P + 4), INVALID),             # neither beam_scores itself nor apart from it
    (dict(cand_scores=P + 4000), INVALID),
    (dict(workspace=P), INVALID),
])
def test_select_refuses(kw, code):
    assert _select(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


def _fork(**kw):
    a = dict(block_tables_out=P, context_lens_out=2 * P, block_tables=3 * P, context_lens=4 * P,
             parents=5 * P, ref_counts=6 * P, free_blocks=7 * P, num_free=8 * P, taken=0,
             copy_pairs=9 * P, new_lens=0, counts=10 * P, workspace=11 * P, workspace_bytes=1 << 40,
             num_seqs=4, max_num_blocks_per_seq=8, block_size=16, num_blocks=100)
    a.update(kw)
    return _lib.lib().swiftllm_hip_fork_pages(*a.values(), None)


def _compact(**kw):
    a = dict(block_tables_out=P, ref_counts_out=2 * P, block_tables=3 * P, context_lens=4 * P,
             ref_counts=5 * P, free_blocks=6 * P, num_free=7 * P, copy_pairs=8 * P, new_ids=9 * P,
             counts=10 * P, workspace=11 * P, workspace_bytes=1 << 40, num_seqs=4,
             max_num_blocks_per_seq=8, block_size=16, num_blocks=100, max_moves=50)
    a.update(kw)
    return _lib.lib().swiftllm_hip_compact_pages(*a.values(), None)


SIZES = [
    (dict(num_seqs=-1), INVALID),
    (dict(num_seqs=65536), UNSUP),
    (dict(max_num_blocks_per_seq=-1), INVALID),
    (dict(max_num_blocks_per_seq=1 << 27), UNSUP),
    (dict(block_size=0), INVALID),
    (dict(block_size=32), UNSUP),
    (dict(num_blocks=0), INVALID),
    (dict(num_blocks=1 << 27), UNSUP),
    (dict(workspace=0), INVALID),
    (dict(workspace=11 * P + 64), INVALID),
    (dict(workspace_bytes=64), INVALID),
]


@pytest.mark.parametrize("kw,code", SIZES + [
    *[({k: 0}, INVALID) for k in ("block_tables_out", "context_lens_out", "block_tables", "context_lens",
                                  "parents", "ref_counts", "free_blocks", "num_free", "copy_pairs",
                                  "counts")],
    (dict(copy_pairs=9 * P + 4), INVALID),
    (dict(taken=12 * P + 2), INVALID),
    (dict(block_tables_out=3 * P), INVALID),            # tables are not forked in place
    (dict(context_lens_out=4 * P), INVALID),
    (dict(taken=7 * P + 8), INVALID),
    (dict(new_lens=5 * P), INVALID),
    (dict(new_lens=12 * P + 1), INVALID),
    (dict(counts=6 * P + 396), INVALID),
])
def test_fork_refuses(kw, code):
    assert _fork(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


@pytest.mark.parametrize("kw,code", SIZES + [
    *[({k: 0}, INVALID) for k in ("block_tables_out", "ref_counts_out", "block_tables", "context_lens",
                                  "ref_counts", "free_blocks", "num_free", "copy_pairs", "new_ids",
                                  "counts")],
    (dict(max_moves=-1), INVALID),
    (dict(max_moves=101), INVALID),
    (dict(ref_counts_out=5 * P), INVALID),
    (dict(block_tables_out=3 * P + 4), INVALID),        # the tables themselves, or apart from them
    (dict(new_ids=6 * P), INVALID),
])
def test_compact_refuses(kw, code):
    assert _compact(**kw) == code
    assert _lib.last_error()[0] == code and _lib.last_error()[1]


def test_python_refusals():
    with pytest.raises(pa.NotSupported):
        beam_search.beam_select(P, P, P, P, P, P, P, P, P, 0, 1, 1, 10, 1, dtype="f64")
    with pytest.raises(pa.InvalidParameter):
        beam_search.beam_select_workspace_size(1, 0, 10, 1)
    with pytest.raises(pa.InvalidParameter):
        pages.pages_workspace_size(1, 0)
    assert pages.pages_workspace_size(1, 1) > 0
    assert beam_search.beam_select_workspace_size(0, 1, 10, 1) > 0


def test_oracle_select_by_hand():
    log = np.log
    x = np.array([[[log(1.0), log(2.0), log(5.0)], [log(4.0), log(4.0), -np.inf]]])
    got = oracle.beam_select(x, np.array([[log(0.5), log(0.25)]]), 4, eos_id=2)
    # beam 0: 1/16, 1/8, 5/16; beam 1: 1/8 twice. The tie goes to the lower beam, then the lower token.
    assert np.allclose(np.exp(got[0]), [[5 / 16, 1 / 8, 1 / 8, 1 / 8]])
    assert got[1].tolist() == [[0, 0, 1, 1]] and got[2].tolist() == [[2, 1, 0, 1]]
    assert got[4].tolist() == [[0, 1]] and got[5].tolist() == [[1, 0]]
    got = oracle.beam_select(np.array([[[np.inf, 0.0, np.inf, np.nan]]]), np.array([[-1.0]]), 3)
    assert got[2].tolist() == [[0, 2, -1]] and np.allclose(got[0][0, :2], -1 - log(2))


def test_oracle_fork_by_hand():
    # A prompt of 20 tokens in blocks 5 and 3, held by row 0; row 1 holds 2.
    bt = np.array([[5, 3, 0], [2, 0, 0], [0, 0, 0]], np.int32)
    refs = np.array([0, 0, 1, 1, 0, 1], np.int32)
    out = oracle.fork_pages(np.full((3, 3), -7, np.int32), bt, [20, 16, 0], [0, 0, 0], refs,
                            np.zeros(6, np.int32), 0)
    tables, ctx, refs, free, n, pairs, counts = out
    assert tables.tolist() == [[5, 0, -7], [5, 1, -7], [5, 3, -7]]    # the last child keeps block 3
    assert ctx.tolist() == [20] * 3 and counts.tolist() == [2, 0]
    assert pairs.tolist() == [[3, 0], [3, 1], [-1, -1]]
    assert refs.tolist() == [1, 1, 0, 1, 0, 3] and free[:n].tolist() == [2, 4]
    # and all of them end but one; then a pool without room
    out = oracle.fork_pages(tables, tables, ctx, [-1, 9, 2], refs, free, n)
    assert out[1].tolist() == [0, 0, 20] and out[2].tolist() == [0, 0, 0, 1, 0, 1]
    out = oracle.fork_pages(np.zeros((2, 2), np.int32), [[0, 1], [0, 0]], [30, 0], [0, 0], [1, 1], [0, 0], 0)
    assert out[1].tolist() == [16, 30] and out[6].tolist() == [0, 1] and out[2].tolist() == [2, 1]


def test_oracle_compact_by_hand():
    out = oracle.compact_pages(np.array([[6, 2], [2, 9]], np.int32), [32, 16], [0, 0, 2, 0, 0, 0, 1, 1],
                               np.zeros(8, np.int32), 8)
    assert out[4][:2].tolist() == [[7, 0], [6, 1]] and (out[4][2:] == -1).all()
    assert out[0].tolist() == [[1, 2], [2, 9]] and out[1].tolist() == [1, 1, 2, 0, 0, 0, 0, 0]
    assert out[2][:out[3]].tolist() == [3, 4, 5, 6, 7] and out[6].tolist() == [2, 3]
