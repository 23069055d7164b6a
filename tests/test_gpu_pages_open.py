"""Forks of rows that hold the same partly filled block with different parents (one
prompt in two requests, a prompt's tail kept for later ones): one of its holders
keeps it. The rule by hand, without a GPU; then fork_pages against the oracle,
every array to the bit, and what the rule is for: no block is lost."""

import numpy as np
import pytest

import oracle
from test_gpu_pages import Pool


def _fork(tables, ctx, parents, refs):
    tables = np.array(tables, np.int32)
    free = np.flatnonzero(np.array(refs) == 0)
    return oracle.fork_pages(tables, tables, ctx, parents, refs, np.pad(free, (0, len(refs) - len(free))), len(free))


def test_two_requests_of_one_prompt_by_hand():
    # 20 tokens in blocks 0 and 1, held by rows 0 and 2, each with two beams to be.
    out = _fork([[0, 1], [9, 9], [0, 1], [9, 9]], [20, 0, 20, 0], [0, 0, 2, 2], [2, 2, 0, 0, 0])
    tables, ctx, refs, free, n, pairs, counts = out
    assert tables.tolist() == [[0, 2], [0, 3], [0, 4], [0, 1]]     # the last of them keeps block 1
    assert ctx.tolist() == [20] * 4 and counts.tolist() == [3, 0] and refs.tolist() == [4, 1, 1, 1, 1] and n == 0
    assert pairs.tolist() == [[1, 2], [1, 3], [1, 4], [-1, -1]]
    # one free block for two rows that go on: both do
    tables, ctx, refs, free, n, _, counts = _fork([[0, 1], [0, 1]], [20, 20], [0, 1], [2, 2, 0])
    assert tables.tolist() == [[0, 2], [0, 1]] and ctx.tolist() == [20, 20]
    assert refs.tolist() == [2, 1, 1] and n == 0 and counts.tolist() == [1, 0]
    # no free block: one row is cut, the other goes on
    _, ctx, refs, _, _, _, counts = _fork([[0, 1], [0, 1]], [20, 20], [0, 1], [2, 2])
    assert ctx.tolist() == [16, 20] and refs.tolist() == [2, 1] and counts.tolist() == [0, 1]
    # somebody else holds it too: both copy
    tables, _, refs, _, _, _, counts = _fork([[0, 1], [0, 1]], [20, 20], [0, 1], [2, 3, 0, 0])
    assert tables.tolist() == [[0, 2], [0, 3]] and refs.tolist() == [2, 1, 1, 1] and counts.tolist() == [2, 0]
    # a row that holds it filled reads on: the other one copies
    tables, _, refs, _, _, _, counts = _fork([[0, 1], [0, 1]], [32, 20], [0, 1], [2, 2, 0])
    assert tables.tolist() == [[0, 1], [0, 2]] and refs.tolist() == [2, 1, 1] and counts.tolist() == [1, 0]


class Shared(Pool):
    def prompts(self, rng, lens, rows):
        """Row s holds prompt rows[s] (below 0: none), each with blocks of its own."""
        ids, at, blocks = rng.permutation(self.NB), 0, []
        for n in lens:
            k = -(-int(n) // 16)
            blocks.append(ids[at:at + k])
            at += k
        for s, r in enumerate(rows):
            if r >= 0:
                self.h["tables"][s, :len(blocks[r])] = blocks[r]
                self.h["refs"][blocks[r]] += 1
                self.h["ctx"][s] = lens[r]
        rest = np.flatnonzero(self.h["refs"] == 0)
        self.h["free"][:len(rest)] = rest
        self.h["n"][0] = len(rest)
        return self.upload()

    def whole(self):
        """Every block is held or free, and every hold is counted."""
        held = np.zeros(self.NB, int)
        for row, n in zip(self.h["tables"], self.h["ctx"]):
            np.add.at(held, row[:-(-int(n) // 16)], 1)
        assert np.array_equal(held, self.h["refs"])
        assert np.array_equal(np.flatnonzero(held == 0), self.h["free"][:self.h["n"][0]])


@pytest.mark.gpu
@pytest.mark.parametrize("S,R,MB,NB", [(2, 1, 2, 8), (8, 2, 3, 64), (64, 5, 9, 1000), (65, 3, 30, 4097), (300, 7, 20, 9000),
                                       (1024, 40, 8, 40000), (5000, 11, 3, 20000)])
def test_forks_of_shared_prompts(dev, S, R, MB, NB):
    """R prompts, each in many rows, small pools by one workgroup and others; the rows'
    children, and children of those, after tokens of their own."""
    rng = np.random.default_rng(S + R)
    for low in (0, -1):
        p = Shared(S, MB, NB).prompts(rng, rng.integers(1, 16 * MB - 7, R), rng.integers(low, R, S))
        for parents in (np.arange(S), rng.integers(-1, S, S), rng.integers(0, S, S) // 3 * 3):
            p.fork(parents)
            p.whole()
            taken = p.grow((rng.random(S) < 0.8).astype(np.int32))
            p.fork(np.arange(S), taken)
            p.whole()


@pytest.mark.gpu
@pytest.mark.parametrize("NB", [10, 5000])
@pytest.mark.parametrize("spare", [0, 1, 2, 6])
def test_without_room(dev, NB, spare):
    """Four rows of one prompt and as many free blocks as `spare`: as many copies, and one row keeps the block."""
    p = Shared(4, 3, NB).prompts(np.random.default_rng(1), [40], [0, 0, 0, 0])
    for b in p.h["free"][spare:p.h["n"][0]]:
        p.h["refs"][b] += 1
    p.h["n"][0] = spare
    p.upload()
    _, counts = p.fork([0, 1, 2, 3])
    assert counts.tolist() == [min(spare, 3), 3 - min(spare, 3)]
    assert sorted(p.h["ctx"].tolist()) == [32] * (3 - min(spare, 3)) + [40] * (1 + min(spare, 3))


@pytest.mark.gpu
def test_a_prompt_in_two_requests(dev):
    """What a search starts with: requests on one prompt, its rest partly filled."""
    from swiftllm_amd.beam_search import BeamSearch
    from swiftllm_amd._hip import DeviceArray, synchronize

    R, W, NB = 3, 2, 12
    s = BeamSearch(R, W, 64, 4, NB)
    s.start(np.array([[4, 7]] * R), np.array([20] * R))
    logits = DeviceArray.from_numpy(np.random.default_rng(2).standard_normal((R * W, 64)).astype(np.float32))
    kv = DeviceArray.zeros((NB, 1, 64, 16), np.uint16)
    s.select(logits)
    s.fork([kv], [kv], 1, 64)
    synchronize()
    refs, tables = s.ref_counts.numpy(), s.block_tables.numpy()
    assert refs[4] == R * W and refs[7] == 1 and (np.sort(refs)[::-1][1:R * W + 1] == 1).all()
    assert int(s.num_free.numpy()[0]) == NB - 1 - R * W and s.counts.numpy().tolist() == [R * W - 1, 0]
    assert sorted(set(tables[:, 1].tolist())) == sorted(tables[:, 1].tolist())
