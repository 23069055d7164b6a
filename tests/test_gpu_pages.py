"""fork_pages and compact_pages on the GPU against the oracle, every array to the bit."""

import numpy as np
import pytest

import oracle
from swiftllm_amd import attention_step as step
from swiftllm_amd import pages
from swiftllm_amd import paged_attention as pa
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Pool:
    """Rows over a pool, here and on the device. What no call writes holds -9."""

    def __init__(self, S, MB, NB):
        self.S, self.MB, self.NB = S, MB, NB
        self.h = dict(tables=np.full((S, MB), -9, np.int32), other=np.full((S, MB), -9, np.int32),
                      ctx=np.zeros(S, np.int32), refs=np.zeros(NB, np.int32),
                      free=np.full(NB, -9, np.int32), n=np.zeros(1, np.int32), taken=np.zeros(3, np.int32))
        self.d = {}
        self.pairs, self.counts = DeviceArray((S, 2), np.int64), DeviceArray((2,), np.int32)
        self.ctx_out, self.parents = DeviceArray((S,), np.int32), DeviceArray((S,), np.int32)
        self.new = DeviceArray((S,), np.int32)
        self.refs_out, self.ids = DeviceArray((NB,), np.int32), DeviceArray((NB,), np.int32)
        self.ws = DeviceArray((pages.pages_workspace_size(S, NB),), np.uint8)
        self.ws.fill_byte(0xFF)

    def lone(self, rng, lens):
        """Every row with blocks of its own, anywhere in the pool."""
        ids, at = rng.permutation(self.NB), 0
        for i, n in enumerate(lens):
            k = min(-(-int(n) // 16), self.MB)
            self.h["tables"][i, :k] = ids[at:at + k]
            self.h["refs"][ids[at:at + k]] += 1
            at += k
        self.h["ctx"][:] = lens
        rest = np.sort(ids[at:])
        self.h["free"][:len(rest)] = rest
        self.h["n"][0] = len(rest)
        return self.upload()

    def upload(self):
        for k, v in self.h.items():
            if k in self.d:
                self.d[k].upload(v)
            else:
                self.d[k] = DeviceArray.from_numpy(v)
        return self

    def enqueue_fork(self, taken=False, stream=None):
        d = self.d
        pages.fork_pages(d["other"], self.ctx_out, d["tables"], d["ctx"], self.parents, d["refs"], d["free"], d["n"],
                         self.pairs, self.counts, self.ws, self.ws.nbytes, self.S, self.MB, 16, self.NB,
                         taken=d["taken"] if taken else None, new_lens=self.new if taken else None, stream=stream)

    def fork(self, parents, taken=None):
        """A fork, checked; the new tables are the pool's then."""
        h = self.h
        self.parents.upload(np.asarray(parents, np.int32))
        if taken is not None:
            h["taken"][0] = taken
            self.d["taken"].upload(h["taken"])
        self.enqueue_fork(taken is not None)
        return self.check_fork(parents, taken)

    def check_fork(self, parents, taken=None):
        h = self.h
        synchronize()
        want = oracle.fork_pages(h["other"], h["tables"], h["ctx"], parents, h["refs"], h["free"], int(h["n"][0]), taken or 0)
        got = (self.d["other"].numpy(), self.ctx_out.numpy(), self.d["refs"].numpy(), self.d["free"].numpy(),
               int(self.d["n"].numpy()[0]), self.pairs.numpy(), self.counts.numpy())
        for name, g, w in zip(("tables", "contexts", "references", "free", "num_free", "pairs", "counts"), got, want):
            assert np.array_equal(g, w), name
        if taken is not None:
            p = np.asarray(parents)
            new = (p >= 0) & (p < self.S)
            new[new] &= want[1][new] == np.maximum(h["ctx"][p[new]], 0)     # not cut
            assert np.array_equal(self.new.numpy(), new.astype(np.int32))
        h["other"], h["tables"], h["ctx"] = h["tables"], want[0], want[1]
        h["refs"], h["free"], h["n"][0] = want[2], want[3], want[4]
        self.d["other"], self.d["tables"] = self.d["tables"], self.d["other"]
        self.d["ctx"].upload(h["ctx"])
        return want[5], want[6]

    def grow(self, by):
        """by new tokens a row, their blocks from the front of the free list, as a plan
        takes them; how many."""
        h = self.h
        bt, ctx, _, _, _, counts = oracle.plan_step(h["tables"], h["ctx"], by, h["free"][:h["n"][0]], 1 << 20, self.NB)
        h["tables"], h["ctx"] = bt, ctx
        self.upload()
        return int(counts[0])

    def compact(self, most, in_place=False):
        h, d = self.h, self.d
        pairs = DeviceArray((max(most, 1), 2), np.int64)
        to = d["tables"] if in_place else d["other"]
        pages.compact_pages(to, self.refs_out, d["tables"], d["ctx"], d["refs"], d["free"], d["n"], pairs, self.ids,
                            self.counts, self.ws, self.ws.nbytes, self.S, self.MB, 16, self.NB, most)
        synchronize()
        want = oracle.compact_pages(h["tables"], h["ctx"], h["refs"], h["free"], most)
        tables = want[0]
        if not in_place:     # only what rows use is written
            for i, c in enumerate(h["ctx"]):
                tables[i, min(-(-max(int(c), 0) // 16), self.MB):] = h["other"][i, min(-(-max(int(c), 0) // 16), self.MB):]
        got = (to.numpy(), self.refs_out.numpy(), d["free"].numpy(), int(d["n"].numpy()[0]),
               pairs.numpy()[:most], self.ids.numpy(), self.counts.numpy())
        for name, g, w in zip(("tables", "references", "free", "num_free", "pairs", "new ids", "counts"), got, want):
            assert np.array_equal(g, w), name
        h["tables"], h["refs"], h["free"], h["n"][0] = tables, want[1], want[2], want[3]
        self.upload()
        return want


@pytest.mark.parametrize("S,MB,NB,most", [(1, 1, 1, 16), (4, 6, 30, 90), (7, 3, 4095, 48), (64, 40, 4096, 600),
                                          (300, 20, 9000, 300), (1024, 8, 4097, 50), (5000, 3, 20000, 45)])
def test_forks(dev, S, MB, NB, most):
    """Steps of a search: rows go on from any of their neighbours, end, and grow."""
    rng = np.random.default_rng(S + NB)
    lens = rng.integers(0, most + 1, S)
    while (-(-lens // 16)).sum() > NB * 0.8:
        lens //= 2
    p = Pool(S, MB, NB).lone(rng, lens)
    W = int(rng.integers(1, min(S, 33) + 1))
    for i in range(6):
        parents = np.minimum(np.arange(S) // W * W + rng.integers(0, W, S), S - 1)
        parents[rng.random(S) < 0.1] = -1
        parents[rng.random(S) < 0.02] = S
        p.fork(parents)
        taken = p.grow((rng.random(S) < 0.8).astype(np.int32) * rng.integers(1, 3))
        p.fork(np.arange(S), taken)
        assert (p.h["refs"] >= 0).all()


def test_fork_of_one_prompt(dev):
    """A prompt for all rows, and its references while other tables hold some of it."""
    p = Pool(40, 10, 200).lone(np.random.default_rng(0), [150] + [0] * 39)
    pairs, counts = p.fork(np.zeros(40, int))
    assert counts.tolist() == [39, 0]
    p.h["refs"][p.h["tables"][3, 9]] += 1       # somebody else holds a partly filled block
    p.upload()
    pairs, counts = p.fork([3] * 40)
    assert counts.tolist() == [40, 0] and len(set(pairs[:, 1].tolist())) == 40
    pairs, counts = p.fork([-1] * 40)
    assert p.h["refs"].sum() == 1


@pytest.mark.parametrize("spare", [0, 1, 5, 6, 7])
def test_fork_without_room(dev, spare):
    """Rows that find no block end with their whole ones."""
    NB = 3 + spare
    p = Pool(8, 4, NB).lone(np.random.default_rng(1), [40] + [0] * 7)
    _, counts = p.fork(np.zeros(8, int))
    assert counts.tolist() == [min(spare, 7), 7 - min(spare, 7)]
    assert sorted(p.h["ctx"].tolist()) == [32] * (7 - min(spare, 7)) + [40] * (1 + min(spare, 7))
    p.fork(np.arange(8), taken=0)
    p = Pool(4, 4, 4).lone(np.random.default_rng(1), [40, 0, 0, 0])
    p.fork([0, 0, 0, -1], taken=0)


def test_fork_of_odd_rows(dev):
    """Contexts past the table and below zero, block ids of no pool, the same block twice in a row."""
    p = Pool(6, 3, 20)
    p.h["tables"][:] = [[1, 2, 3], [4, -5, 99], [6, 6, 6], [7, 8, 9], [2, 3, 10], [11, 12, 20]]
    p.h["ctx"][:] = [1000, 40, 35, -3, 20, 48]
    for i, n in enumerate([3, 3, 3, 0, 2, 3]):
        for b in p.h["tables"][i, :n]:
            if 0 <= b < 20:
                p.h["refs"][b] += 1
    p.upload()
    p.fork([0, 0, 1, 2, 2, 4])
    p.fork([5, 4, 3, 2, 1, 0])
    p.fork([2 ** 31 - 1, -2 ** 31, 0, 0, 1, 1])


def test_taken_blocks_are_counted_once(dev):
    p = Pool(3, 8, 64).lone(np.random.default_rng(2), [16, 30, 0])
    assert p.grow(np.array([1, 3, 17], np.int32)) == 4
    p.fork([0, 1, 2], taken=4)
    assert p.h["refs"].sum() == 7
    p.fork([0, 1, 2], taken=-3)
    p.fork([0, 1, 2], taken=0)
    p.fork([-1, -1, -1], taken=10 ** 6)       # more than there are: those of the list


@pytest.mark.parametrize("S,MB,NB,most", [(1, 1, 1, 16), (5, 9, 40, 100), (30, 20, 4096, 300), (64, 30, 4097, 400),
                                          (200, 10, 12345, 100), (3, 2000, 70000, 30000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compaction(dev, S, MB, NB, most, in_place):
    rng = np.random.default_rng(S + NB)
    lens = rng.integers(0, most + 1, S)
    while (-(-lens // 16)).sum() > NB * 0.7:
        lens //= 2
    p = Pool(S, MB, NB).lone(rng, lens)
    p.fork(np.where(rng.random(S) < 0.5, np.arange(S), rng.integers(0, S, S)))    # and shared blocks
    for k in (0, 1, min(NB, 100), NB):
        want = p.compact(k, in_place)
    assert (want[1][:want[6][1]] > 0).all() and (want[1][want[6][1]:] == 0).all()
    assert p.compact(NB, in_place)[6][0] == 0


def test_compaction_of_full_and_empty_pools(dev):
    p = Pool(2, 4, 8).lone(np.random.default_rng(3), [64, 64])
    assert p.compact(8)[6].tolist() == [0, 8]
    p.fork([-1, -1])
    assert p.compact(8)[6].tolist() == [0, 0]


def test_compaction_keeps_what_rows_hold(dev):
    """With copy_blocks, every row reads the same values as before."""
    rng = np.random.default_rng(4)
    S, MB, NB, Hkv, D = 12, 6, 128, 2, 64
    p = Pool(S, MB, NB).lone(rng, rng.integers(1, 90, S))
    caches = [rng.integers(0, 1 << 16, (NB, Hkv, D, 16)).astype(np.uint16) for _ in range(4)]
    dev_caches = [DeviceArray.from_numpy(c) for c in caches]
    before = [[c[p.h["tables"][i, :-(-p.h["ctx"][i] // 16)]] for i in range(S)] for c in caches]
    want = p.compact(NB)
    pairs = DeviceArray.from_numpy(want[4])
    pa.copy_blocks(dev_caches[:2], dev_caches[2:], pairs, NB, Hkv, D, 16)
    synchronize()
    for c, rows in zip(dev_caches, before):
        c = c.numpy()
        for i, row in enumerate(rows):
            assert np.array_equal(c[p.h["tables"][i, :-(-p.h["ctx"][i] // 16)]], row)


def test_fork_in_a_graph(dev):
    """Two forks, there and back, replayed while the parents change."""
    rng = np.random.default_rng(5)
    S, stream = 24, Stream()
    p = Pool(S, 8, 300).lone(rng, rng.integers(0, 100, S))
    d = p.d

    def enqueue():
        p.enqueue_fork(stream=stream)
        pages.fork_pages(d["tables"], d["ctx"], d["other"], p.ctx_out, p.parents, d["refs"], d["free"], d["n"], p.pairs,
                         p.counts, p.ws, p.ws.nbytes, S, 8, 16, 300, stream=stream)

    g = Graph(stream, enqueue)
    h = p.h
    for _ in range(4):
        parents = rng.integers(-1, S, S).astype(np.int32)
        p.parents.upload(parents)
        synchronize()
        g.launch(stream)
        stream.synchronize()
        for a, b in (("tables", "other"), ("other", "tables")):
            want = oracle.fork_pages(h[b], h[a], h["ctx"], parents, h["refs"], h["free"], int(h["n"][0]))
            h[b], h["ctx"], h["refs"], h["free"], h["n"][0] = *want[:4], want[4]
        for k in ("tables", "other", "ctx", "refs", "free", "n"):
            assert np.array_equal(d[k].numpy(), h[k]), k
        assert np.array_equal(p.pairs.numpy(), want[5]) and np.array_equal(p.counts.numpy(), want[6])


@pytest.mark.parametrize("NB", [4096, 4097])
@pytest.mark.parametrize("S,MB", [(1, 4096), (1, 4097), (64, 64), (65, 64), (4096, 1)])
def test_forks_of_small_pools(dev, S, MB, NB):
    """At the sizes where one workgroup does all of it and where it does not."""
    rng = np.random.default_rng(S + MB)
    free = NB - 200
    lens = rng.integers(0, 16 * min(MB, max(free // S, 1)) + 1, S)
    if S > 1000:
        lens[rng.permutation(S)[:S - 3500]] = 0
    p = Pool(S, MB, NB).lone(rng, lens)
    for _ in range(4):
        p.fork(rng.integers(-1, S, S).astype(np.int32))


@pytest.mark.parametrize("NB", [1, 2, 3, 5, 4095, 4096, 4097, 65533, 65536, 65537])
@pytest.mark.parametrize("used", [0.0, 0.3, 0.97, 1.0])
def test_compactions_by_groups_of_ids(dev, NB, used):
    """Pools that end inside and at the edges of a group of ids, up to the most that every workgroup counts."""
    rng = np.random.default_rng(NB + int(10 * used))
    n = int(used * NB)
    lens = [16 * (n // 3), 16 * (n - n // 3) - (n > 1)] if n else [0, 0]
    for moves in (NB, max(NB // 50, 1)):
        p = Pool(2, max(n, 1), NB).lone(rng, lens)
        p.compact(moves)
