"""plan_step on the GPU against the oracle, exactly: block edges, empty
sequences, padding, more sequences than one chunk, and every refusal."""

import numpy as np
import pytest

import oracle
from swiftllm_amd import attention_step as step
from swiftllm_amd import _hip
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


def _tables(rng, cached, MB, pool):
    S = len(cached)
    ids = rng.permutation(pool).astype(np.int32)
    bt = np.full((S, MB), -7, np.int32)      # entries that nobody reads
    at = 0
    for s, c in enumerate(cached):
        n = min(-(-max(int(c), 0) // 16), MB)
        bt[s, :n] = ids[at:at + n]
        at += n
    return bt, ids[at:]


class Plan:
    def __init__(self, bt, cached, new, free, T, num_free=None, num_blocks=0):
        up = lambda x: DeviceArray.from_numpy(np.ascontiguousarray(x, np.int32))  # noqa: E731
        self.S, self.MB = bt.shape
        self.T, self.F, self.num_blocks = T, len(free), num_blocks
        self.bt, self.cached, self.new = up(bt), up(cached), up(new)
        self.free = up(free if len(free) else [0])
        self.nfree = up([len(free) if num_free is None else num_free])
        self.ctx, self.off = DeviceArray(max(self.S, 1), np.int32), DeviceArray(self.S + 1, np.int32)
        # one row more than asked for on each side of what is written
        self.pos, self.slots = DeviceArray(T + 1, np.int32), DeviceArray(T + 1, np.int32)
        self.counts = DeviceArray(3, np.int32)
        for d in (self.ctx, self.off, self.pos, self.slots, self.counts):
            d.fill_byte(0x55)

    def run(self, stream=None):
        step.plan_step(self.bt, self.cached, self.new, self.free, self.nfree, self.F, self.S,
                       self.MB, 16, self.T, self.ctx, self.off, self.pos, self.slots, self.counts,
                       num_blocks=self.num_blocks, stream=stream)

    def check(self, want):
        got = (self.bt.numpy(), self.ctx.numpy()[:self.S], self.off.numpy(),
               self.pos.numpy()[:self.T], self.slots.numpy()[:self.T], self.counts.numpy())
        for g, w, name in zip(got, want, ("tables", "context", "offsets", "positions", "slots", "counts")):
            assert np.array_equal(g, w), f"{name}: {np.flatnonzero(g.ravel() != w.ravel())[:8]}"
        assert self.pos.numpy()[self.T] == self.slots.numpy()[self.T] == 0x55555555


def _check(bt, cached, new, free, T, num_blocks=0, num_free=None):
    p = Plan(bt, cached, new, free, T, num_free, num_blocks)
    p.run()
    synchronize()
    n = len(free) if num_free is None else min(max(num_free, 0), len(free))
    want = oracle.plan_step(bt, cached, new, free[:n], T, num_blocks)
    p.check(want)
    return want


@pytest.mark.parametrize("S,most_cached,most_new,pad", [
    (1, 0, 1, 0), (1, 40, 300, 5), (5, 33, 17, 0), (64, 4000, 1, 0), (65, 300, 90, 1030),
    (300, 100, 40, 3), (1023, 20, 5, 0), (1025, 40, 9, 1), (2500, 30, 3, 2)])
def test_plan_matches_the_oracle(dev, S, most_cached, most_new, pad):
    rng = np.random.default_rng(S * 7 + pad)
    cached = rng.integers(0, most_cached + 1, S)
    new = rng.integers(0, most_new + 1, S)
    cached[rng.random(S) < 0.2] //= 16
    cached[rng.random(S) < 0.2] = cached[0] // 16 * 16
    MB = (most_cached + most_new) // 16 + 2
    pool = int((cached // 16 + 1).sum() + (new // 16 + 2).sum()) + 9
    bt, free = _tables(rng, cached, MB, pool)
    want = _check(bt, cached, new, free, int(new.sum()) + pad, num_blocks=pool)
    assert want[5][2] == 0


def test_plan_one_long_prompt_among_empty_ones(dev):
    """A sequence over many workgroups, between runs of sequences without tokens."""
    new = np.zeros(1500, np.int64)
    cached = np.full(1500, 16)
    new[[0, 700, 1400]] = [1, 70001, 2]
    cached[700] = 5
    bt, free = _tables(np.random.default_rng(1), cached, 4400, 12000)
    _check(bt, cached, new, free, int(new.sum()) + 100)


def test_plan_without_sequences_or_rows(dev):
    bt = np.zeros((0, 4), np.int32)
    _check(bt, [], [], np.arange(3), 70)
    _check(bt, [], [], np.arange(0), 0)
    bt, free = _tables(np.random.default_rng(2), [16, 3], 4, 20)
    _check(bt, [16, 3], [0, 0], free, 0)


@pytest.mark.parametrize("num_free", [0, 1, 4, 5, 6, 100, -3])
def test_plan_refuses_when_the_free_list_runs_out(dev, num_free):
    """Sequences that need no block go on being planned behind one whose
    blocks are missing; the count in device memory is bounded by the list."""
    cached = np.array([15, 16, 0, 31, 17, 32, 3])
    new = np.array([1, 1, 40, 1, 15, 17, 13])
    bt, free = _tables(np.random.default_rng(3), cached, 6, 60)
    want = _check(bt, cached, new, free[:7], int(new.sum()), num_free=num_free)
    assert want[5][2] == (0 if num_free >= 6 else want[5][2]) and (num_free >= 6 or want[5][2] > 0)


def test_plan_refuses_lengths_tables_and_rows(dev):
    """Negative lengths, a context past its table, the largest lengths there
    are, and more tokens than rows: refused one by one, the others planned."""
    big = 2 ** 31 - 1
    cached = np.array([4, -1, 4, 60, big, 0, 0, 64, 9])
    new = np.array([3, 2, -1, 5, big, big, 6, 0, 2])
    bt, free = _tables(np.random.default_rng(4), cached, 4, 400)
    want = _check(bt, cached, new, free, 20)
    assert want[5].tolist()[2] == 5
    want = _check(bt, cached, new, free, 10)     # the last sequence's rows do not fit
    assert want[5].tolist()[2] == 6


def test_plan_blocks_outside_the_pool_have_no_slot(dev):
    cached, new = np.array([20, 16, 0]), np.array([5, 3, 33])
    bt = np.array([[3, 99, 0, 0], [-1, 0, 0, 0], [0, 0, 0, 0]], np.int32)
    free = np.array([7, -2, 40, 2 ** 27], np.int32)
    _check(bt, cached, new, free, 50, num_blocks=50)
    _check(bt, cached, new, free, 50)


def test_plan_in_a_captured_graph(dev):
    """Replays follow what the buffers hold: the lengths of the step before
    become the cached ones, and the free list moves on."""
    rng = np.random.default_rng(5)
    S, MB, T = 70, 12, 400
    cached = rng.integers(0, 40, S)
    new = rng.integers(0, 6, S)
    bt, free = _tables(rng, cached, MB, 900)
    p = Plan(bt, cached, new, free, T)
    stream = Stream()
    p.run(stream)
    stream.synchronize()
    g = Graph(stream, lambda: p.run(stream))
    table = bt
    for _ in range(4):
        p.bt.upload(table)
        p.cached.upload(np.asarray(cached, np.int32))
        p.new.upload(np.asarray(new, np.int32))
        listed = np.concatenate([free, np.zeros(p.F - len(free), np.int32)]).astype(np.int32)
        p.free.upload(listed)
        p.nfree.upload(np.array([len(free)], np.int32))
        _hip.synchronize()
        g.launch(stream)
        stream.synchronize()
        want = oracle.plan_step(table, cached, new, free, T)
        p.check(want)
        table, cached, free = want[0], want[1], free[want[5][0]:]
        new = rng.integers(0, 6, S)


def test_plan_on_unaligned_outputs(dev):
    """Outputs at odd 4-byte offsets take the scalar stores."""
    cached, new = np.array([7, 0, 31]), np.array([9, 23, 2])
    bt, free = _tables(np.random.default_rng(6), cached, 6, 40)
    p = Plan(bt, cached, new, free, 40)
    pos, slots = DeviceArray(44, np.int32), DeviceArray(44, np.int32)
    step.plan_step(p.bt, p.cached, p.new, p.free, p.nfree, p.F, 3, 6, 16, 40, p.ctx, p.off,
                   pos.ptr + 4, slots.ptr + 12, p.counts)
    synchronize()
    want = oracle.plan_step(bt, cached, new, free, 40)
    assert np.array_equal(pos.numpy()[1:41], want[3])
    assert np.array_equal(slots.numpy()[3:43], want[4])
