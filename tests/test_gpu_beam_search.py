"""A beam search as a server runs it: selection, fork and copies, the step's plan,
rotary positions, cache write and attention over what the beams share, in every
layer, step after step. Each array against the oracle (scores and choices as
test_gpu_beam_select, tables exactly, outputs by scored_bound on the cache and the
queries that the GPU made); and every row's values, read through its table, are
those that its own chain of tokens wrote, whichever rows it came of."""

import numpy as np
import pytest

import oracle
from step_helpers import normal, scored_bound, to_float
from swiftllm_amd import attention_step as step
from swiftllm_amd import beam_search as bs
from swiftllm_amd import paged_attention as pa
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu

SCORE_ERROR = 2.0 ** -17     # of a log softmax (test_gpu_beam_select), and a rounding to 32 bits


class Search:
    def __init__(self, rng, lens, W, vocab, MB, NB, H, Hkv, D, dtype, layers=2, eos=-1, common=0, **score):
        self.rng, self.R, self.W, self.V, self.MB, self.NB = rng, len(lens), W, vocab, MB, NB
        self.H, self.Hkv, self.D, self.dtype, self.eos = H, Hkv, D, dtype, eos
        self.S = S = self.R * W
        self.score = dict(scale=D ** -0.5, softcap=score.get("softcap", 0.0),
                          slopes=step.alibi_slopes(H) if score.get("alibi") else None)
        slopes = None if self.score["slopes"] is None else DeviceArray.from_numpy(self.score["slopes"])
        p = step.ScoreParams(self.score["scale"], self.score["softcap"], alibi_slopes=slopes)
        inv, self.factor = step.rotary_inv_freq(D)
        self.step = step.AttentionStep(S, S, MB, H, Hkv, D, p, inv, self.factor, dtype=dtype, num_groups=self.R)
        self.search = bs.BeamSearch(self.R, W, vocab, MB, NB, eos_id=eos)
        ids, at = rng.permutation(NB).astype(np.int32), common
        used = [-(-n // 16) for n in lens]
        bt = np.zeros((self.R, max(used)), np.int32)
        kc, vc = ([np.full((NB, Hkv, D, 16), 0x7FFF, np.uint16) for _ in range(layers)] for _ in range(2))
        for r, n in enumerate(used):
            m = min(common, n)
            bt[r, :n] = np.concatenate([ids[:m], ids[at:at + n - m]])
            at += n - m
        self.chains = [[[] for _ in range(S)] for _ in range(layers)]     # every row's values, [Hkv, D] a token
        for l in range(layers):
            for b in np.unique(np.concatenate([bt[r, :n] for r, n in enumerate(used)])):
                kc[l][b], vc[l][b] = (normal(rng, (Hkv, D, 16), dtype) for _ in range(2))
            for r, n in enumerate(lens):
                self.chains[l][r * W] = [vc[l][bt[r, t // 16], :, :, t % 16] for t in range(n)]
        self.caches = [[DeviceArray.from_numpy(x) for x in kv] for kv in zip(kc, vc)]
        self.row = (H + 2 * Hkv) * D
        self.d_logits = DeviceArray((S, vocab), np.float32)
        self.d_qkv = [DeviceArray((S, self.row), np.uint16) for _ in range(layers)]
        self.out = [DeviceArray((S, H, D), np.uint16) for _ in range(layers)]
        self.search.start(bt, np.array(lens))
        self.read()

    def read(self):
        s = self.search
        synchronize()
        self.bt, self.ctx, self.refs = s.block_tables.numpy(), s.context_lens.numpy()[:self.S], s.ref_counts.numpy()
        self.n = int(s.num_free.numpy()[0])
        self.free, self.scores = s.free_blocks.numpy(), s.scores.numpy()
        self.kv = [[c.numpy() for c in kv] for kv in self.caches]

    def inputs(self, banned=()):
        self.x = self.rng.standard_normal((self.S, self.V)).astype(np.float32) * 2
        self.x[:, list(banned)] = -np.inf
        self.d_logits.upload(self.x)
        self.qkv = [normal(self.rng, (self.S, self.row), self.dtype, 2.0) for _ in self.caches]
        for d, x in zip(self.d_qkv, self.qkv):
            d.upload(x)
        for o in self.out:
            o.fill_byte(0x7F)
        synchronize()

    def forked(self, stream=None):
        s = self.search
        s.select(self.d_logits, stream=stream)
        s.fork([k for k, _ in self.caches], [v for _, v in self.caches], self.Hkv, self.D, stream=stream)

    def layers(self, stream=None):
        self.search.plan(self.step, stream=stream)
        for (kc, vc), x, out in zip(self.caches, self.d_qkv, self.out):
            q, k, v = (x.ptr + 2 * self.D * n for n in (0, self.H, self.H + self.Hkv))
            self.step.layer(q, k, v, kc, vc, out, query_stride=self.row, key_stride=self.row, value_stride=self.row,
                            num_blocks=self.NB, decode=True, stream=stream)

    def check(self, taken):
        """The step just run, from the state of the last read(); what was taken since the fork before."""
        R, W, S, st, s = self.R, self.W, self.S, self.step, self.search
        before = (self.bt, self.ctx, self.refs, self.free, self.n)
        scores = self.scores
        # the selection
        C = s.num_candidates
        want = oracle.beam_select(self.x.reshape(R, W, -1), scores, C, self.eos)
        got = [a.numpy() for a in (s.cand_scores, s.cand_rows, s.cand_tokens, s.scores, s.next_rows, s.next_tokens)]
        for a, b in zip((0, 3), (0, 3)):
            some = np.isfinite(want[b])
            assert np.array_equal(np.isfinite(got[a]), some)
            err = np.abs(got[a][some] - want[b][some])
            assert (err <= SCORE_ERROR + 2.0 ** -24 * np.abs(want[b][some])).all()
        # (choices where no neighbour in the order is within both errors)
        more = oracle.beam_select(self.x.reshape(R, W, -1), scores, C + 1, self.eos)[0]
        with np.errstate(invalid="ignore"):
            near = -np.diff(more, axis=1) < 2 * (SCORE_ERROR + 2.0 ** -24 * np.abs(more[:, :-1]))
        clear = ~(near | np.pad(near, ((0, 0), (1, 0)))[:, :-1])
        for k in (1, 2):
            assert np.array_equal(got[k][clear], want[k][clear])
        for r in np.flatnonzero(clear.all(axis=1)):
            assert all(np.array_equal(got[k][r], want[k][r]) for k in (4, 5))
        assert clear.mean() > 0.5
        parents = got[4].reshape(S)
        # the fork: the tables before the step's plan come of the one before
        after = s.block_tables.numpy()
        free = s.free_blocks.numpy()
        bt, ctx, refs, left, n, pairs, counts = oracle.fork_pages(
            self.spare, before[0], before[1], parents, before[2], before[3], before[4], taken)
        assert np.array_equal(s.ref_counts.numpy(), refs) and np.array_equal(free[:n], left[:n])
        assert int(s.num_free.numpy()[0]) == n and np.array_equal(s.counts.numpy(), counts)
        assert np.array_equal(s.copy_pairs.numpy(), pairs)
        cut = ctx < np.where((parents >= 0) & (parents < S), before[1][parents], 0)
        new = np.where((parents >= 0) & ~cut, 1, 0)
        assert np.array_equal(s.new_lens.numpy(), new)
        # the step
        bt, now, off, pos, slots, took = oracle.plan_step(bt, ctx, new, left[:n], S, self.NB)
        assert np.array_equal(after, bt)
        for a, b in ((st.context_lens, now), (st.query_offsets, off), (st.positions, pos), (st.slot_mapping, slots),
                     (st.counts, took)):
            assert np.array_equal(a.numpy(), b)
        assert np.array_equal(st.shared_blocks.numpy(), oracle.shared_blocks(bt, now, np.arange(R + 1) * W))
        rows = int(off[-1])
        token = {i: off[i] for i in range(S) if off[i + 1] > off[i]}
        spare = before[0]
        self.read()
        self.spare = spare
        f = lambda x: to_float(x, self.dtype)  # noqa: E731
        for l, (x, out) in enumerate(zip(self.qkv, self.out)):
            v = x[:, (self.H + self.Hkv) * self.D:].reshape(S, self.Hkv, self.D)
            old = self.chains[l]
            self.chains[l] = [[] if p < 0 else old[p][:ctx[i]] for i, p in enumerate(parents)]
            for i, t in token.items():
                self.chains[l][i] = self.chains[l][i] + [v[t]]
            for i, chain in enumerate(self.chains[l]):
                assert len(chain) == now[i]
                have = [self.kv[l][1][bt[i, t // 16], :, :, t % 16] for t in range(now[i])]
                assert np.array_equal(np.array(have), np.array(chain)), f"layer {l} row {i}"
            assert (out.numpy()[rows:] == 0x7F7F).all()
        q = st.query.numpy().reshape(S, self.H, self.D)[:rows]
        a = (f(q), f(self.kv[-1][0]), f(self.kv[-1][1]), bt, now, off)
        want = oracle.scored_attention(*a, **self.score)
        bound = scored_bound(*a, self.dtype, 1, want, **self.score)
        err = np.abs(f(out.numpy()[:rows]) - want)
        assert (err <= bound).all(), f"{(err / bound).max():.2f} of the bound"
        return took, counts, parents

    def steps(self, n, taken=0, **kw):
        for _ in range(n):
            self.inputs(**kw)
            self.forked()
            self.layers()
            synchronize()
            took, counts, _ = self.check(taken)
            taken = int(took[0])
        return taken


def start(*a, **kw):
    s = Search(*a, **kw)
    s.spare = np.zeros((s.S, s.MB), np.int32)
    return s


@pytest.mark.parametrize("dtype,H,Hkv,D,score", [
    ("f16", 8, 2, 64, dict(softcap=20.0)), ("bf16", 4, 4, 128, dict()), ("f16", 16, 2, 128, dict(alibi=True))])
@pytest.mark.parametrize("W", [1, 3, 8])
def test_steps_of_a_search(dev, dtype, H, Hkv, D, score, W):
    """Prompts that end in every part of a block, two of them with common blocks;
    tables long and short enough for both ways through the attention."""
    rng = np.random.default_rng(100 * W + D + H)
    s = start(rng, [37, 48, 65, 1], W, 40, 60 if W == 3 else 8, 160, H, Hkv, D, dtype, eos=7, common=2, **score)
    s.steps(20)


def test_narrow_vocabulary_and_bans(dev):
    """Fewer tokens than beams: rows without a candidate end, the others' tokens
    move up, and later steps fill the beam again."""
    s = start(np.random.default_rng(3), [20, 33], 6, 4, 6, 60, 4, 2, 64, "f16")
    taken = s.steps(1, banned=[1, 3])
    assert (s.search.next_rows.numpy()[:, 2:] == -1).all()
    s.steps(4, taken=taken, banned=[2])
    assert (s.search.next_rows.numpy() >= 0).all()


def test_request_that_is_given_up(dev):
    """Its scores -inf: the blocks are free again, the others go on."""
    s = start(np.random.default_rng(4), [40, 50, 60], 4, 32, 8, 100, 4, 2, 64, "bf16")
    taken = s.steps(3)
    held = (s.refs > 0).sum()
    scores = s.scores.copy()
    scores[1] = -np.inf
    s.search.scores.upload(scores)
    s.read()
    s.steps(3, taken=taken)
    assert (s.refs > 0).sum() < held and (s.ctx.reshape(3, 4)[1] == 0).all()
    b = np.concatenate([s.bt[i, :-(-int(n) // 16)] for i, n in enumerate(s.ctx)])
    assert (np.bincount(b, minlength=s.NB) > 0).sum() <= (s.refs > 0).sum() + 12


def test_pool_that_runs_out(dev):
    """Rows without a block for their copy end with their whole blocks and are
    left out; rows without one for their next token are refused by the plan."""
    s = start(np.random.default_rng(5), [30, 30], 4, 32, 8, 7, 4, 2, 64, "f16")
    s.inputs()
    s.forked()
    s.layers()
    _, counts, _ = s.check(0)
    assert counts[1] > 0


def test_compacted_between_steps(dev):
    s = start(np.random.default_rng(6), [37, 90], 4, 32, 8, 300, 4, 2, 64, "f16")
    taken = s.steps(5)
    ids = DeviceArray((s.NB,), np.int32)
    for moves in (3, 300):
        s.inputs()
        s.forked()
        s.read()
        bt, refs, free, n, pairs, new_ids, counts = oracle.compact_pages(s.bt, s.ctx, s.refs, s.free, moves)
        before = s.bt
        s.search.compact([k for k, _ in s.caches], [v for _, v in s.caches], 2, 64, ids, moves)
        old = [[c.copy() for c in kv] for kv in s.kv]
        s.read()
        assert np.array_equal(s.refs, refs) and np.array_equal(ids.numpy(), new_ids)
        assert np.array_equal(s.free[:n], free[:n]) and s.n == n
        for i, c in enumerate(s.ctx):
            u = -(-int(c) // 16)
            assert np.array_equal(s.bt[i, :u], new_ids[before[i, :u]])
            for kv, was in zip(s.kv, old):
                for a, b in zip(kv, was):
                    assert np.array_equal(a[s.bt[i, :u]], b[before[i, :u]])
    assert max(s.bt[i, :-(-int(c) // 16)].max() for i, c in enumerate(s.ctx) if c) < (refs > 0).sum()
    assert taken >= 0


def test_two_steps_in_a_graph(dev):
    """The whole of two steps captured and replayed, beside a search of its own on
    another stream; each replay against eager steps of a search with the same
    inputs, bit by bit."""
    a, b, c = (start(np.random.default_rng(7), [37, 90, 16], 4, 32, 60, 200, 8, 2, 128, "f16", eos=3)
               for _ in range(3))
    stream, aside = Stream(), Stream()

    def both(s, stream):
        for _ in range(2):
            s.forked(stream)
            s.layers(stream)

    for s in (a, b, c):
        s.rng = np.random.default_rng(8)
        s.inputs()
        both(s, None)
    synchronize()
    g = Graph(stream, lambda: both(a, stream))
    for _ in range(5):
        for s in (a, b, c):
            s.inputs()
        g.launch(stream)
        both(c, aside)
        both(b, None)
        synchronize()
        for s in (a, c):
            for x, y in ((s.search, b.search), (s.step, b.step)):
                for k in ("scores", "cand_scores", "cand_rows", "cand_tokens", "next_rows", "next_tokens", "ref_counts",
                          "num_free", "copy_pairs", "counts", "new_lens", "block_tables", "context_lens", "positions",
                          "slot_mapping", "query_offsets", "shared_blocks"):
                    if hasattr(x, k):
                        assert np.array_equal(getattr(x, k).numpy(), getattr(y, k).numpy()), k
            for x, y in zip(s.out + sum(s.caches, []), b.out + sum(b.caches, [])):
                assert np.array_equal(x.numpy(), y.numpy())


def test_refusals(dev):
    s = start(np.random.default_rng(9), [20, 20], 2, 16, 4, 20, 4, 2, 64, "f16")
    se = s.search
    p = step.ScoreParams(0.1)
    for other in (step.AttentionStep(5, 5, 4, 4, 2, 64, p, np.ones(32)),
                  step.AttentionStep(4, 4, 5, 4, 2, 64, p, np.ones(32)),
                  step.AttentionStep(4, 4, 4, 4, 2, 64, p, np.ones(32), num_groups=1)):
        with pytest.raises(pa.InvalidParameter):
            se.plan(other)
    for tables, lens in (([[0, 1]], [20]), ([[0, 1], [2, 20]], [20, 20]), ([[0, 1], [2, -1]], [20, 20]),
                         ([[0], [1]], [17, 3]), ([[0], [1]], [16, -1]), (np.zeros((2, 5)), [1, 1])):
        with pytest.raises(pa.InvalidParameter):
            se.start(np.array(tables), np.array(lens))
    s.inputs()
    s.forked()
    s.layers()
    with pytest.raises(pa.InvalidParameter):
        se.plan(s.step)
    with pytest.raises(pa.InvalidParameter):
        se.compact([], [], 2, 64, DeviceArray((20,), np.int32), 3)
    with pytest.raises(pa.InvalidParameter):
        s.step.plan(se.block_tables, se.context_lens, se.new_lens, se.free_blocks, se.num_free, -1)
    for kw in (dict(num_requests=0), dict(beam_width=0), dict(num_blocks=0), dict(num_candidates=1)):
        with pytest.raises(pa.InvalidParameter):
            bs.BeamSearch(**{**dict(num_requests=2, beam_width=2, vocab=16, max_num_blocks_per_seq=4, num_blocks=20), **kw})
    for kw in (dict(beam_width=65), dict(dtype="f64"), dict(block_size=32)):
        with pytest.raises((pa.NotSupported, pa.InvalidParameter)):
            bs.BeamSearch(**{**dict(num_requests=2, beam_width=2, vocab=16, max_num_blocks_per_seq=4, num_blocks=20), **kw})


def test_groups_of_a_step(dev):
    """A step without group offsets decodes as one without groups; a window has none."""
    s = start(np.random.default_rng(10), [20, 20], 2, 16, 4, 20, 4, 2, 64, "f16")
    with pytest.raises(pa.NotSupported):
        step.AttentionStep(4, 4, 4, 4, 2, 64, step.ScoreParams(0.1, window=8), np.ones(32), num_groups=2)
    lone = step.AttentionStep(4, 4, 4, 4, 2, 64, step.ScoreParams(0.1), np.ones(32))
    se = s.search
    with pytest.raises(pa.InvalidParameter):
        lone.plan(se.block_tables, se.context_lens, se.new_lens, se.free_blocks, se.num_free, 20,
                  group_offsets=se.group_offsets)
    s.inputs()
    s.forked()
    s.layers()
    with_groups = s.out[0].numpy()
    synchronize()
    args = (se.block_tables, se._lens[se._now], DeviceArray.zeros((4,), np.int32), se.free_blocks, se.num_free, 20)
    x = s.d_qkv[0]
    q, k, v = (x.ptr + 2 * 64 * n for n in (0, 4, 6))
    plain = step.AttentionStep(4, 4, 4, 4, 2, 64, step.ScoreParams(s.score["scale"]), step.rotary_inv_freq(64)[0],
                               s.factor, num_groups=2)
    for st in (plain, s.step):
        st.plan(se.block_tables, args[1], se.new_lens, se.free_blocks, se.num_free, 20, num_blocks=20)
        s.out[0].fill_byte(0x7F)
        st.layer(q, k, v, *s.caches[0], s.out[0], query_stride=s.row, key_stride=s.row, value_stride=s.row,
                 num_blocks=20, decode=True)
        synchronize()
        f = to_float(s.out[0].numpy(), "f16")
        assert np.isfinite(f).all()
        # weights of 16 bits there (half a step of 2^-11 over and under the line), of two
        # parts here, and a rounding each: four half steps of the largest value, under 16
        assert np.abs(to_float(s.qkv[0], "f16")).max() < 16
        assert np.abs(f - to_float(with_groups, "f16")).max() <= 4 * 2.0 ** -11 * 16
