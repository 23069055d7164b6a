"""The attention step's operators as a server runs them together: plan, then
rotary + cache write + attention in each layer, over mixed steps, decode steps,
refused sequences, and captured in a graph. Every array against the oracle:
plans exactly, keys in the cache to their rounding, outputs by scored_bound on
the cache and queries that the GPU itself made."""

import numpy as np
import pytest

import oracle
from step_helpers import HALF_STEP, normal, scored_bound, to_float
from swiftllm_amd import attention_step as step
from swiftllm_amd import paged_attention as pa
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Server:
    """Sequences over a pool; device arrays of the step's inputs."""

    def __init__(self, rng, S, T, MB, NB, H, Hkv, D, dtype, score, rot, layers=2, **kw):
        self.rng, self.S, self.T, self.MB, self.NB = rng, S, T, MB, NB
        self.H, self.Hkv, self.D, self.dtype, self.score = H, Hkv, D, dtype, score
        self.inv, self.factor = step.rotary_inv_freq(rot, 10000.0, "yarn", factor=4.0, original_context=256)
        self.inter = kw.get("interleaved", False)
        up = DeviceArray.from_numpy
        self.slopes, self.prefix = score.get("slopes"), score.get("prefix")
        p = step.ScoreParams(score["scale"], score.get("softcap", 0.0), score.get("window", 0),
                             None if self.slopes is None else up(self.slopes),
                             None if self.prefix is None else up(self.prefix))
        self.step = step.AttentionStep(S, T, MB, H, Hkv, D, p, self.inv, self.factor, dtype=dtype, **kw)
        self.bt = np.zeros((S, MB), np.int32)
        self.cached = np.zeros(S, np.int32)
        self.free = rng.permutation(NB).astype(np.int32)
        self.cap = len(self.free)
        self.d = {"bt": up(self.bt), "cached": up(self.cached), "new": DeviceArray(S, np.int32),
                  "free": DeviceArray(self.cap, np.int32), "num_free": DeviceArray(1, np.int32)}
        self.caches = [[up(np.full((NB, Hkv, D, 16), 0x7FFF, np.uint16)) for _ in range(2)] for _ in range(layers)]
        self.row = (H + 2 * Hkv) * D
        self.d["qkv"] = [DeviceArray((T, self.row), np.uint16) for _ in range(layers)]
        self.out = [DeviceArray((T, H, D), np.uint16) for _ in range(layers)]

    def inputs(self, new):
        self.new = np.asarray(new, np.int32)
        self.qkv = [normal(self.rng, (self.T, self.row), self.dtype, 2.0) for _ in self.caches]
        for d, x in zip(self.d["qkv"], self.qkv):
            d.upload(x)
        for o in self.out:
            o.fill_byte(0x7F)
        self.d["cached"].upload(self.cached)
        self.d["new"].upload(self.new)
        self.d["free"].upload(np.concatenate([self.free, np.zeros(self.cap - len(self.free), np.int32)]).astype(np.int32))
        self.d["num_free"].upload(np.array([len(self.free)], np.int32))
        synchronize()

    def enqueue(self, decode, stream=None):
        d = self.d
        self.step.plan(d["bt"], d["cached"], d["new"], d["free"], d["num_free"], self.cap,
                       num_blocks=self.NB, stream=stream)
        for (kc, vc), x, out in zip(self.caches, d["qkv"], self.out):
            q, k, v = (x.ptr + 2 * self.D * n for n in (0, self.H, self.H + self.Hkv))
            self.step.layer(q, k, v, kc, vc, out, query_stride=self.row, key_stride=self.row,
                            value_stride=self.row, num_blocks=self.NB, decode=decode, stream=stream)

    def check(self):
        """The step just run, and the state that it leaves."""
        st = self.step
        bt, ctx, off, pos, slots, counts = oracle.plan_step(self.bt, self.cached, self.new, self.free, self.T, self.NB)
        assert np.array_equal(self.d["bt"].numpy(), bt)
        for got, want in ((st.context_lens, ctx), (st.query_offsets, off), (st.positions, pos),
                          (st.slot_mapping, slots), (st.counts, counts)):
            assert np.array_equal(got.numpy(), want)
        n = int(off[-1])
        f = lambda x: to_float(x, self.dtype)  # noqa: E731
        for (kc, vc), x, out in zip(self.caches, self.qkv, self.out):
            kc, vc = kc.numpy(), vc.numpy()
            k = x[:n, self.H * self.D:(self.H + self.Hkv) * self.D].reshape(n, self.Hkv, self.D)
            v = x[:n, (self.H + self.Hkv) * self.D:].reshape(n, self.Hkv, self.D)
            b, o = slots[:n] // 16, slots[:n] % 16
            assert np.array_equal(vc[b, :, :, o], v)
            want = oracle.rotary(f(k), pos[:n], self.inv, 2 * len(self.inv), self.inter, self.factor)
            err = np.abs(f(kc[b, :, :, o]) - want)
            assert (err <= HALF_STEP[self.dtype] * np.abs(want) + 2.0 ** -18 * self.factor * np.abs(f(k)).max()).all()
            got = out.numpy()
            assert (got[n:] == 0x7F7F).all()
        # the queries of the last layer are still there
        q = st.query.numpy().reshape(self.T, self.H, self.D)
        a = (f(q[:n]), f(kc), f(vc), bt, ctx, off)
        score = {k: s for k, s in self.score.items()}
        want = oracle.scored_attention(*a, **score)
        bound = scored_bound(*a, self.dtype, 1, want, **score)
        err = np.abs(f(got[:n]) - want)
        assert (err <= bound).all(), f"{(err / bound).max():.2f} of the bound"
        self.bt, self.cached, self.free = bt, ctx, self.free[counts[0]:]
        return counts


SCORES = [dict(scale=0.09, softcap=30.0), dict(scale=0.09, window=40, slopes=True, prefix=True),
          dict(scale=0.12, softcap=20.0, window=64)]


def _score(rng, S, H, score):
    score = dict(score)
    if score.get("slopes"):
        score["slopes"] = step.alibi_slopes(H)
    if score.get("prefix"):
        score["prefix"] = rng.integers(0, 30, S).astype(np.int32)
    return score


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("H,Hkv,D,rot,dtype,inter", [(8, 2, 128, 128, "bf16", False), (4, 4, 64, 32, "f16", True)])
def test_steps_of_a_server(dev, H, Hkv, D, rot, dtype, inter, score):
    """Prompts come in whole and in chunks beside decoding sequences, then all decode."""
    rng = np.random.default_rng(D + rot)
    S = 7
    s = Server(rng, S, 160, 24, 130, H, Hkv, D, dtype, _score(rng, S, H, score), rot, interleaved=inter)
    for new in ([50, 1, 33, 0, 16, 0, 0], [1, 64, 31, 0, 1, 17, 0], [1, 40, 1, 100, 1, 1, 0]):
        s.inputs(new)
        s.enqueue(False)
        synchronize()
        assert s.check()[2] == 0
    for new in ([1] * 7, [1, 1, 0, 1, 1, 1, 1], [1] * 7):
        s.inputs(new)
        s.enqueue(True)
        synchronize()
        assert s.check()[2] == 0


def test_step_with_refused_sequences(dev):
    """The free list runs out: sequences that need a block stay as they are and
    the rows of the others move up, in prefill and in decode steps."""
    rng = np.random.default_rng(5)
    s = Server(rng, 5, 120, 8, 9, 8, 2, 64, "f16", dict(scale=0.1, softcap=10.0), 64)
    s.inputs([16, 40, 31, 0, 15])       # 1 + 3 + 2 + 1 of 9 blocks
    s.enqueue(False)
    synchronize()
    assert s.check().tolist() == [7, 102, 0]
    s.inputs([1, 9, 1, 33, 1])          # one block, one, none, three, none
    s.enqueue(False)
    synchronize()
    assert s.check().tolist() == [2, 12, 1]
    s.inputs([1, 1, 1, 1, 1])           # sequences 2, 3 and 4 need a block
    s.enqueue(True)
    synchronize()
    assert s.check().tolist() == [0, 2, 3]


def test_decode_step_in_a_captured_graph(dev):
    """One graph of a whole decode step, replayed while sequences grow, join and end."""
    rng = np.random.default_rng(6)
    s = Server(rng, 6, 8, 12, 60, 8, 2, 64, "bf16", dict(scale=0.1, softcap=30.0, window=50), 64)
    stream = Stream()
    s.inputs([1, 1, 0, 0, 0, 0])
    s.enqueue(True, stream)
    stream.synchronize()
    s.check()
    s.inputs([0] * 6)
    g = Graph(stream, lambda: s.enqueue(True, stream))
    for i in range(20):
        new = np.ones(6, np.int32)
        new[3:] = i >= 5
        if i == 12:
            s.cached[1] = 0             # a sequence ends; its blocks stay with its row
            new[1] = 0
        s.inputs(new)
        g.launch(stream)
        stream.synchronize()
        s.check()


def test_step_refuses(dev):
    with pytest.raises(pa.InvalidParameter):
        step.AttentionStep(2, 4, 4, 4, 2, 64, step.ScoreParams(0.1), np.ones(40))
    with pytest.raises(pa.NotSupported):
        step.AttentionStep(2, 4, 4, 4, 2, 64, step.ScoreParams(0.1), np.ones(32), dtype="f32")
    s = step.AttentionStep(2, 4, 4, 4, 2, 64, step.ScoreParams(0.1), np.ones(32))
    with pytest.raises(pa.InvalidParameter):
        s.layer(0, 0, 0, 0, 0, 0)


def _check_layers(s, decode):
    """Layer after layer: the rotated queries against the oracle's of the host's
    inputs, and the outputs against the oracle's of those queries and the
    layer's own cache; then the whole step once more, to the same bits."""
    d, st = s.d, s.step
    f = lambda x: to_float(x, s.dtype)  # noqa: E731
    st.plan(d["bt"], d["cached"], d["new"], d["free"], d["num_free"], s.cap, num_blocks=s.NB)
    bt, ctx, off, pos, _, _ = oracle.plan_step(s.bt, s.cached, s.new, s.free, s.T, s.NB)
    n, half = int(off[-1]), len(s.inv)
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if s.inter else (i, i + half)
    last = np.zeros(s.T, bool)
    last[off[1:][off[1:] > off[:-1]] - 1] = True
    outs = []
    for (kc, vc), x, dx, out in zip(s.caches, s.qkv, d["qkv"], s.out):
        q, k, v = (dx.ptr + 2 * s.D * h for h in (0, s.H, s.H + s.Hkv))
        st.layer(q, k, v, kc, vc, out, query_stride=s.row, key_stride=s.row, value_stride=s.row,
                 num_blocks=s.NB, decode=decode)
        synchronize()
        mine = x[:n, :s.H * s.D].reshape(n, s.H, s.D)
        want = oracle.rotary(f(mine), pos[:n], s.inv, 2 * half, s.inter, s.factor)
        size = np.zeros((n, s.H, s.D))
        size[..., first] = size[..., second] = np.abs(f(mine))[..., first] + np.abs(f(mine))[..., second]
        q = st.query.numpy().reshape(s.T, s.H, s.D)
        err = np.abs(f(q[:n]) - want)
        assert (err <= HALF_STEP[s.dtype] * np.abs(want) + 2.0 ** -19 * s.factor * size).all(), "queries"
        a = (f(q[:n]), f(kc.numpy()), f(vc.numpy()), bt, ctx, off)
        want = oracle.scored_attention(*a, **s.score)
        bound = scored_bound(*a, s.dtype, 2 if decode else 1, want, **s.score)
        got = out.numpy()
        err = np.abs(f(got[:n]) - want)
        rows = last[:n] if decode else np.ones(n, bool)
        assert (err <= bound)[rows].all(), f"{(err / bound)[rows].max():.2f} of the bound"
        outs.append(got)
    for o in s.out:
        o.fill_byte(0x7F)
    s.enqueue(decode)
    synchronize()
    for o, want in zip(s.out, outs):
        assert np.array_equal(o.numpy(), want)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("H,Hkv,D,rot,dtype,inter", [(8, 2, 128, 128, "bf16", False), (4, 4, 64, 32, "f16", True),
                                                     (6, 1, 64, 64, "bf16", False), (16, 2, 128, 64, "f16", True)])
def test_every_layer_of_a_step(dev, H, Hkv, D, rot, dtype, inter, score):
    """Queries and outputs of all three layers, in mixed steps and in decode
    steps, one of them with long contexts beside short ones. (The second step has
    614 tokens for 600 rows: its last sequence is refused.)"""
    rng = np.random.default_rng(H + rot)
    S = 6
    s = Server(rng, S, 600, 80, 420, H, Hkv, D, dtype, _score(rng, S, H, score), rot, layers=3, interleaved=inter)
    for new, decode, refused in (([500, 1, 33, 0, 16, 0], False, 0), ([1, 64, 31, 500, 1, 17], False, 1),
                                 ([1, 1, 40, 1, 1, 0], False, 0), ([1] * 6, True, 0), ([1, 0, 1, 1, 0, 1], True, 0)):
        s.inputs(new)
        _check_layers(s, decode)
        assert s.check()[2] == refused
