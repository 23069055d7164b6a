"""scored_prefill on the GPU against the oracle in float64 (tolerance:
step_helpers.scored_bound, weights in one 16-bit part): caps, biases, windows
and prefixes, whole prompts and chunks on a cached context, both types, empty
and malformed sequences, garbage in every slot that nobody sees and values that
are not finite in slots that only later rows see."""

import numpy as np
import pytest

import oracle
from step_helpers import NAN16, normal, scored_bound, to_float, to_half
from swiftllm_amd import attention_step as step
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Prefill:
    def __init__(self, rng, new, H, Hkv, D, dtype, cached=None, cap=0.0, alibi=False, window=0,
                 prefix=None, scale=None, MB=None, lead=0, tail=3, qstd=3.0, spare=3):
        new = np.asarray(new)
        cached = np.zeros_like(new) if cached is None else np.asarray(cached)
        self.S, self.H, self.Hkv, self.D, self.dtype = len(new), H, Hkv, D, dtype
        self.ctx = (cached + new).astype(np.int32)
        self.off = (lead + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        self.T = int(self.off[-1]) + tail
        need = [-(-int(c) // 16) for c in self.ctx]
        self.MB = max(max(need, default=0), 1) if MB is None else MB
        self.NB = sum(need) + spare
        ids = rng.permutation(self.NB).astype(np.int32)
        self.bt = np.full((self.S, self.MB), 2 ** 31 - 1, np.int32)
        self.kc = np.full((self.NB, Hkv, D, 16), NAN16, np.uint16)
        self.vc = np.full((self.NB, Hkv, D, 16), NAN16, np.uint16)
        self.score = dict(scale=D ** -0.5 if scale is None else scale, softcap=cap, window=window,
                          slopes=step.alibi_slopes(H) if alibi else None,
                          prefix=None if prefix is None else np.asarray(prefix, np.int32))
        at = 0
        for s, n in enumerate(need):
            mine = ids[at:at + n]
            at += n
            self.bt[s, :n] = mine[:self.MB]
            low = max(int(cached[s]) + 1 - window, 0) if window else 0
            pre = 0 if prefix is None else int(prefix[s])
            for i, b in enumerate(mine):
                j = np.arange(16 * i, 16 * i + 16)
                t = np.flatnonzero((j < self.ctx[s]) & ((j >= low) | (j < pre)))
                self.kc[b][:, :, t] = normal(rng, (Hkv, D, t.size), dtype)
                self.vc[b][:, :, t] = normal(rng, (Hkv, D, t.size), dtype)
        self.q = normal(rng, (self.T, H, D), dtype, qstd)
        self.upload()

    def upload(self):
        up = DeviceArray.from_numpy
        self.d = {k: up(getattr(self, k)) for k in ("q", "kc", "vc", "bt", "ctx", "off")}
        sl, pre = self.score["slopes"], self.score["prefix"]
        self.d["slopes"] = None if sl is None else up(sl)
        self.d["prefix"] = None if pre is None else up(pre)
        self.out = DeviceArray((self.T, self.H, self.D), np.uint16)
        self.out.fill_byte(0x7F)

    def run(self, stream=None, bounded=True, out=None, q=None):
        p = step.ScoreParams(self.score["scale"], self.score["softcap"], self.score["window"],
                             self.d["slopes"], self.d["prefix"])
        step.scored_prefill(out or self.out, q or self.d["q"], self.d["kc"], self.d["vc"],
                            self.d["bt"], self.d["ctx"], self.d["off"], p, self.T, self.S, self.H,
                            self.Hkv, self.D, 16, self.MB, dtype=self.dtype,
                            num_blocks=self.NB if bounded else 0, stream=stream)

    def want(self):
        f = lambda x: to_float(x, self.dtype)  # noqa: E731
        a = (f(self.q), f(self.kc), f(self.vc), self.bt, self.ctx, self.off)
        with np.errstate(all="ignore"):
            w = oracle.scored_attention(*a, **self.score)
            return w, scored_bound(*a, self.dtype, 1, w, **self.score)

    def rows(self):
        """Which rows belong to a sequence."""
        mine = np.zeros(self.T, bool)
        for a, b in zip(self.off[:-1], self.off[1:]):
            if 0 <= a < b <= self.T:
                mine[a:b] = True
        return mine

    def check(self, what="", got=None):
        synchronize()
        got = self.out.numpy() if got is None else got
        mine = self.rows()
        assert (got[~mine] == 0x7F7F).all(), "rows of no sequence"
        got = to_float(got, self.dtype)[mine]
        want, bound = (x[mine] for x in self.want())
        assert np.isfinite(got).all(), f"{what}: not finite"
        err = np.abs(got - want)
        assert (err <= bound).all(), f"{what}: {(err / bound).max():.2f} of the bound, error {err.max():.2e}"


HEADS = [(8, 8, 64), (32, 8, 128), (64, 8, 128), (16, 16, 128), (40, 1, 64), (6, 2, 128), (1, 1, 64)]
LENS = [1, 15, 16, 17, 33, 64, 65, 130]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("score", [dict(), dict(cap=20.0), dict(alibi=True), dict(cap=30.0, alibi=True)])
def test_prefill_scores_and_heads(dev, H, Hkv, D, score, dtype):
    p = Prefill(np.random.default_rng(H + D), LENS, H, Hkv, D, dtype, **score)
    p.run()
    p.check(f"{H}/{Hkv}x{D} {score}")


@pytest.mark.parametrize("window", [1, 2, 16, 17, 63, 64, 65, 1000])
@pytest.mark.parametrize("prefix", [None, [0, 3, 16, 17, 40, 64, 65, 1]])
@pytest.mark.parametrize("shape", [dict(), dict(cap=25.0), dict(alibi=True), dict(cap=25.0, alibi=True)])
def test_prefill_windows_and_prefixes(dev, window, prefix, shape):
    p = Prefill(np.random.default_rng(window), LENS, 8, 2, 64, "f16", window=window, prefix=prefix, **shape)
    p.run()
    p.check(f"window {window} prefix {prefix}")


@pytest.mark.parametrize("prefix", [[200, 70, 500, 1], [64, 128, 0, 5]])
@pytest.mark.parametrize("shape", [dict(), dict(cap=25.0), dict(alibi=True), dict(cap=25.0, alibi=True)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prefill_prefix_both_ways(dev, prefix, shape, dtype):
    """Rows inside a prefix see keys ahead of them, by the two-sided distance."""
    p = Prefill(np.random.default_rng(1), [200, 300, 270, 5], 8, 2, 128, dtype, prefix=prefix, **shape)
    p.run()
    p.check()


@pytest.mark.parametrize("new,cached", [([1, 5, 70, 128], [300, 17, 64, 1000]), ([260], [1500]), ([3, 0, 40], [0, 50, 15])])
@pytest.mark.parametrize("kw", [dict(), dict(window=100, cap=15.0), dict(window=300, prefix=True, alibi=True)])
def test_prefill_chunks_on_a_cached_context(dev, new, cached, kw):
    kw = dict(kw)
    if kw.get("prefix"):
        kw["prefix"] = [70, 5, 130, 64][:len(new)]
    p = Prefill(np.random.default_rng(2), new, 8, 4, 64, "bf16", cached=cached, **kw)
    p.run()
    p.check(f"{new} on {cached}")


@pytest.mark.parametrize("H,Hkv,D", [(32, 8, 128), (16, 4, 64)])
@pytest.mark.parametrize("kw", [dict(), dict(cap=30.0), dict(window=700, prefix=[100, 64, 3], alibi=True)])
def test_prefill_long_prompts(dev, H, Hkv, D, kw):
    """Walks of more than one chunk of block ids (1024 keys), and jumps."""
    p = Prefill(np.random.default_rng(3), [2300, 1100, 5], H, Hkv, D, "f16", **kw)
    p.run()
    p.check()


@pytest.mark.parametrize("S", [65, 300, 1024, 1025, 2500])
def test_prefill_many_sequences(dev, S):
    """Tile lists in registers, in LDS, and past it in sequence order."""
    rng = np.random.default_rng(S)
    new = rng.integers(0, 7, S)
    new[[0, S // 2, S - 1]] = [0, 90, 33]
    p = Prefill(rng, new, 8, 2, 64, "f16", cached=rng.integers(0, 20, S), cap=10.0, window=25,
                prefix=rng.integers(0, 9, S))
    p.run()
    p.check(f"S {S}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0), dict(alibi=True), dict(cap=20.0, alibi=True, window=50)])
def test_prefill_workgroups_of_many_tiles(dev, D, kw):
    """More tiles of more sequences than stay on the GPU at once: a workgroup's
    next tile is another sequence's, shorter or longer."""
    rng = np.random.default_rng(D)
    p = Prefill(rng, rng.integers(0, 150, 90), 16, 16, D, "f16", cached=rng.integers(0, 70, 90), **kw)
    p.run()
    p.check(str(kw))


@pytest.mark.parametrize("S", [3, 1100])
def test_prefill_malformed_offsets_and_lengths(dev, S):
    """Offsets that run backwards or out of the rows have no rows; contexts
    shorter than the chunk leave rows before position 0 that see nothing;
    lengths past the table end there."""
    rng = np.random.default_rng(4)
    p = Prefill(rng, [40, 20, 30] + [1] * (S - 3), 8, 2, 64, "f16", alibi=True, lead=5)
    p.ctx[:3] = [25, -4, 0]
    p.upload()
    p.run()
    p.check("short contexts")
    got = p.out.numpy()
    assert (got[5:20] == 0).all() and (got[45:95] == 0).all()
    p = Prefill(rng, [40, 20, 30] + [1] * (S - 3), 8, 2, 64, "f16", lead=5)
    p.off[1:3] = [p.T + 1, 50]
    p.ctx[2] = 30 + 65 - 50 + 16      # offsets 50 .. 95: a longer chunk of it
    p.ctx[2] = min(p.ctx[2], 30)
    p.upload()
    p.run()
    p.check("offsets")


def test_prefill_context_past_the_table(dev):
    p = Prefill(np.random.default_rng(5), [40, 16], 8, 2, 64, "f16", cap=20.0)
    p.MB = 2
    p.bt = np.ascontiguousarray(p.bt[:, :2])
    p.upload()
    p.run()
    p.check()


def test_prefill_prefixes_out_of_range(dev):
    p = Prefill(np.random.default_rng(6), [40, 20, 33], 8, 2, 64, "bf16", window=5, prefix=[0, 20, 33])
    p.score["prefix"] = np.array([-7, 1 << 30, 2 ** 31 - 1], np.int32)
    p.upload()
    p.run()
    p.check()


def test_prefill_blocks_outside_the_pool(dev):
    p = Prefill(np.random.default_rng(7), [100, 64, 300], 8, 2, 64, "f16", cap=30.0)
    p.bt[0, [0, 3]] = [-1, p.NB]
    p.bt[1, :4] = [-5, 1 << 30, -(1 << 31), p.NB]
    p.bt[2, [5, 17]] = -1
    p.upload()
    p.run()
    p.check()
    assert (p.out.numpy()[100:164] == 0).all()
    p.bt[(p.bt >= p.NB)] = -2
    p.upload()
    p.run(bounded=False)
    p.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0), dict(alibi=True), dict(window=40), dict(window=40, prefix=[3, 70])])
def test_prefill_values_that_are_not_finite(dev, dtype, kw):
    """NaN and infinite keys and values at single tokens: rows that do not see
    them are untouched (causality, window), rows that do are not finite."""
    inf = {"f16": 0x7C00, "bf16": 0x7F80}[dtype]
    p = Prefill(np.random.default_rng(8), [150, 200], 8, 2, 64, dtype, **kw)
    bad = [(0, 70, 0, "k", NAN16), (0, 77, 1, "v", NAN16), (1, 30, 0, "v", inf), (1, 130, 0, "v", inf | 0x8000),
           (1, 190, 1, "k", NAN16)]
    for s, j, kvh, which, x in bad:
        getattr(p, which + "c")[p.bt[s, j // 16], kvh, 9, j % 16] = x
    p.upload()
    p.run()
    synchronize()
    got = to_float(p.out.numpy(), dtype)
    want, bound = p.want()
    mine = p.rows()
    touched = np.zeros((p.T, 8), bool)
    window = p.score["window"] or 10 ** 9
    for s, j, kvh, which, x in bad:
        pos = np.arange(p.ctx[s])
        sees = (j <= pos) & (pos - j < window)
        if p.score["prefix"] is not None:
            sees |= j < p.score["prefix"][s]
        touched[p.off[s]:p.off[s + 1], 4 * kvh:4 * kvh + 4] |= sees[:, None]
    clean = mine[:, None] & ~touched
    assert np.isfinite(got[clean]).all()
    assert (np.abs(got[clean] - want[clean]) <= bound[clean]).all()
    assert not np.isfinite(got[mine[:, None] & touched]).all(axis=-1).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_prefill_large_scores(dev, dtype, cap):
    p = Prefill(np.random.default_rng(9), [200, 77], 8, 2, 128, dtype, cap=cap, qstd=100.0)
    p.run()
    p.check()


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
@pytest.mark.parametrize("kw", [dict(), dict(cap=9.0), dict(alibi=True), dict(cap=9.0, alibi=True, window=20)])
def test_prefill_scales(dev, scale, kw):
    p = Prefill(np.random.default_rng(10), [90, 5], 8, 2, 64, "f16", scale=scale, qstd=1.0, **kw)
    p.run()
    p.check()


def test_prefill_query_and_output_8_byte_aligned(dev):
    p = Prefill(np.random.default_rng(11), [70, 20], 8, 2, 128, "f16", cap=20.0)
    n = p.q.nbytes
    q, out = DeviceArray((n + 16,), np.uint8), DeviceArray((n + 16,), np.uint8)
    q.upload_at(8, p.q)
    out.fill_byte(0x7F)
    p.run(q=q.ptr + 8, out=out.ptr + 8)
    synchronize()
    p.check(got=out.download_at(8, p.q.shape, np.uint16))


@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (40, 1, 128)])
def test_prefill_into_the_queries(dev, H, Hkv, D):
    """output may be query; rows of no sequence stay."""
    p = Prefill(np.random.default_rng(13), [1, 150, 33], H, Hkv, D, "f16", cached=[40, 3, 0], cap=20.0, tail=0)
    p.out.upload(p.q)
    p.run(q=p.out)
    p.check("in place")
    p = Prefill(np.random.default_rng(14), [5], H, Hkv, D, "f16", lead=4, tail=7)
    p.run(q=p.d["q"], out=p.d["q"])
    synchronize()
    got = p.d["q"].numpy()
    assert np.array_equal(got[:4], p.q[:4]) and np.array_equal(got[9:], p.q[9:])


def test_prefill_rows_that_sequences_share(dev):
    """Offsets that run back and forth make rows of several sequences: the
    output is unspecified, but the call ends and writes within its rows."""
    p = Prefill(np.random.default_rng(15), [7] * 70, 8, 2, 64, "f16", cached=[9] * 70)
    good = p.off.copy()
    p.off[1:40] = [0, 200] * 19 + [0]
    p.upload()
    p.run()
    synchronize()
    assert (p.out.numpy()[490:] == 0x7F7F).all()
    p.off = good
    p.d["off"].upload(good)
    p.out.fill_byte(0x7F)
    p.run()
    p.check("separate rows")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(cap=1000.0), dict(window=30000)])
def test_prefill_sums_small_weights(dev, dtype, kw):
    """Some 20000 keys 22 binary places below the largest: their weights are
    below fp16's normal range and count, in the sum as in the output. Of values
    of 1 the output is 1: every weight is rounded to a power of two and every sum
    exact (with a cap the scores are off by under 2^-11, the same for all of
    those keys), so only the last division and the rounding to the type are left.
    Of a 0 for the largest it is their share: off by half a step of their weight
    (2^-10 of it in fp16, 2^-9 in bf16), of the output's, and of the cap."""
    p = Prefill(np.random.default_rng(16), [40], 2, 1, 64, dtype, cached=[19970], scale=1.0, tail=0, **kw)
    p.kc[:], p.vc[:], p.q[:] = 0, to_half(np.ones(1), dtype)[0], 0
    p.kc[p.bt[0, 0], 0, 0, 0] = to_half(np.array([15.25]), dtype)[0]     # 22 / log2(e)
    p.q[:, :, 0] = to_half(np.ones(1), dtype)[0]
    p.upload()
    p.run()
    synchronize()
    got = to_float(p.out.numpy(), dtype)
    assert (np.abs(got - 1.0) <= 2.0 ** (-11 if dtype == "f16" else -8)).all(), np.abs(got - 1).max()
    p.vc[p.bt[0, 0], 0, :, 0] = 0
    p.d["vc"].upload(p.vc)
    p.run()
    synchronize()
    got = to_float(p.out.numpy(), dtype)
    top = 1000 * np.tanh(0.01525) if "cap" in kw else 15.25
    n = 19970 + np.arange(40)[:, None, None]      # keys behind the first that row t sees
    want = n / (n + np.exp(top))
    assert (np.abs(got / want - 1) <= 2.0 ** (-8 if dtype == "f16" else -7)).all(), np.abs(got / want - 1).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0), dict(alibi=True)])
def test_prefill_a_query_that_is_not_finite(dev, dtype, kw):
    """It makes NaN of its own row and head and of no other."""
    p = Prefill(np.random.default_rng(17), [70, 20], 8, 2, 64, dtype, **kw)
    want, bound = p.want()
    for t, h in ((0, 0), (33, 5), (75, 7)):
        p.q[t, h, 11] = NAN16
    p.upload()
    p.run()
    synchronize()
    got, mine = to_float(p.out.numpy(), dtype), p.rows()
    bad = np.zeros(got.shape[:2], bool)
    bad[0, 0] = bad[33, 5] = bad[75, 7] = True
    assert np.isnan(got[bad]).all()
    fine = mine[:, None] & ~bad
    assert (np.abs(got - want)[fine] <= bound[fine]).all()


def test_prefill_nothing_to_do(dev):
    p = Prefill(np.random.default_rng(12), [0, 0], 8, 2, 64, "f16", tail=20)
    p.run()
    p.check()


def test_prefill_in_a_captured_graph(dev):
    """Replays follow offsets and lengths in the buffers, padded rows behind."""
    rng = np.random.default_rng(13)
    p = Prefill(rng, [60, 40, 30], 8, 2, 64, "f16", cached=[20, 0, 100], window=50, cap=20.0, tail=70)
    p.kc[:], p.vc[:] = normal(rng, p.kc.shape, "f16"), normal(rng, p.vc.shape, "f16")
    p.upload()
    stream = Stream()
    p.run(stream)
    stream.synchronize()
    g = Graph(stream, lambda: p.run(stream))
    for new, ctx in (([60, 40, 30], [80, 40, 130]), ([1, 0, 1], [81, 33, 128]), ([10, 64, 90], [10, 64, 129])):
        p.off = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        p.ctx = np.asarray(ctx, np.int32)
        need = -(-p.ctx // 16)
        p.bt = np.where(np.arange(p.MB)[None] < need[:, None], rng.permutation(p.NB)[:p.MB][None], 0).astype(np.int32)
        p.d["off"].upload(p.off)
        p.d["ctx"].upload(p.ctx)
        p.d["bt"].upload(p.bt)
        p.out.fill_byte(0x7F)
        synchronize()
        g.launch(stream)
        stream.synchronize()
        p.check(f"{new}")


def _with_offsets(rng, S, off, T, **kw):
    """S sequences of rows off[s] .. off[s + 1] - 1 of T, their whole contexts in the cache."""
    off = np.asarray(off)
    n = off[1:] - off[:-1]
    n[(off[:-1] < 0) | (off[1:] > T)] = 0
    p = Prefill(rng, np.maximum(n, 0), 8, 8, 64, "f16", tail=0, **kw)
    p.off, p.T = off.astype(np.int32), T
    p.q = normal(rng, (T, 8, 64), "f16", 3.0)
    p.upload()
    return p


def test_prefill_offsets_in_any_order(dev):
    """More than 1024 sequences whose offsets go back and forth within the rows:
    the rows of two of them, and a sequence between without any."""
    S = 1100
    off = np.full(S + 1, 1280)
    off[:4] = [1280, 2560, 0, 1280]
    p = _with_offsets(np.random.default_rng(18), S, off, 2560, window=50)
    p.run()
    assert p.rows().all()
    p.check()


@pytest.mark.parametrize("S", [1000, 1100])
@pytest.mark.parametrize("at", [275, 550, 825])
@pytest.mark.parametrize("bad", [-1, -(1 << 31), 1109, 10 ** 6, 2 ** 31 - 1])
def test_prefill_one_bad_offset_among_many(dev, S, at, bad):
    """It takes the rows of the two sequences that it belongs to and no other."""
    off = 3 + np.arange(S + 1)
    off[at] = bad
    p = _with_offsets(np.random.default_rng(19), S, off, S + 8)
    p.run()
    assert p.rows().sum() == S - 2
    p.check()


@pytest.mark.parametrize("S", [1025, 4096, 4097, 20000, 65535])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (8, 1), (3, 1)])
def test_prefill_few_tokens_among_many_sequences(dev, S, H, Hkv):
    """Mostly sequences without tokens, with one or two tiles or more at either end and at random."""
    rng = np.random.default_rng(S)
    new = np.zeros(S, np.int64)
    new[rng.choice(S, 100, replace=False)] = rng.integers(1, 40, 100)
    new[[0, 63, 64, S - 1]] = [130, 1, 300, 65]
    p = Prefill(rng, new, H, Hkv, 64, "bf16", cap=20.0, lead=3)
    p.run()
    p.check(f"S {S}")


@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0), dict(alibi=True), dict(window=70, prefix=[40, 3, 1])])
@pytest.mark.parametrize("D", [64, 128])
def test_prefill_of_large_values(dev, kw, D):
    """bfloat16 has values near 2^128: a weighted mean of values of 2^116, at
    most 2^121 of them, is a number like any other."""
    p = Prefill(np.random.default_rng(20), [150, 64, 1], 8, 2, D, "bf16", cached=[70, 0, 0], **kw)
    hidden = p.vc == NAN16
    p.vc = np.where(hidden, p.vc, normal(np.random.default_rng(21), p.vc.shape, "bf16", 2.0 ** 116))
    p.upload()
    p.run()
    p.check()


def test_prefill_of_the_largest_value(dev):
    """One key: its value, whatever it is."""
    p = Prefill(np.random.default_rng(22), [1, 1], 8, 2, 64, "bf16", tail=0)
    top = to_half(np.array([2.0 ** 127 * (2 - 2.0 ** -7)]), "bf16")[0]
    for s in range(2):
        p.vc[p.bt[s, 0], :, :, 0] = top if s == 0 else top | 0x8000
    p.upload()
    p.run()
    synchronize()
    got = p.out.numpy()
    assert (got[0] == top).all() and (got[1] == (top | 0x8000)).all()


@pytest.mark.parametrize("kw", [dict(cap=0.0), dict(cap=1e-39), dict(cap=1e-39, alibi=True), dict(cap=20.0)])
def test_prefill_scale_of_zero(dev, kw):
    """Every key counts the same but for its bias, whatever the cap."""
    p = Prefill(np.random.default_rng(23), [90, 5], 8, 2, 64, "f16", scale=0.0, **kw)
    p.run()
    p.score["softcap"] = 0.0
    p.check()


@pytest.mark.parametrize("S", [3, 70, 1100])
@pytest.mark.parametrize("ctx", [-(1 << 31), -(1 << 31) + 20, -1])
def test_prefill_lengths_far_below_zero(dev, S, ctx):
    """Their rows are zero, and the sum of a length and a row count stays a number."""
    p = Prefill(np.random.default_rng(24), [40, 300] + [2] * (S - 2), 8, 2, 64, "f16", alibi=True, window=9,
                prefix=[4] * S)
    p.ctx[[1, S - 1]] = ctx
    p.upload()
    p.run()
    p.check()
    assert (p.out.numpy()[p.off[1]:p.off[2]] == 0).all()
