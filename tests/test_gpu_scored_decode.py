"""scored_decode on the GPU against the oracle in float64 (tolerance:
step_helpers.scored_bound): caps, biases, windows and prefixes around block
edges, both types, short and split contexts, empty and malformed sequences,
garbage in every slot that nobody sees."""

import numpy as np
import pytest

import oracle
from step_helpers import NAN16, normal, scored_bound, to_float, to_half
from swiftllm_amd import attention_step as step
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Decode:
    def __init__(self, rng, ctx, H, Hkv, D, dtype, cap=0.0, alibi=False, window=0, prefix=None,
                 MB=None, scale=None, spare=3, qstd=3.0):
        self.ctx = np.asarray(ctx, np.int32)
        self.S, self.H, self.Hkv, self.D, self.dtype = len(ctx), H, Hkv, D, dtype
        need = [-(-max(int(c), 0) // 16) for c in ctx]
        self.MB = max(max(need), 1) if MB is None else MB
        self.NB = sum(need) + spare
        ids = rng.permutation(self.NB).astype(np.int32)
        self.bt = np.full((self.S, self.MB), 2 ** 31 - 1, np.int32)   # nobody reads these
        self.kc = np.full((self.NB, Hkv, D, 16), NAN16, np.uint16)
        self.vc = np.full((self.NB, Hkv, D, 16), NAN16, np.uint16)
        at = 0
        self.score = dict(scale=D ** -0.5 if scale is None else scale, softcap=cap, window=window,
                          slopes=step.alibi_slopes(H) if alibi else None,
                          prefix=None if prefix is None else np.asarray(prefix, np.int32))
        for s, n in enumerate(need):
            mine = ids[at:at + n]
            at += n
            self.bt[s, :n] = mine[:self.MB]
            for i, b in enumerate(mine):
                # only what the query sees is a number
                j = np.arange(16 * i, 16 * i + 16)
                seen = j < self.ctx[s]
                if window:
                    seen &= j > self.ctx[s] - 1 - window
                if prefix is not None:
                    seen |= (j < prefix[s]) & (j < self.ctx[s])
                t = np.flatnonzero(seen)
                self.kc[b][:, :, t] = normal(rng, (Hkv, D, t.size), dtype)
                self.vc[b][:, :, t] = normal(rng, (Hkv, D, t.size), dtype)
        self.q = normal(rng, (self.S, H, D), dtype, qstd)
        self.upload()

    def upload(self):
        up = DeviceArray.from_numpy
        self.d = {k: up(getattr(self, k)) for k in ("q", "kc", "vc", "bt", "ctx")}
        sl, pre = self.score["slopes"], self.score["prefix"]
        self.d["slopes"] = None if sl is None else up(sl)
        self.d["prefix"] = None if pre is None else up(pre)
        self.out = DeviceArray((self.S + 1, self.H, self.D), np.uint16)
        self.out.fill_byte(0x7F)
        n = step.scored_decode_workspace_size(self.S, self.H, self.Hkv, self.D, 16, self.MB)
        self.ws = DeviceArray((n,), np.uint8)
        self.ws.fill_byte(0xFF)

    def run(self, stream=None, bounded=True, out=None):
        p = step.ScoreParams(self.score["scale"], self.score["softcap"], self.score["window"],
                             self.d["slopes"], self.d["prefix"])
        step.scored_decode(out or self.out, self.ws, self.ws.nbytes, self.d["q"], self.d["kc"],
                           self.d["vc"], self.d["bt"], self.d["ctx"], p, self.S, self.H, self.Hkv,
                           self.D, 16, self.MB, dtype=self.dtype,
                           num_blocks=self.NB if bounded else 0, stream=stream)

    def want(self):
        f = lambda x: to_float(x, self.dtype)  # noqa: E731
        a = (f(self.q), f(self.kc), f(self.vc), self.bt, np.minimum(self.ctx, 16 * self.MB), np.arange(self.S + 1))
        w = oracle.scored_attention(*a, **self.score)
        return w, scored_bound(*a, self.dtype, 2, w, **self.score)

    def check(self, what=""):
        synchronize()
        got = self.out.numpy()
        assert (got[self.S] == 0x7F7F).all(), "row behind the last sequence"
        got = to_float(got[:self.S], self.dtype)
        want, bound = self.want()
        assert np.isfinite(got).all(), f"{what}: not finite"
        err = np.abs(got - want)
        assert (err <= bound).all(), f"{what}: {(err / bound).max():.2f} of the bound, error {err.max():.2e}"


HEADS = [(8, 8, 64), (32, 8, 128), (64, 8, 128), (16, 16, 128), (40, 2, 64), (3, 1, 128), (1, 1, 64)]
EDGES = [1, 2, 15, 16, 17, 31, 33, 64, 65, 100]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("score", [dict(), dict(cap=20.0), dict(alibi=True), dict(cap=30.0, alibi=True)])
def test_decode_scores_and_heads(dev, H, Hkv, D, score, dtype):
    d = Decode(np.random.default_rng(H * 3 + D), EDGES, H, Hkv, D, dtype, **score)
    d.run()
    d.check(f"{H}/{Hkv}x{D} {score}")


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 33, 64, 1000])
@pytest.mark.parametrize("prefix", [None, [0, 1, 2, 3, 15, 16, 17, 40, 100, 0]])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_windows_and_prefixes(dev, window, prefix, wide):
    """Window and prefix edges in every place of a block, and overlapping; a
    wide table takes the split path."""
    d = Decode(np.random.default_rng(window), EDGES, 8, 2, 64, "f16", window=window, prefix=prefix,
               cap=25.0, alibi=True, MB=300 if wide else None)
    d.run()
    d.check(f"window {window} prefix {prefix}")


@pytest.mark.parametrize("ctx", [[5000], [7919, 1, 300], [1] * 30 + [4001], [2000, 0, 1999, 16, 0]])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(8, 8, 64, "f16"), (32, 8, 128, "bf16"), (40, 2, 128, "f16")])
def test_decode_long_contexts_are_split(dev, ctx, H, Hkv, D, dtype):
    d = Decode(np.random.default_rng(len(ctx)), ctx, H, Hkv, D, dtype, cap=30.0, alibi=True)
    d.run()
    d.check(f"{ctx[:3]}")


@pytest.mark.parametrize("S", [200, 257, 700])
def test_decode_many_ragged_sequences(dev, S):
    """More sequences than threads look at one each, empty ones among them."""
    rng = np.random.default_rng(S)
    ctx = np.minimum(rng.lognormal(3.0, 1.2, S).astype(int), 1500)
    ctx[rng.random(S) < 0.1] = 0
    ctx[S // 2] = 1700
    d = Decode(rng, ctx, 8, 4, 64, "bf16", window=400, prefix=rng.integers(0, 40, S), alibi=True)
    d.run()
    d.check(f"S {S}")


def test_decode_split_windowed_long(dev):
    """A window far into long contexts, with a long prefix: the walk jumps."""
    d = Decode(np.random.default_rng(3), [9000, 3000, 12], 8, 2, 128, "f16", window=2500,
               prefix=[1000, 900, 12], cap=15.0)
    d.run()
    d.check()


def test_decode_empty_and_malformed_lengths(dev):
    """Lengths of zero and below write zeros; one past the table is cut there."""
    d = Decode(np.random.default_rng(4), [0, 20, 64, 0, 33], 8, 2, 64, "f16", alibi=True)
    d.ctx = np.array([0, 20, 100000, -5, 33], np.int32)
    d.upload()
    d.run()
    synchronize()
    assert (d.out.numpy()[[0, 3]] == 0).all()
    d.check()


@pytest.mark.parametrize("prefix", [[-3, 5, 1 << 30, -(1 << 31), 0]])
def test_decode_prefixes_out_of_range(dev, prefix):
    d = Decode(np.random.default_rng(5), [20, 20, 64, 7, 33], 8, 2, 64, "bf16", window=5,
               prefix=np.clip(prefix, 0, 1 << 20))
    d.score["prefix"] = np.array(prefix, np.int32)
    d.upload()
    d.run()
    d.check()


@pytest.mark.parametrize("wide", [False, True])
def test_decode_blocks_outside_the_pool(dev, wide):
    """Bad ids hold no key: whole sequences of them write zeros."""
    d = Decode(np.random.default_rng(6), [100, 64, 48, 300], 8, 2, 64, "f16", cap=30.0,
               MB=400 if wide else None)
    d.bt[0, [0, 3]] = [-1, d.NB]
    d.bt[1, :4] = [-5, 1 << 30, -(1 << 31), d.NB]
    d.bt[3, 18] = -1
    d.upload()
    d.run()
    d.check()
    assert (d.out.numpy()[1] == 0).all()
    d.bt[d.bt == d.NB] = -2      # no bound: only negative ids are known to be bad
    d.bt[d.bt >= 1 << 30] = -2
    d.upload()
    d.run(bounded=False)
    d.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_values_that_are_not_finite(dev, dtype, wide):
    """A NaN key that is seen makes NaN of the heads that see it and of no
    other; infinite and NaN values make their own element not finite."""
    inf = {"f16": 0x7C00, "bf16": 0x7F80}[dtype]
    for cap in (0.0, 20.0):
        d = Decode(np.random.default_rng(7), [40, 40, 700 if wide else 40, 40], 4, 2, 64, dtype, cap=cap)
        d.kc[d.bt[0, 1], 0, 5, 3] = NAN16
        d.vc[d.bt[1, 2], 0, 9, 1] = inf
        d.vc[d.bt[2, 0], 1, 63, 15] = inf | 0x8000
        d.vc[d.bt[3, 1], 1, 0, 0] = NAN16
        d.upload()
        d.run()
        synchronize()
        with np.errstate(all="ignore"):
            want, bound = d.want()
        got = to_float(d.out.numpy()[:4], dtype)
        # (an infinite value times a part of a weight that is 0 is NaN)
        fine = np.isfinite(want)
        assert np.array_equal(fine, np.isfinite(got))
        assert fine.sum() == want.size - 2 * 64 - 6
        assert (np.abs(got - np.where(fine, want, 0))[fine] <= bound[fine]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(cap=1000.0)])
def test_decode_sums_small_weights(dev, dtype, kw):
    """20000 keys 22 binary places below the largest count; of values of 1 the
    output is 1 (powers of two and exact sums, but for a cap's, which are off
    alike), and of a 0 for the largest it is their share, off by a step of their
    weight in fp16 (2^-9 of it), half a step of the output and the cap's 2^-11."""
    d = Decode(np.random.default_rng(17), [20010, 40], 2, 1, 64, dtype, scale=1.0, **kw)
    d.kc[:], d.vc[:], d.q[:] = 0, to_half(np.ones(1), dtype)[0], 0
    d.kc[d.bt[0, 0], 0, 0, 0] = to_half(np.array([15.25]), dtype)[0]     # 22 / log2(e)
    d.q[:, :, 0] = to_half(np.ones(1), dtype)[0]
    d.upload()
    d.run()
    synchronize()
    got = to_float(d.out.numpy()[:2], dtype)
    assert (np.abs(got - 1.0) <= 2.0 ** (-11 if dtype == "f16" else -8)).all(), np.abs(got - 1).max()
    d.vc[d.bt[0, 0], 0, :, 0] = 0
    d.d["vc"].upload(d.vc)
    d.run()
    synchronize()
    got = to_float(d.out.numpy()[:1], dtype)
    want = 20009 / (20009 + np.exp(1000 * np.tanh(0.01525) if kw else 15.25))
    assert (np.abs(got / want - 1) <= 2.0 ** (-8 if dtype == "f16" else -7)).all(), np.abs(got / want - 1).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("wide", [False, True])
def test_decode_a_query_that_is_not_finite(dev, dtype, wide):
    """It makes NaN of its own head and of no other."""
    d = Decode(np.random.default_rng(18), [40, 3000 if wide else 40], 8, 2, 64, dtype, alibi=True)
    want, bound = d.want()
    d.q[0, 1, 7] = d.q[1, 6, 63] = NAN16
    d.upload()
    d.run()
    synchronize()
    got = to_float(d.out.numpy()[:2], dtype)
    fine = np.ones((2, 8), bool)
    fine[0, 1] = fine[1, 6] = False
    assert np.isnan(got[~fine]).all()
    assert (np.abs(got - want)[fine] <= bound[fine]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_large_scores(dev, dtype):
    """Scores of hundreds, far above and below each other; a cap bounds them."""
    for cap in (0.0, 50.0):
        d = Decode(np.random.default_rng(9), [500, 77], 8, 2, 128, dtype, cap=cap, qstd=100.0)
        d.run()
        d.check(f"cap {cap}")


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_decode_scales(dev, scale):
    d = Decode(np.random.default_rng(10), [70, 5], 8, 2, 64, "f16", scale=scale, cap=9.0, alibi=True, qstd=1.0)
    d.run()
    d.check()


def test_decode_block_offsets_past_32_bits(dev):
    """Blocks more than 2^32 bytes into the pool."""
    H, Hkv, D, NB = 8, 8, 128, 140000      # 32 KiB a block and cache: 4.6 GB each
    rng = np.random.default_rng(11)
    kc, vc = DeviceArray((NB, Hkv, D, 16), np.uint16), DeviceArray((NB, Hkv, D, 16), np.uint16)
    d = Decode(rng, [40, 33], H, Hkv, D, "f16", cap=20.0)
    far = NB - 1 - np.arange(d.NB)
    n = Hkv * D * 16 * 2
    for b in range(d.NB):
        kc.upload_at(int(far[b]) * n, d.kc[b])
        vc.upload_at(int(far[b]) * n, d.vc[b])
    bt = np.where(d.bt < d.NB, far[np.minimum(d.bt, d.NB - 1)], 0).astype(np.int32)
    d.d["bt"] = DeviceArray.from_numpy(bt)
    d.d["kc"], d.d["vc"], small = kc, vc, d.NB
    d.NB = NB
    d.run()
    d.NB = small
    d.check()


@pytest.mark.parametrize("ctx", [[33, 1, 300], [4000, 16, 700]])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_decode_output_2_byte_aligned(dev, ctx, shift):
    """Any alignment of the output gives the same bits, and nothing beside it is written."""
    d = Decode(np.random.default_rng(19), ctx, 6, 2, 128, "f16", cap=20.0)
    d.run()
    d.check()
    n = d.S * d.H * d.D
    buf = DeviceArray((n + 8,), np.uint16)
    buf.fill_byte(0x7F)
    d.run(out=buf.ptr + 2 * shift)
    synchronize()
    got = buf.numpy()
    assert np.array_equal(got[shift:shift + n], d.out.numpy()[:d.S].ravel())
    assert (got[:shift] == 0x7F7F).all() and (got[shift + n:] == 0x7F7F).all()


def test_decode_leaves_no_trace_between_calls(dev):
    """One workspace for calls of other shapes in turn, and the same call twice: the same bits."""
    a = Decode(np.random.default_rng(12), [3000, 1, 500], 8, 2, 64, "f16", alibi=True)
    b = Decode(np.random.default_rng(13), [1] * 20 + [4000], 8, 2, 64, "f16", cap=10.0)
    b.ws = a.ws
    a.run()
    a.check()
    first = a.out.numpy()
    b.run()
    b.check()
    a.run()
    synchronize()
    assert np.array_equal(first, a.out.numpy())


@pytest.mark.parametrize("ctx,H,Hkv", [([33, 1, 16, 0, 300], 8, 2), ([5000, 9, 700], 40, 2)])
def test_decode_into_the_queries(dev, ctx, H, Hkv):
    """output may be query: sequences taken whole, and cut ones that a join writes."""
    d = Decode(np.random.default_rng(16), ctx, H, Hkv, 64, "f16", cap=20.0)
    d.run()
    synchronize()
    d.out.upload(np.concatenate([d.q, np.full((1, H, 64), 0x7F7F, np.uint16)]))
    d.d["q"] = d.out
    d.run()
    d.check("in place")


def test_decode_in_a_captured_graph(dev):
    """Replays follow the lengths and tables in the buffers; two graphs with a
    workspace each on two streams at once."""
    rng = np.random.default_rng(14)
    cs = [Decode(rng, [2000, 900, 1, 40], 8, 2, 64, "f16", window=700, cap=20.0),
          Decode(rng, [100, 2500], 8, 2, 128, "bf16", alibi=True)]
    streams = [Stream(), Stream()]
    graphs = []
    for c, s in zip(cs, streams):
        c.run(s)
        s.synchronize()
        graphs.append(Graph(s, lambda c=c, s=s: c.run(s)))
    for step_ in range(3):
        for c in cs:
            c.ctx = np.maximum(c.ctx - step_ * np.array([16, 1, 0, 3])[:c.S], 0).astype(np.int32)
            if c.score["window"]:
                c.kc[:], c.vc[:] = normal(rng, c.kc.shape, c.dtype), normal(rng, c.vc.shape, c.dtype)
                c.d["kc"].upload(c.kc)
                c.d["vc"].upload(c.vc)
            c.d["ctx"].upload(c.ctx)
            c.out.fill_byte(0x7F)
        synchronize()
        for g, s in zip(graphs, streams):
            g.launch(s)
        for s in streams:
            s.synchronize()
        for c in cs:
            c.check(f"replay {step_}")


@pytest.mark.parametrize("wide", [False, True])
def test_decode_rows_of_a_packed_step(dev, wide):
    """With offsets: the last row of each sequence, none for one without rows
    or with offsets out of range; other rows are left as they were."""
    rng = np.random.default_rng(15)
    d = Decode(rng, [40, 700, 33, 5, 64, 20], 8, 2, 64, "f16", cap=20.0, MB=300 if wide else 44)
    off = np.array([2, 3, 6, 6, 7, 40, 41], np.int32)     # 0, 1 and 3 have rows; 5's lie past them
    T = 12
    q = normal(rng, (T, 8, 64), "f16", 3.0)
    rows = {0: 2, 1: 5, 3: 6}
    for s in range(6):
        d.q[s] = q[rows.get(s, 0)]
    out, d_q, d_off = DeviceArray((T, 8, 64), np.uint16), DeviceArray.from_numpy(q), DeviceArray.from_numpy(off)
    out.fill_byte(0x7F)
    p = step.ScoreParams(d.score["scale"], 20.0)
    step.scored_decode(out, d.ws, d.ws.nbytes, d_q, d.d["kc"], d.d["vc"], d.d["bt"], d.d["ctx"], p, 6, 8, 2,
                       64, 16, d.MB, num_blocks=d.NB, query_offsets=d_off, num_tokens=T)
    synchronize()
    got = out.numpy()
    want, bound = d.want()
    for s, r in rows.items():
        assert (np.abs(to_float(got[r], "f16") - want[s]) <= bound[s]).all()
    assert (np.delete(got, list(rows.values()), axis=0) == 0x7F7F).all()


@pytest.mark.parametrize("ctx", [[1, 20, 64, 100], [3000, 40, 7]])
@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0, alibi=True)])
def test_decode_of_large_values(dev, ctx, kw):
    """bfloat16 has values near 2^128: a weighted mean of values of 2^116, at
    most 2^121 of them, is a number like any other."""
    d = Decode(np.random.default_rng(20), ctx, 8, 2, 64, "bf16", **kw)
    for s, n in enumerate(ctx):
        for i in range(-(-n // 16)):
            t = np.arange(min(n - 16 * i, 16))
            b = d.bt[s, i]
            d.vc[b][:, :, t] = normal(np.random.default_rng(i), (2, 64, t.size), "bf16", 2.0 ** 116)
    d.upload()
    d.run()
    d.check()


def test_decode_of_the_largest_value(dev):
    """One key: its value, whatever it is."""
    d = Decode(np.random.default_rng(21), [1, 1], 8, 2, 64, "bf16")
    top = to_half(np.array([2.0 ** 127 * (2 - 2.0 ** -7)]), "bf16")[0]
    for s in range(2):
        d.vc[d.bt[s, 0], :, :, 0] = top if s == 0 else top | 0x8000
    d.upload()
    d.run()
    synchronize()
    got = d.out.numpy()
    assert (got[0] == top).all() and (got[1] == (top | 0x8000)).all()


@pytest.mark.parametrize("cap", [0.0, 1e-39, 20.0])
def test_decode_scale_of_zero(dev, cap):
    """Every key counts the same, whatever the cap."""
    d = Decode(np.random.default_rng(22), [70, 5], 8, 2, 64, "f16", scale=0.0, cap=cap)
    d.run()
    d.score["softcap"] = 0.0
    d.check()


def test_decode_weights_in_two_parts(dev):
    """bfloat16 weights are kept in two parts, each rounded to nearest: off by
    2^-8 and then by 2^-9 of that, 2^-17 of the weight. Seen where a block's 15
    equal weights of values of 1 are taken against one of 1 of a value of some
    -15 of them; the exponent, exp2, sums and the quotient add less than 2^-20."""
    x = to_float(np.arange(0x3F80, 0x4040, dtype=np.uint16), "bf16").astype(np.float64)   # 1 .. 3
    p = np.exp(-x)
    v = to_float(to_half(-15 * p, "bf16"), "bf16").astype(np.float64)
    want = (15 * p + v) / (15 * p + 1)
    best = np.argsort(np.abs(want))[:16]        # near 0, so that their rounding is small
    x, p, v, want = x[best], p[best], v[best], want[best]
    d = Decode(np.random.default_rng(23), [16], 16, 16, 64, "bf16", scale=1.0)
    one = to_half(np.ones(1), "bf16")[0]
    d.q[:], d.kc[:], d.vc[:] = 0, 0, one
    d.q[0, :, 0] = to_half(x, "bf16")
    d.kc[d.bt[0, 0], :, 0, :] = one | 0x8000    # scores of -x
    d.kc[d.bt[0, 0], :, 0, 5] = 0               # but one of 0
    d.vc[d.bt[0, 0], :, :, 5] = to_half(v, "bf16")[:, None]
    d.upload()
    d.run()
    synchronize()
    err = np.abs(to_float(d.out.numpy()[0], "bf16") - want[:, None]).max(axis=1)
    bound = 2.0 ** -17 * 15 * p / (15 * p + 1) + 2.0 ** -20 + 2.0 ** -8 * np.abs(want)
    assert (err <= bound).all(), (err / bound).max()
