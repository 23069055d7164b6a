"""plan_shared and shared_decode on the GPU against the oracle in float64
(tolerance: step_helpers.scored_bound, weights in one 16-bit part): groups whose
tables begin alike, partly, wholly or not at all, sequences without a context
among them, both types, caps and biases, garbage in every slot that nobody sees."""

import numpy as np
import pytest

import oracle
from step_helpers import NAN16, normal, scored_bound, to_float, to_half
from swiftllm_amd import attention_step as step
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Shared:
    """groups: of each, (tokens of whole shared blocks, the contexts of its sequences)."""

    def __init__(self, rng, groups, H, Hkv, D, dtype, cap=0.0, alibi=False, MB=None, scale=None, spare=3, qstd=3.0,
                 lone=0, tight=False, min_saved=0):
        self.min_saved = min_saved      # what is alike is shared, but where a test asks for the rule
        ctx = [c for _, cs in groups for c in cs]
        self.ctx = np.array(ctx + [int(rng.integers(0, 50)) for _ in range(lone)], np.int32)
        self.S, self.H, self.Hkv, self.D, self.dtype = len(self.ctx), H, Hkv, D, dtype
        used = [-(-max(int(c), 0) // 16) for c in self.ctx]
        # (tables of up to 48 blocks are taken whole where they are few: tight ones)
        self.MB = max(used + [1 if tight else 97]) if MB is None else MB
        common = [p // 16 for p, _ in groups]
        need = sum(common) + sum(used) + 1
        self.NB = need + spare
        ids = rng.permutation(self.NB).astype(np.int32)
        self.bt = np.full((self.S, self.MB), 2 ** 31 - 1, np.int32)   # nobody reads these
        self.kc = np.full((self.NB, Hkv, D, 16), NAN16, np.uint16)
        self.vc = np.full((self.NB, Hkv, D, 16), NAN16, np.uint16)
        self.off = np.cumsum([0] + [len(cs) for _, cs in groups]).astype(np.int32)
        at = s = 0
        filled = {}
        for (_, cs), n in zip(groups, common):
            lead = ids[at:at + n]
            at += n
            for c in cs:
                k = used[s]
                mine = np.concatenate([lead[:k], ids[at:at + max(k - n, 0)]])
                at += max(k - n, 0)
                self.bt[s, :min(k, self.MB)] = mine[:self.MB]
                for i, b in enumerate(mine):
                    filled[int(b)] = max(filled.get(int(b), 0), min(16, int(c) - 16 * i))
                s += 1
        for s in range(s, self.S):
            k = used[s]
            self.bt[s, :min(k, self.MB)] = ids[at:at + k][:self.MB]
            for i, b in enumerate(ids[at:at + k]):
                filled[int(b)] = min(16, int(self.ctx[s]) - 16 * i)
            at += k
        for b, n in filled.items():
            self.kc[b][:, :, :n] = normal(rng, (Hkv, D, n), dtype)
            self.vc[b][:, :, :n] = normal(rng, (Hkv, D, n), dtype)
        self.score = dict(scale=D ** -0.5 if scale is None else scale, softcap=cap,
                          slopes=step.alibi_slopes(H) if alibi else None)
        self.q = normal(rng, (self.S, H, D), dtype, qstd)
        self.upload()

    def upload(self):
        up = DeviceArray.from_numpy
        self.d = {k: up(getattr(self, k)) for k in ("q", "kc", "vc", "bt", "ctx", "off")}
        self.d["slopes"] = None if self.score["slopes"] is None else up(self.score["slopes"])
        self.N = len(self.off) - 1
        self.sizes = (self.S, self.H, self.Hkv, self.D, 16, self.MB)
        self.out = DeviceArray((self.S + 1, self.H, self.D), np.uint16)
        self.out.fill_byte(0x7F)
        self.sh = DeviceArray((max(self.N, 1),), np.int32)
        self.plan = DeviceArray((step.plan_shared_size(*self.sizes),), np.uint8)
        self.ws = DeviceArray((step.shared_decode_workspace_size(*self.sizes),), np.uint8)
        for x in (self.plan, self.ws, self.sh):
            x.fill_byte(0xFF)

    def run_plan(self, stream=None):
        step.plan_shared(self.plan, self.plan.nbytes, self.sh, self.d["bt"], self.d["ctx"], self.d["off"], self.N,
                         *self.sizes, min_saved=self.min_saved, stream=stream)

    def run_decode(self, stream=None, bounded=True, out=None, **kw):
        p = step.ScoreParams(self.score["scale"], self.score["softcap"], alibi_slopes=self.d["slopes"])
        step.shared_decode(self.out if out is None else out, self.ws, self.ws.nbytes, self.plan, self.plan.nbytes, self.d["q"],
                           self.d["kc"], self.d["vc"], self.d["bt"], p, *self.sizes, dtype=self.dtype,
                           num_blocks=self.NB if bounded else 0, stream=stream, **kw)

    def run(self, stream=None, **kw):
        self.run_plan(stream)
        self.run_decode(stream, **kw)
        return self

    def want(self):
        f = lambda x: to_float(x, self.dtype)  # noqa: E731
        a = (f(self.q), f(self.kc), f(self.vc), self.bt, np.minimum(self.ctx, 16 * self.MB), np.arange(self.S + 1))
        w = oracle.scored_attention(*a, **self.score)
        return w, scored_bound(*a, self.dtype, 1, w, **self.score)

    def check(self, what=""):
        synchronize()
        assert np.array_equal(self.sh.numpy()[:self.N], oracle.shared_blocks(self.bt, self.ctx, self.off)), what
        got = self.out.numpy()
        assert (got[self.S] == 0x7F7F).all(), "row behind the last sequence"
        want, bound = self.want()
        got = to_float(got[:self.S], self.dtype)
        assert np.isfinite(got).all(), what
        err = np.abs(got - want)
        assert (err <= bound).all(), f"{what}: {(err / bound).max():.2f} of the bound"
        return got


def whole(s):
    """Whether every sequence is read whole, by the launcher's rule."""
    G = s.H // s.Hkv
    parts = -(-min(G, 32) // 16)
    return s.MB <= 48 and s.S * s.Hkv * -(-G // 32) * parts * s.MB * 64 * s.D <= 64e6


HEADS = [(8, 8, 64), (32, 8, 128), (16, 2, 128), (6, 2, 64), (5, 1, 128), (1, 1, 64), (40, 1, 64), (96, 2, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
def test_heads(dev, H, Hkv, D, dtype):
    """Groups of several sizes, one of more than a tile's rows, a sequence of no group."""
    rng = np.random.default_rng(H + D)
    groups = [(320, [321, 340, 365, 400]), (64, [70, 64, 100]), (0, [33]), (160, [161 + 3 * i for i in range(36)])]
    Shared(rng, groups, H, Hkv, D, dtype, lone=2).run().check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
def test_heads_whole(dev, H, Hkv, D, dtype):
    """Short tables, each sequence read whole; those without a context, odd block ids, an output at any address."""
    rng = np.random.default_rng(H + D)
    groups = [(160, [165, 170, 0]), (64, [70, 64, 100, 1, 16]), (0, [33])]
    for cap, alibi in ((0.0, False), (25.0, True)):
        s = Shared(rng, groups, H, Hkv, D, dtype, cap=cap, alibi=alibi, lone=2, tight=True)
        assert whole(s)
        s.bt[1, 3], s.bt[5, 5] = -3, s.NB
        s.bt[0, 3] = s.bt[2, 3] = -3
        s.upload()
        s.run().check()
        out = DeviceArray((s.q.size + 3,), np.uint16)
        s.run_decode(out=out.ptr + 2)
        synchronize()
        assert np.array_equal(out.numpy()[1:-2].reshape(s.q.shape), s.out.numpy()[:s.S])


@pytest.mark.parametrize("cap,alibi", [(0.0, False), (20.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(8, 2, 128, "bf16"), (16, 2, 64, "f16"), (4, 4, 128, "f16"), (8, 1, 64, "bf16")])
def test_scores(dev, H, Hkv, D, dtype, cap, alibi):
    rng = np.random.default_rng(D)
    groups = [(1024, [1030, 1025, 1500, 1024, 1100]), (48, [60, 50]), (256, [300] * 3)]
    Shared(rng, groups, H, Hkv, D, dtype, cap=cap, alibi=alibi).run().check()


@pytest.mark.parametrize("extra", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("tight", [False, True])
@pytest.mark.parametrize("H", [8, 24])
def test_lengths_around_stages(dev, extra, tight, H):
    """Shared and own parts that end inside a block and a step, and at their edges."""
    rng = np.random.default_rng(extra)
    groups = [(p, [p + extra, p + extra + 1, p + max(extra - 1, 0)]) for p in (16, 48, 64, 80, 128, 272)]
    s = Shared(rng, groups, H, 2, 128, "f16", tight=tight)
    assert whole(s) == tight
    s.run().check()


@pytest.mark.parametrize("each", [1, 2, 7, 8, 9, 31, 32, 33, 70, 131])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (8, 8, 64), (6, 2, 64)])
def test_group_sizes(dev, each, H, Hkv, D):
    """Tiles that fill their waves' rows, and that do not."""
    rng = np.random.default_rng(each)
    Shared(rng, [(144, [145 + i % 40 for i in range(each)]), (96, [100] * each)], H, Hkv, D, "bf16").run().check()


def test_sequences_without_context(dev):
    """They count for nothing in their group, and their rows are zero."""
    rng = np.random.default_rng(1)
    groups = [(160, [0, 170, 0, 180, 200, 0]), (160, [0, 0]), (160, [0, 0, 165]), (80, [-5, 90, 91, 92])]
    s = Shared(rng, groups, 8, 2, 64, "f16").run()
    got = s.check()
    assert (got[s.ctx <= 0] == 0).all()


@pytest.mark.parametrize("min_saved", [-1, 0, 1, 400, 10 ** 6])
@pytest.mark.parametrize("H,Hkv", [(16, 8), (4, 4)])
def test_what_is_worth_sharing(dev, H, Hkv, min_saved):
    """By the rule, by a number of blocks, never: the same outputs. Several tiles of a
    group that begin with ranges, beside others that do not."""
    rng = np.random.default_rng(H)
    groups = [(1600, [1610 + i % 90 for i in range(70)]), (32, [40, 50]), (320, [333, 321, 400])]
    Shared(rng, groups, H, Hkv, 64, "f16", min_saved=min_saved).run().check()


@pytest.mark.parametrize("each", [33, 64, 100, 129])
def test_aligned_tiles(dev, each):
    """Groups of several tiles whose walks begin and end with ranges."""
    rng = np.random.default_rng(each)
    groups = [(9600, [9600 + i % 70 for i in range(each)]), (64, [70, 80, 90]), (4800, [4810] * (each + 1))]
    Shared(rng, groups, 8, 2, 64, "bf16", lone=2).run().check()


def test_nothing_shared_and_everything(dev):
    rng = np.random.default_rng(2)
    s = Shared(rng, [(0, [100, 200, 300])], 8, 2, 128, "f16").run()
    s.check()
    assert s.sh.numpy()[0] == 0
    s = Shared(rng, [(320, [320] * 5), (304, [300] * 4)], 8, 2, 128, "f16").run()
    s.check()
    assert s.sh.numpy().tolist() == [20, 19]


def test_tables_that_part_and_meet(dev):
    """What is alike behind a difference is not shared; neither is a block in another place."""
    rng = np.random.default_rng(3)
    s = Shared(rng, [(640, [650, 660, 700])], 8, 2, 64, "bf16")
    s.bt[1, 30] = s.bt[1, 29]
    s.upload()
    s.run()
    s.check()
    assert s.sh.numpy()[0] == 30
    s.bt[2, 0], s.bt[2, 1] = s.bt[2, 1], s.bt[2, 0]
    s.upload()
    s.run()
    s.check()
    assert s.sh.numpy()[0] == 0


@pytest.mark.parametrize("off", [[0, 2, 1, 6], [0, 4, 7], [-1, 3, 6], [3, 2], [0, 3, 2 ** 31 - 1], [5, 5, 4, 4, 6]])
def test_offsets_out_of_order_share_nothing(dev, off):
    rng = np.random.default_rng(4)
    s = Shared(rng, [(320, [330, 340, 350, 360, 370, 380])], 8, 2, 64, "f16")
    s.off = np.array(off, np.int32)
    s.upload()
    s.run()
    s.check()
    assert (s.sh.numpy() == 0).all()


@pytest.mark.parametrize("off", [[0, 0, 0, 6, 6], [1, 4], [2, 2], [0, 1, 2, 3, 4, 5, 6], [4, 6], []])
def test_groups_that_leave_sequences_out(dev, off):
    rng = np.random.default_rng(5)
    s = Shared(rng, [(320, [330, 340, 350, 360, 370, 380])], 8, 2, 64, "f16")
    s.off = np.array(off or [0], np.int32)
    s.upload()
    s.run()
    s.check()


@pytest.mark.parametrize("n", [300, 1100, 4200])
def test_many_small_groups(dev, n):
    """More sequences than the list's kernel has threads, and more groups than its window holds."""
    rng = np.random.default_rng(6)
    groups = [(32, [33 + int(rng.integers(0, 20)) for _ in range(2)]) for _ in range(n)]
    s = Shared(rng, groups, 2, 1, 64, "f16")
    s.run()
    synchronize()
    assert np.array_equal(s.sh.numpy(), np.full(n, 2))
    s.check()


def test_long_contexts(dev):
    """Walks cut into many ranges; own parts longer than what is shared; lone long sequences."""
    rng = np.random.default_rng(7)
    for groups in ([(30000, [30010, 30500, 31000])], [(64, [20000, 70]), (0, [9000])], [(4096, [4100] * 40)]):
        Shared(rng, groups, 8, 1, 64, "f16", alibi=len(groups) == 1).run().check()


def test_blocks_outside_the_pool(dev):
    """They hold no key, shared or own."""
    rng = np.random.default_rng(8)
    s = Shared(rng, [(320, [400, 410, 420]), (320, [330, 340])], 8, 2, 128, "f16")
    s.bt[:3, 4] = [-7, -7, -7]
    s.bt[1, 22] = s.NB
    s.bt[3:, :21] = -1
    s.bt[4, 21] = 2 ** 31 - 1
    s.upload()
    s.run()
    s.check()


def test_context_longer_than_the_table(dev):
    rng = np.random.default_rng(9)
    s = Shared(rng, [(96, [97, 98, 99])], 8, 2, 64, "f16", MB=7, alibi=True)
    s.ctx[:] = [113, 5000, 2 ** 31 - 1]
    for b in s.bt[:, 6]:
        s.kc[b] = normal(rng, s.kc[b].shape, "f16")
        s.vc[b] = normal(rng, s.vc[b].shape, "f16")
    s.upload()
    s.run()
    synchronize()
    # the keys end with the table, and so do the bias's distances: the same weights
    f = lambda x: to_float(x, "f16")  # noqa: E731
    a = (f(s.q), f(s.kc), f(s.vc), s.bt, np.minimum(s.ctx, 112), np.arange(4))
    want = oracle.scored_attention(*a, **s.score)
    err = np.abs(to_float(s.out.numpy()[:3], "f16") - want)
    assert (err <= scored_bound(*a, "f16", 1, want, **s.score)).all()


def test_values_that_are_not_finite(dev):
    """A key or a value that is not finite stays with the sequences that see it."""
    rng = np.random.default_rng(10)
    s = Shared(rng, [(160, [200, 210, 220]), (160, [170, 171])], 8, 2, 64, "f16")
    clean = s.want()
    s.vc[s.bt[1, 11]][0, 5, 3] = 0x7C00       # an own value of sequence 1, kv head 0
    s.kc[s.bt[4, 10]][1, 0, 0] = NAN16        # an own key of sequence 4, kv head 1
    s.upload()
    s.run()
    synchronize()
    got = to_float(s.out.numpy()[:5], "f16")
    touched = np.zeros((5, 8), bool)
    touched[1, :4] = touched[4, 4:] = True
    assert not np.isfinite(got[1, :4]).all(axis=1).any() and not np.isfinite(got[4, 4:]).all(axis=1).any()
    assert (np.abs(got - clean[0]) <= clean[1])[~touched].all()
    s.vc[s.bt[0, 2]][1, 7, 7] = NAN16         # a shared value: every sequence of the group
    s.upload()
    s.run()
    synchronize()
    got = to_float(s.out.numpy()[:5], "f16")
    assert np.isnan(got[:3, 4:, 7]).all()
    touched[:3, 4:] = True
    assert (np.abs(got - clean[0]) <= clean[1])[~touched].all()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-30])
@pytest.mark.parametrize("cap", [0.0, 10.0])
def test_scales(dev, scale, cap):
    rng = np.random.default_rng(11)
    Shared(rng, [(160, [200, 210]), (0, [64])], 8, 2, 64, "bf16", cap=cap, scale=scale, qstd=1.0).run().check()


@pytest.mark.parametrize("tight", [False, True])
def test_packed_rows(dev, tight):
    """Rows of a step: the last of each sequence's; sequences without rows, and rows of none."""
    rng = np.random.default_rng(12)
    s = Shared(rng, [(160, [170, 180, 190, 200])], 8, 2, 64, "f16", tight=tight)
    off = np.array([0, 1, 1, 4, 5], np.int32)     # rows 0, none, 1-3, 4; row 5 of none
    q = normal(rng, (6, 8, 64), "f16", 3.0)
    s.q = np.stack([q[0], np.zeros_like(q[0]), q[3], q[4]])
    s.d["q"] = DeviceArray.from_numpy(q)
    d_off, out = DeviceArray.from_numpy(off), DeviceArray((7, 8, 64), np.uint16)
    out.fill_byte(0x7F)
    s.run_plan()
    s.run_decode(out=out, query_offsets=d_off, num_tokens=6)
    synchronize()
    got = out.numpy()
    want, bound = s.want()
    for row, seq in ((0, 0), (3, 2), (4, 3)):
        assert (np.abs(to_float(got[row], "f16") - want[seq]) <= bound[seq]).all()
    assert (got[[1, 2, 5, 6]] == 0x7F7F).all()
    # offsets that run backwards or out of the rows have none
    out.fill_byte(0x7F)
    d_off.upload(np.array([0, 1, 0, 9, 5], np.int32))
    s.run_decode(out=out, query_offsets=d_off, num_tokens=6)
    synchronize()
    assert (out.numpy()[1:] == 0x7F7F).all()


def test_odd_addresses(dev):
    """Outputs at any 2-byte address, queries at any 8-byte one."""
    rng = np.random.default_rng(13)
    s = Shared(rng, [(160, [170, 180]), (0, [20, 30])], 8, 2, 64, "bf16")
    raw = DeviceArray((s.q.size + 4,), np.uint16)
    raw.upload_at(8, s.q.reshape(-1))
    out = DeviceArray((s.q.size + 3,), np.uint16)
    s.d["q"] = raw.ptr + 8
    s.run(out=out.ptr + 2)
    synchronize()
    got = to_float(out.numpy()[1:-2].reshape(s.q.shape), "bf16")
    want, bound = s.want()
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("tight", [False, True])
def test_plan_of_other_sizes_writes_nothing(dev, tight):
    rng = np.random.default_rng(14)
    s = Shared(rng, [(160, [170, 180])], 8, 2, 64, "f16", tight=tight)
    t = Shared(rng, [(160, [170, 180])], 4, 2, 64, "f16", tight=tight)
    t.run_plan()
    s.plan.upload(t.plan.numpy())
    s.run_decode()
    synchronize()
    assert (s.out.numpy() == 0x7F7F).all()
    s.plan.fill_byte(0)
    s.run_decode()
    synchronize()
    assert (s.out.numpy() == 0x7F7F).all()


def test_the_same_bits_each_time(dev):
    rng = np.random.default_rng(15)
    s = Shared(rng, [(2048, [2049 + 31 * i for i in range(20)])], 32, 8, 128, "f16").run()
    first = s.check()
    for _ in range(3):
        s.ws.fill_byte(0xAB)
        s.run(bounded=False)
        assert np.array_equal(s.check(), first)


def test_graph_of_a_plan_and_layers(dev):
    """One graph of a plan and two layers, replayed while contexts and groups change,
    beside eager calls of another object on another stream."""
    rng = np.random.default_rng(16)
    s = Shared(rng, [(320, [400, 390, 380, 370]), (160, [200, 210])], 8, 2, 128, "f16")
    other = Shared(rng, [(480, [490] * 6)], 8, 2, 128, "f16")
    out2 = DeviceArray((s.S + 1, s.H, s.D), np.uint16)
    stream, aside = Stream(), Stream()

    def enqueue():
        s.run_plan(stream)
        s.run_decode(stream)
        s.run_decode(stream, out=out2)

    enqueue()
    stream.synchronize()
    s.check()
    g = Graph(stream, enqueue)
    for i in range(4):
        s.ctx[:] = [400 - 40 * i, 390, 0 if i == 2 else 380, 370 - i, 200 - 17 * i, 210]
        s.off[:] = [[0, 4, 6], [0, 3, 6], [0, 4, 6], [1, 4, 5]][i]
        s.d["ctx"].upload(s.ctx)
        s.d["off"].upload(s.off)
        s.out.fill_byte(0x7F)
        synchronize()
        g.launch(stream)
        other.run(aside)
        stream.synchronize()
        s.check()
        assert np.array_equal(out2.numpy()[:s.S], s.out.numpy()[:s.S])
        aside.synchronize()
        other.check()


def test_random_sweep(dev):
    rng = np.random.default_rng(17)
    for _ in range(40):
        H, Hkv, D = HEADS[rng.integers(len(HEADS))]
        groups = []
        for _ in range(int(rng.integers(1, 6))):
            p = 16 * int(np.exp(rng.uniform(0, np.log(100))))
            n = int(np.exp(rng.uniform(0, np.log(40))))
            groups.append((p, [0 if rng.random() < 0.1 else p + int(rng.integers(0, 150)) - int(rng.integers(0, 2)) * 16 for _ in range(n)]))
        dtype = ["f16", "bf16"][rng.integers(2)]
        kw = dict(cap=float(rng.choice([0, 0, 25])), alibi=bool(rng.random() < 0.3), lone=int(rng.integers(0, 3)), tight=bool(rng.random() < 0.3))
        print(H, Hkv, D, dtype, [(p, len(c)) for p, c in groups], kw, flush=True)
        Shared(rng, groups, H, Hkv, D, dtype, **kw).run().check()


@pytest.mark.parametrize("Hkv,G", [(300, 1), (520, 1), (130, 2)])
def test_more_heads_than_workgroups(dev, Hkv, G):
    """Two ranges for each chunk of heads, one of what is wide and one of what is not."""
    rng = np.random.default_rng(Hkv)
    s = Shared(rng, [(336, [340 + i for i in range(20)]), (64, [70, 90])], Hkv * G, Hkv, 64, "f16")
    s.run().check()
    s = Shared(rng, [(336, [336] * 20)], Hkv * G, Hkv, 64, "f16")      # nothing but what is wide
    s.run().check()


@pytest.mark.parametrize("each,shared,own", [(24, 800, 3), (24, 48, 900), (3, 640, 400), (130, 1600, 1)])
def test_shares_of_what_is_wide(dev, each, shared, own):
    """Mostly wide, mostly narrow, wholly narrow, and tiles that share with others."""
    rng = np.random.default_rng(each + own)
    for D, dtype in ((64, "bf16"), (128, "f16")):
        s = Shared(rng, [(shared, [shared + int(rng.integers(0, own + 1)) for _ in range(each)]) for _ in range(3)], 8, 2, D, dtype)
        s.run().check()
