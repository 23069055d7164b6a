"""beam_select on the GPU against the oracle in float64.

Scores: the rounding to 32 bits, half a step of 2^-24 of the score, and lse's
error. That is of a sum of exponentials, each off by its exponent's rounding
(2^-24 of the distance from the maximum in log2 units, whose mean under the
softmax is at most log2 V + 2 < 20, once for the product and once for log2 e),
by exp2 (2^-23) and by the sum (32 additions in a thread, 8 between threads, 2^-24
each, and four products): under 2^-24 (40 + 2 + 44) < 2^-17.

Rows and tokens are those of the oracle wherever its neighbours in the order are
further apart than both scores' errors; of a beam's own logits, whose order no
rounding touches, always."""

import numpy as np
import pytest

import oracle
from step_helpers import to_float, to_half
from swiftllm_amd import beam_search as bs
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu

LSE = 2.0 ** -17


class Select:
    def __init__(self, x, scores, C, dtype="f32", eos=-1, stride=None, shift=0):
        """x float32 [R, W, V]; rows `stride` apart from `shift` values on, NaN between them."""
        self.R, self.W, self.V = x.shape
        self.C, self.dtype, self.eos = C, dtype, eos
        self.stride = self.V if stride is None else stride
        raw = np.full(shift + self.R * self.W * self.stride, np.nan, np.float32)
        rows = raw[shift:].reshape(self.R * self.W, self.stride)
        rows[:, :self.V] = x.reshape(-1, self.V)
        flat = raw if dtype == "f32" else to_half(raw, dtype)
        self.x = rows[:, :self.V] if dtype == "f32" else to_float(flat, dtype)[shift:].reshape(rows.shape)[:, :self.V]
        self.x = self.x.reshape(x.shape)
        self.scores = np.asarray(scores, np.float32).reshape(self.R, self.W)
        size = 4 if dtype == "f32" else 2
        self.d_x, self.d_s = DeviceArray.from_numpy(flat), DeviceArray.from_numpy(self.scores)
        self.at = self.d_x.ptr + shift * size
        self.out = {k: DeviceArray((self.R, C if k < 3 else self.W), np.float32 if k % 3 == 0 else np.int32)
                    for k in range(6)}
        n = bs.beam_select_workspace_size(self.R, self.W, self.V, C)
        self.ws = DeviceArray((n,), np.uint8)
        self.fill()

    def fill(self):
        for o in self.out.values():
            o.fill_byte(0x5A)
        self.ws.fill_byte(0xFF)

    def run(self, stream=None):
        bs.beam_select(self.at, self.d_s, *self.out.values(), self.ws, self.ws.nbytes, self.R, self.W, self.V,
                       self.C, dtype=self.dtype, logits_stride=self.stride, eos_id=self.eos, stream=stream)

    def check(self):
        synchronize()
        got = [o.numpy() for o in self.out.values()]
        want = oracle.beam_select(self.x, self.scores, self.C, self.eos)
        for k in (0, 3):
            w, g = want[k], got[k].astype(np.float64)
            assert np.array_equal(np.isfinite(w), np.isfinite(g)) and not (g[~np.isfinite(w)] > -np.inf).any()
            fin = np.isfinite(w)
            bound = np.where(fin, 2.0 ** -24 * np.abs(np.where(fin, w, 0)) + LSE, 0)
            err = np.where(fin, np.abs(np.where(fin, g, 0) - np.where(fin, w, 0)), 0)
            assert (err <= bound).all(), f"{err.max():.2e}"
            # ties and near ones: within a beam the oracle's own order, between beams either
            apart = np.full(w.shape, True)
            rows = want[k + 1]
            for step in (1, -1):
                near = np.roll(w, step, axis=1)
                other = np.roll(rows, step, axis=1)
                close = (np.abs(np.where(fin, w, 0) - np.where(np.isfinite(near), near, 0)) <= 4 * bound) & (other != rows)
                close[:, 0 if step == 1 else -1] = False
                apart &= ~close | ~fin
            if k == 0 and not apart.all():
                # every candidate still is one of the request's, once
                for r in range(self.R):
                    seen = list(zip(got[1][r].tolist(), got[2][r].tolist()))
                    assert len(set(seen)) == len([s for s in seen if s[0] >= 0]) + (1 if (-1, -1) in seen else 0)
            for i in (k + 1, k + 2):
                assert np.array_equal(got[i][apart], want[i][apart])
        return got, want


def _logits(rng, R, W, V, std=3.0):
    return rng.standard_normal((R, W, V)).astype(np.float32) * std


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,W,V,C", [(1, 1, 1, 1), (2, 3, 7, 6), (1, 4, 8192, 8), (3, 4, 8193, 8), (2, 5, 8185, 10),
                                     (1, 32, 9001, 64), (2, 1, 40000, 2), (1, 64, 300, 64), (5, 2, 16391, 4)])
def test_sizes(dev, dtype, R, W, V, C):
    """One chunk and more, vocabularies that end inside a vector, the widest search,
    fewer tokens than candidates."""
    rng = np.random.default_rng(V + W)
    s = Select(_logits(rng, R, W, V), -10 * rng.random((R, W)), C, dtype, eos=V // 2)
    s.run()
    s.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 3), (5, 7), (64, 2)])
def test_rows_at_any_address(dev, dtype, pad, shift):
    """Rows of a padded vocabulary that begin off 16-byte addresses; what lies between them is not read as logits."""
    rng = np.random.default_rng(pad)
    s = Select(_logits(rng, 3, 2, 8190), -rng.random((3, 2)), 4, dtype, stride=8190 + pad, shift=shift)
    s.run()
    s.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_first_step_and_dead_beams(dev, dtype):
    """Beams without a score give nothing; requests without any end; NaN scores count as none."""
    rng = np.random.default_rng(3)
    scores = np.full((4, 3), -np.inf, np.float32)
    scores[0, 0] = 0.0
    scores[1] = [-3.0, -np.inf, -1.0]
    scores[3] = [np.nan, -2.0, np.nan]
    s = Select(_logits(rng, 4, 3, 20011), scores, 6, dtype)
    s.run()
    got, _ = s.check()
    assert (got[1][2] == -1).all() and (got[5][2] == -1).all() and (got[1][3] // 3 == 3).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_banned_tokens(dev, dtype):
    """Most tokens banned, by -inf, by NaN and by the type's lowest value, whole
    chunks among them; rows with fewer candidates than asked for, and with none."""
    rng = np.random.default_rng(4)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[dtype]
    x = _logits(rng, 6, 2, 25000)
    x[0][rng.random(x[0].shape) < 0.99] = -np.inf
    x[1][:, 500:] = low
    x[2][:, :24000] = np.nan
    x[3] = -np.inf
    x[3, 1, 8191:8194] = [1.0, 1.0, -2.0]
    x[4] = low
    x[4, 0, 24999] = 2.0
    x[5] = -np.inf
    s = Select(x, -rng.random((6, 2)), 4, dtype)
    s.run()
    got, _ = s.check()
    assert got[2][3].tolist() == [8191, 8192, 8193, -1] and (got[2][5] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_nothing_but_the_lowest_value(dev, dtype):
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[dtype]
    s = Select(np.full((1, 2, 9000), low, np.float32), [[0.0, -1.0]], 3, dtype)
    s.run()
    got, _ = s.check()
    assert got[2][0].tolist() == [0, 1, 2] and np.allclose(got[0], -np.log(9000), atol=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_large_and_infinite_logits(dev, dtype):
    rng = np.random.default_rng(5)
    x = _logits(rng, 3, 2, 10000)
    x[0, 0, [17, 9000]] = np.inf
    x[1] *= 1e37 if dtype == "f32" else 5000
    x[2, 1, 5] = 3.3e38 if dtype == "f32" else 65504
    with np.errstate(over="ignore"):
        s = Select(x, [[-1.0, -2.0]] * 3, 4, dtype)
    s.run()
    got, _ = s.check()
    assert got[2][0][:2].tolist() == [17, 9000]


@pytest.mark.parametrize("R,W,V,C", [(2, 4, 30000, 8), (1, 64, 9000, 64), (3, 1, 130, 64), (1, 3, 70000, 50)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties(dev, dtype, R, W, V, C):
    """Equal logits everywhere, and few distinct ones: the lower token; equal beams: the lower beam."""
    for x in (np.zeros((R, W, V), np.float32), np.full((R, W, V), -0.0, np.float32),
              np.random.default_rng(1).integers(0, 3, (R, W, V)).astype(np.float32)):
        s = Select(x, np.zeros((R, W)), C, dtype)
        s.run()
        got, want = s.check()
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
        assert np.array_equal(got[4], want[4]) and np.array_equal(got[5], want[5])


def test_signed_zeros_tie(dev):
    x = np.full((1, 1, 9000), -5.0, np.float32)
    x[0, 0, [3, 100, 8500]] = [-0.0, 0.0, -0.0]
    s = Select(x, [[0.0]], 2)
    s.run()
    assert s.check()[0][2].tolist() == [[3, 100]]


@pytest.mark.parametrize("C", [4, 6, 8])
def test_end_token(dev, C):
    """Every beam's best token ends it; what goes on comes of the rest, as far as there are candidates."""
    rng = np.random.default_rng(6)
    x = _logits(rng, 3, 4, 1000)
    x[:, :, 77] = 30.0
    s = Select(x, -rng.random((3, 4)), C, eos=77)
    s.run()
    got, _ = s.check()
    assert (got[2][:, :4] == 77).all() and (got[5] != 77).all()
    assert ((got[5] >= 0).sum(1) == C - 4).all()


def test_scores_in_place_and_in_a_graph(dev):
    """next_scores in beam_scores' place, step after step in a captured graph; another stream; two workspaces."""
    rng = np.random.default_rng(7)
    R, W, V, C = 3, 4, 12000, 8
    stream = Stream()
    a = Select(_logits(rng, R, W, V), np.zeros((R, W)), C, "bf16", eos=5)
    b = Select(_logits(rng, 1, 2, 500), np.zeros((1, 2)), 4)
    a.out[3] = a.d_s

    def enqueue():
        a.run(stream)
        b.run(stream)

    enqueue()
    stream.synchronize()
    a.d_s.upload(a.scores)
    g = Graph(stream, enqueue)
    for step in range(4):
        x = _logits(rng, R, W, V)
        a.d_x.upload(to_half(x.reshape(-1), "bf16"))
        a.x = to_float(to_half(x, "bf16"), "bf16").reshape(x.shape)
        synchronize()
        g.launch(stream)
        stream.synchronize()
        a.check()
        b.check()
        a.scores = a.d_s.numpy().reshape(R, W)


def test_no_requests(dev):
    s = Select(np.zeros((1, 2, 10), np.float32), [[0, 0]], 2)
    bs.beam_select(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 2, 10, 2)
    s.run()
    s.check()


def test_random_sweep(dev):
    rng = np.random.default_rng(8)
    for _ in range(40):
        W = int(rng.integers(1, 17))
        C = min(64, W * int(rng.integers(1, 4)))
        V = int(np.exp(rng.uniform(0, np.log(30000))))
        R = int(rng.integers(1, 5))
        dtype = ["f32", "f16", "bf16"][rng.integers(3)]
        x = _logits(rng, R, W, V, float(rng.choice([0.1, 2.0, 10.0])))
        x[rng.random(x.shape) < rng.choice([0.0, 0.5, 0.98])] = -np.inf
        s = Select(x, -20 * rng.random((R, W)), C, dtype, eos=int(rng.integers(-1, V)),
                   stride=V + int(rng.integers(0, 9)), shift=int(rng.integers(0, 9)))
        print(R, W, V, C, dtype, flush=True)
        s.run()
        s.check()
