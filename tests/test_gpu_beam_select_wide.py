"""beam_select of requests with more than 64 lists (beams x chunks of 8192 logits),
whose first line is of the lists' maxima, against the oracle in float64 with
test_gpu_beam_select's tolerances (a vocabulary below 2^18)."""

import numpy as np
import pytest

from test_gpu_beam_select import Select, _logits

pytestmark = pytest.mark.gpu

SIZES = [(1, 32, 100003, 64), (2, 4, 150000, 8), (2, 16, 50257, 32), (1, 64, 16391, 64), (1, 9, 65536, 18)]
DTYPES = ["f32", "f16", "bf16"]


def _run(x, scores, C, dtype="f32", **kw):
    s = Select(x, scores, C, dtype, **kw)
    s.run()
    return s.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,W,V,C", SIZES)
def test_scores_apart(dev, dtype, R, W, V, C):
    """Beams near each other and far apart, one of them well ahead."""
    rng = np.random.default_rng(V + W)
    scores = -30 * rng.random((R, W))
    scores[-1, W // 2] = 25.0
    _run(_logits(rng, R, W, V), scores, C, dtype, eos=V // 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ban", [-np.inf, np.nan])
@pytest.mark.parametrize("W,V,C", [(32, 100003, 64), (4, 150000, 8)])
def test_beams_that_allow_nothing(dev, dtype, ban, W, V, C):
    """Rows of nothing but banned tokens, their beams ahead of the others: all but one
    of the beams, whose row allows 1000 tokens, and half of them."""
    rng = np.random.default_rng(11)
    x = _logits(rng, 2, W, V)
    x[0, 1:] = ban
    keep = rng.permutation(V)[:1000]
    row = x[0, 0, keep]
    x[0, 0] = ban
    x[0, 0, keep] = row
    x[1, ::2] = ban
    scores = np.full((2, W), -1.0)
    scores[0, 0] = -20.0
    scores[1, 1::2] = -9.0
    got, _ = _run(x, scores, C, dtype)
    assert (got[2] >= 0).all() and (got[1][0] == 0).all() and (got[1][1] % 2 == 1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_fewer_candidates_than_asked_for(dev, dtype):
    """Allowed tokens of a few beams only, as many as are asked for, fewer, one and none;
    beams without a score among them, and the type's lowest value as a mask."""
    rng = np.random.default_rng(12)
    low = {"f32": -3.4028235e38, "bf16": -3.3895314e38}[dtype]
    W, V, C = 12, 50257, 24
    x = np.full((5, W, V), -np.inf, np.float32)
    for r, n in enumerate((C, C - 1, 1, 0)):
        for k in range(n):
            x[r, 3 + k % 5, rng.integers(0, V // 4) * 4 + k % 4] = rng.standard_normal() * 4
    x[4] = low
    x[4, 7, 100] = 3.0
    scores = -5 * rng.random((5, W))
    scores[:, 5] = -np.inf
    scores[:, 9] = np.nan
    got, _ = _run(x, scores, C, dtype)
    assert (got[1][3] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_infinite_logits(dev, dtype):
    rng = np.random.default_rng(13)
    x = _logits(rng, 2, 8, 80000)
    x[0, 2, [17, 9000, 79999]] = np.inf
    x[1, :, 40000:] = -np.inf
    x[1, 5] = np.inf
    got, _ = _run(x, -3 * rng.random((2, 8)), 16, dtype)
    assert {17, 9000, 79999} <= set(got[2][0][got[1][0] == 2].tolist())


@pytest.mark.parametrize("W,V", [(16, 100003), (64, 170000)])
def test_more_lists_at_the_line_than_are_held(dev, W, V):
    """Every chunk of every beam has the same maximum, so that all lists reach the line:
    more than the threads keep, and more than are listed by name. The rest is all below."""
    rng = np.random.default_rng(14)
    lists = W * -(-V // 8192)
    assert lists > (1024 if W == 64 else 128)
    # (one to a chunk: a chunk's bounds are at most 7 values off)
    row = np.minimum(rng.standard_normal(V).astype(np.float32), 4.0)
    row[100::8192] = 5.0
    # (rows that begin alike within 16 bytes have the same sum, to the bit)
    got, want = _run(np.broadcast_to(row, (1, W, V)), np.zeros((1, W)), 64, stride=-(-V // 8) * 8)
    assert all(np.array_equal(got[k], want[k]) for k in (1, 2, 4, 5))


@pytest.mark.parametrize("C", [16, 64])
def test_many_ties_over_many_lists(dev, C):
    """More equal candidates than are ranked at once: the lower beam, then the lower token."""
    x = np.random.default_rng(15).integers(0, 3, (1, 16, 100003)).astype(np.float32)
    x[0, 1:] = x[0, 0]
    got, want = _run(x, np.zeros((1, 16)), C, stride=100008)
    assert all(np.array_equal(got[k], want[k]) for k in (1, 2, 4, 5))


def test_random_sweep_of_wide_requests(dev):
    rng = np.random.default_rng(16)
    for _ in range(25):
        W = int(rng.integers(3, 65))
        C = min(64, W * int(rng.integers(1, 4)))
        V = int(np.exp(rng.uniform(np.log(65 * 8192 // W + 1), np.log(180000))))
        dtype = DTYPES[rng.integers(3)]
        x = _logits(rng, 1, W, V, float(rng.choice([0.1, 2.0, 10.0])))
        x[rng.random(x.shape) < rng.choice([0.0, 0.5, 0.999])] = -np.inf
        x[0, rng.random(W) < rng.choice([0.0, 0.5])] = np.nan
        scores = -20 * rng.random((1, W))
        scores[rng.random((1, W)) < 0.1] = -np.inf
        print(W, V, C, dtype, flush=True)
        _run(x, scores, C, dtype, eos=int(rng.integers(-1, V)), stride=V + int(rng.integers(0, 9)),
             shift=int(rng.integers(0, 9)))
