"""rotary_and_cache on the GPU against the oracle in float64.

Tolerance: the rotated value is one rounding to the type (half a step of the
value) of a 32-bit sum of two products, whose sine and cosine come from the
hardware's 32-bit functions (absolute error below 2^-19) of an angle reduced
in 64 bits. Values and everything that is not written are compared bit by bit."""

import numpy as np
import pytest

import oracle
from step_helpers import HALF_STEP, NAN16, TINY, normal, to_float
from swiftllm_amd import attention_step as step
from swiftllm_amd._hip import DeviceArray, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Case:
    """Tokens at `positions` with `slots` in a pool of NB blocks; q, k and v as
    three views of one buffer (fused) or packed rows `extra` elements apart."""

    def __init__(self, rng, positions, slots, H, Hkv, D, rot, dtype, interleaved=False, fused=True,
                 extra=0, shift=0, factor=1.0, NB=None, base=10000.0):
        self.pos, self.slots = np.asarray(positions, np.int32), np.asarray(slots, np.int32)
        T = len(self.pos)
        self.T, self.H, self.Hkv, self.D, self.rot, self.dtype = T, H, Hkv, D, rot, dtype
        self.inter, self.factor = interleaved, factor
        self.NB = NB or int(max(self.slots.max(initial=0), 0)) // 16 + 2
        self.inv = base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
        widths = [H * D, Hkv * D, Hkv * D]
        if fused:
            row = sum(widths) + extra
            buf = normal(rng, T * row + shift, dtype)
            at = np.cumsum([0] + widths[:-1]) + shift
            self.strides = [row] * 3
            self.bufs = [buf]
            self.device = [DeviceArray.from_numpy(buf)]
            self.ptrs = [self.device[0].ptr + 2 * int(a) for a in at]
            host = [np.lib.stride_tricks.as_strided(buf[a:], (T, w), (2 * row, 2)) for a, w in zip(at, widths)]
        else:
            self.strides = [w + extra for w in widths]
            self.bufs = [normal(rng, T * s + shift, dtype) for s in self.strides]
            self.device = [DeviceArray.from_numpy(b) for b in self.bufs]
            self.ptrs = [d.ptr + 2 * shift for d in self.device]
            host = [np.lib.stride_tricks.as_strided(b[shift:], (T, w), (2 * s, 2))
                    for b, w, s in zip(self.bufs, widths, self.strides)]
        self.q, self.k, self.v = (h.reshape(T, n, D).copy() for h, n in zip(host, (H, Hkv, Hkv)))
        self.kc, self.vc = (np.full((self.NB, Hkv, D, 16), NAN16, np.uint16) for _ in range(2))
        self.d_pos, self.d_slots = DeviceArray.from_numpy(self.pos), DeviceArray.from_numpy(self.slots)
        self.d_inv = DeviceArray.from_numpy(self.inv if rot else np.zeros(1))
        self.d_kc, self.d_vc = DeviceArray.from_numpy(self.kc), DeviceArray.from_numpy(self.vc)
        self.out = DeviceArray((T, H, D), np.uint16)
        self.out.fill_byte(0x77)

    def run(self, stream=None, out=None, bounded=True):
        step.rotary_and_cache(out or self.out, *self.ptrs, self.d_kc, self.d_vc, self.d_pos,
                              self.d_slots, self.d_inv, self.T, self.H, self.Hkv, self.D, self.rot,
                              16, dtype=self.dtype, attn_factor=self.factor, interleaved=self.inter,
                              query_stride=self.strides[0], key_stride=self.strides[1],
                              value_stride=self.strides[2], num_blocks=self.NB if bounded else 0,
                              stream=stream)

    def _close(self, got, x, want, what):
        """got [.., heads, D] patterns against float64 want; x the inputs."""
        y = np.abs(to_float(x, self.dtype).astype(np.float64))
        half = self.rot // 2
        i = np.arange(half)
        a, b = (2 * i, 2 * i + 1) if self.inter else (i, i + half)
        size = np.zeros_like(y)
        size[..., a] = size[..., b] = y[..., a] + y[..., b]
        bound = HALF_STEP[self.dtype] * np.abs(want) + 2.0 ** -19 * self.factor * size + TINY[self.dtype]
        err = np.abs(to_float(got, self.dtype) - want)
        assert (err <= bound).all(), f"{what}: {err.max()} at {np.unravel_index((err - bound).argmax(), err.shape)}"
        rest = np.arange(self.rot, self.D)
        assert np.array_equal(got[..., rest], x[..., rest]), f"{what}: past rotary_dim"

    def check(self, out=None):
        synchronize()
        real = self.pos >= 0
        got = (out or self.out).numpy().reshape(self.T, self.H, self.D)
        q = oracle.rotary(to_float(self.q, self.dtype), self.pos, self.inv, self.rot, self.inter, self.factor)
        k = oracle.rotary(to_float(self.k, self.dtype), self.pos, self.inv, self.rot, self.inter, self.factor)
        self._close(got[real], self.q[real], q[real], "queries")
        left = np.full_like(got[~real], 0x7777) if out is None else self.q[~real]
        assert np.array_equal(got[~real], left), "padding rows of the queries"
        kc, vc = self.d_kc.numpy(), self.d_vc.numpy()
        ok = real & (self.slots >= 0) & (self.slots < 16 * self.NB)
        b, o = self.slots[ok] // 16, self.slots[ok] % 16
        self._close(kc[b, :, :, o], self.k[ok], k[ok], "keys")
        assert np.array_equal(vc[b, :, :, o], self.v[ok]), "values"
        kc[b, :, :, o] = vc[b, :, :, o] = NAN16
        assert (kc == NAN16).all() and (vc == NAN16).all(), "cache outside the slots"


def _runs(rng, lens, far, NB):
    """Positions and slots of runs of tokens, each in blocks of its own."""
    ids = rng.permutation(NB)
    pos, slots, at = [], [], 0
    for n in lens:
        p = np.arange(n) + int(rng.integers(0, far))
        blocks = p // 16 - p[0] // 16 if n else p
        pos += p.tolist()
        slots += (ids[at + blocks] * 16 + p % 16).tolist() if n else []
        at += int(blocks[-1]) + 1 if n else 0
    return pos, slots


HEADS = [(8, 8, 64), (32, 8, 128), (64, 8, 128), (5, 5, 64), (3, 1, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
def test_rotary_layouts_and_heads(dev, H, Hkv, D, interleaved, dtype):
    rng = np.random.default_rng(H + D + interleaved)
    pos, slots = _runs(rng, [1, 15, 16, 17, 40, 1, 1, 3], 5000, 40)
    c = Case(rng, pos, slots, H, Hkv, D, D, dtype, interleaved)
    c.run()
    c.check()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 2, 6, 14, 16, 24, 32, 48, 62, 64])
def test_rotary_part_of_the_head(dev, rot, interleaved):
    """Every kind of rotary_dim: none, whole pieces of 8, and odd halves."""
    rng = np.random.default_rng(rot)
    pos, slots = _runs(rng, [33, 2, 9], 300, 12)
    c = Case(rng, pos, slots, 4, 2, 64, rot, "f16", interleaved, factor=1.0 if rot else 3.0)
    c.run()
    c.check()


@pytest.mark.parametrize("fused,extra,shift", [(True, 0, 0), (True, 8, 0), (True, 1, 0), (True, 0, 3),
                                               (False, 0, 0), (False, 24, 8), (False, 5, 1)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rotary_strides_and_alignment(dev, fused, extra, shift, dtype):
    rng = np.random.default_rng(extra + shift)
    pos, slots = _runs(rng, [20, 1, 31], 77, 12)
    c = Case(rng, pos, slots, 6, 3, 64, 64, dtype, fused=fused, extra=extra, shift=shift)
    c.run()
    c.check()


@pytest.mark.parametrize("T", [1, 3, 64, 513, 600, 1100])
def test_rotary_lone_tokens(dev, T):
    """A decode step: every token in a block of its own, short and long calls."""
    rng = np.random.default_rng(T)
    slots = rng.permutation(T + 5)[:T] * 16 + rng.integers(0, 16, T)
    c = Case(rng, rng.integers(0, 100000, T), slots, 8, 2, 128, 128, "bf16", NB=T + 5)
    c.run()
    c.check()


@pytest.mark.parametrize("lens", [[700, 3, 500], [1] * 20 + [1000], [16] * 40, [2] * 400])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_prompts(dev, lens, interleaved):
    rng = np.random.default_rng(len(lens))
    NB = sum(n // 16 + 2 for n in lens)
    pos, slots = _runs(rng, lens, 4096, NB)
    c = Case(rng, pos, slots, 4, 4, 128, 64, "f16", interleaved, factor=1.35, NB=NB)
    c.run()
    c.check()


@pytest.mark.parametrize("H,D,extra,interleaved", [(24, 64, 0, False), (9, 128, 0, True), (20, 64, 3, False)])
def test_rotary_long_calls(dev, H, D, extra, interleaved):
    """Thousands of tokens, more query heads than a wave takes at once, aligned
    and not, padding among them."""
    rng = np.random.default_rng(H)
    pos, slots = _runs(rng, [4000, 1, 150, 30], 4096, 300)
    pos = np.array(pos)
    pos[[0, 77, 4100, 4180]] = -1
    c = Case(rng, pos, slots, H, 1, D, D, "bf16", interleaved, extra=extra, NB=300)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rotary_far_positions(dev, dtype):
    """Angles of positions up to 2^31 - 1: 32-bit angles would be wrong by turns."""
    pos = np.array([0, 1, 131071, 10 ** 6 + 3, 2 ** 24 + 1, 2 ** 30 + 7, 2 ** 31 - 1])
    c = Case(np.random.default_rng(9), pos, np.arange(7) * 16 + 3, 4, 4, 64, 64, dtype, base=500000.0)
    c.run()
    c.check()


def test_rotary_padding_and_missing_slots(dev):
    """Negative positions leave everything, slots outside the pool the cache."""
    rng = np.random.default_rng(10)
    pos, slots = _runs(rng, [40, 30], 50, 8)
    pos, slots = np.array(pos), np.array(slots)
    pos[[0, 5, 6, 39, 69]] = -1
    slots[[2, 17]] = -1
    slots[[50]] = 16 * 10 + 3
    slots[[51]] = 2 ** 31 - 1
    c = Case(rng, pos, slots, 8, 2, 128, 128, "f16", NB=10)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype,rot,interleaved", [("f16", 64, False), ("bf16", 32, True), ("f16", 22, False)])
def test_rotary_in_place(dev, dtype, rot, interleaved):
    rng = np.random.default_rng(11)
    pos, slots = _runs(rng, [50, 1, 20], 900, 12)
    pos[3] = -1
    c = Case(rng, pos, slots, 8, 4, 64, rot, dtype, interleaved, fused=False)
    c.run(out=c.device[0])
    c.check(out=c.device[0])


def test_rotary_in_place_of_a_long_call(dev):
    rng = np.random.default_rng(12)
    pos, slots = _runs(rng, [4090, 60], 900, 280)
    c = Case(rng, pos, slots, 17, 1, 64, 64, "f16", fused=False, NB=280)
    c.run(out=c.device[0])
    c.check(out=c.device[0])


def test_rotary_values_that_are_not_finite(dev):
    """NaN and infinities stay with their pair and token; past rotary_dim they are copied."""
    rng = np.random.default_rng(12)
    pos, slots = _runs(rng, [18, 1], 900, 6)
    c = Case(rng, pos, slots, 4, 2, 64, 32, "f16", fused=False)
    k, q = c.bufs[1].reshape(19, 2, 64), c.bufs[0].reshape(19, 4, 64)
    k[4, 1, 3], k[7, 0, 40], q[2, 3, 20], q[5, 0, 63] = NAN16, 0x7C00, 0xFC00, NAN16
    c.device[0].upload(c.bufs[0])
    c.device[1].upload(c.bufs[1])
    c.run()
    synchronize()
    got = to_float(c.out.numpy().reshape(19, 4, 64), "f16")
    bad = np.argwhere(~np.isfinite(got)).tolist()
    assert bad == [[2, 3, 4], [2, 3, 20], [5, 0, 63]]
    b, o = c.slots // 16, c.slots % 16
    kc = to_float(c.d_kc.numpy()[b, :, :, o], "f16")
    assert np.argwhere(~np.isfinite(kc)).tolist() == [[4, 1, 3], [4, 1, 19], [7, 0, 40]]


def test_rotary_nothing_to_do(dev):
    c = Case(np.random.default_rng(13), [5], [1], 4, 2, 64, 64, "f16")
    c.T = 0
    c.run()
    synchronize()
    assert (c.d_kc.numpy() == NAN16).all()


def test_rotary_in_a_captured_graph(dev):
    """Replays follow the buffers: new positions, slots and padding each time."""
    rng = np.random.default_rng(14)
    c = Case(rng, np.zeros(48), np.arange(48) * 16, 8, 2, 128, 128, "bf16", NB=60)
    stream = Stream()
    c.run(stream)
    stream.synchronize()
    g = Graph(stream, lambda: c.run(stream))
    for i in range(3):
        c.pos = rng.integers(0, 70000, 48).astype(np.int32)
        c.pos[40 + i:] = -1
        c.slots = (rng.permutation(60)[:48] * 16 + rng.integers(0, 16, 48)).astype(np.int32)
        c.d_pos.upload(c.pos)
        c.d_slots.upload(c.slots)
        c.d_kc.upload(c.kc)
        c.d_vc.upload(c.vc)
        c.out.fill_byte(0x77)
        synchronize()
        g.launch(stream)
        stream.synchronize()
        c.check()
