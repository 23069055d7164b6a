"""scored_decode and scored_prefill give the same for the same single-token
sequences: contexts longer than their tables, whose keys end with the table
while the query keeps its position."""

import numpy as np
import pytest

import oracle
from step_helpers import normal, scored_bound, to_float
from swiftllm_amd import attention_step as step
from swiftllm_amd._hip import DeviceArray, synchronize

pytestmark = pytest.mark.gpu

H, HKV, D = 8, 2, 64


@pytest.mark.parametrize("MB", [3, 300])
@pytest.mark.parametrize("window", [0, 1, 20, 21, 37, 1000])
@pytest.mark.parametrize("kw", [dict(), dict(cap=20.0), dict(prefix=True), dict(alibi=True, prefix=True)])
def test_contexts_past_the_table(dev, MB, window, kw):
    """A window that reaches back into the table, to its last key, or not at
    all; a short table is taken whole by the decode, a wide one in ranges."""
    rng = np.random.default_rng(window + MB)
    L = 16 * MB
    far = L + 5000     # past every window
    ctx = np.array([L, L + 1, L + 20, L + 21, L + 36, L + 2000, L - 5,
                    far if kw.get("alibi") else 2 ** 31 - 1], np.int32)
    S = len(ctx)
    NB = S * MB
    bt = rng.permutation(NB).astype(np.int32).reshape(S, MB)
    kc, vc, q = (normal(rng, s, "f16", 2.0) for s in ((NB, HKV, D, 16), (NB, HKV, D, 16), (S, H, D)))
    prefix = rng.integers(0, 30, S).astype(np.int32) if kw.get("prefix") else None
    slopes = step.alibi_slopes(H) if kw.get("alibi") else None
    score = dict(scale=0.1, softcap=kw.get("cap", 0.0), window=window, slopes=slopes, prefix=prefix)
    off = np.arange(S + 1, dtype=np.int32)
    f = lambda x: to_float(x, "f16")  # noqa: E731
    a = (f(q), f(kc), f(vc), bt, ctx, off)
    want = oracle.scored_attention(*a, **score)
    up = DeviceArray.from_numpy
    d_q, d_k, d_v, d_bt, d_ctx, d_off = (up(x) for x in (q, kc, vc, bt, ctx, off))
    p = step.ScoreParams(0.1, score["softcap"], window, None if slopes is None else up(slopes),
                         None if prefix is None else up(prefix))
    ws = DeviceArray((step.scored_decode_workspace_size(S, H, HKV, D, 16, MB),), np.uint8)
    outs = {}
    for name in ("decode", "rows", "prefill"):
        out = DeviceArray((S, H, D), np.uint16)
        out.fill_byte(0x7F)
        rows = dict(query_offsets=d_off, num_tokens=S) if name == "rows" else {}
        if name == "prefill":
            step.scored_prefill(out, d_q, d_k, d_v, d_bt, d_ctx, d_off, p, S, S, H, HKV, D, 16, MB, num_blocks=NB)
        else:
            step.scored_decode(out, ws, ws.nbytes, d_q, d_k, d_v, d_bt, d_ctx, p, S, H, HKV, D, 16, MB,
                               num_blocks=NB, **rows)
        synchronize()
        outs[name] = f(out.numpy())
    for name, got in outs.items():
        bound = scored_bound(f(q), f(kc), f(vc), bt, np.minimum(ctx, far), off, "f16", 1, want, **score)
        err = np.abs(got - want)
        assert (err <= bound).all(), f"{name}: sequences {np.unique(np.argwhere(~(err <= bound))[:, 0])}"
    assert np.array_equal(outs["decode"], outs["rows"])
