"""The measured operators of one attention step around the paged cache, as
swiftllm_amd.attention_step offers them: the step's block tables and slot maps
from request lengths, rotary positions fused with the cache write, and paged
attention of one new token and of packed prompts whose scores are capped,
biased by distance, windowed or opened to a prefix.

`own` False computes each in elementary torch operations, True calls the
library's kernels. A case fixes every size, the sequence lengths included; a
seed gives the values, the block ids and the order of the free list.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BS = 16                      # tokens per cache block
DEV = "cuda"
F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}

# (query heads, kv heads, head_dim): a small MHA model, 8B- and 70B-like GQA
# layers, and a wide MHA layer.
HEADS = [(8, 8, 64), (32, 8, 128), (64, 8, 128), (16, 16, 128)]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _heads(i: int) -> dict:
    H, Hkv, D = HEADS[i]
    return {"heads": H, "kv_heads": Hkv, "head_dim": D}


def _score(cap: float = 0.0, alibi: bool = False, window: int = 0, prefix: int = 0) -> dict:
    """cap: soft cap of the scores, 0 for none; prefix: the longest prefix of a
    sequence that every query sees."""
    return {"cap": cap, "alibi": alibi, "window": window, "prefix": prefix}


def listed() -> list[dict]:
    return [
        # A server's decode step: 64 chats, one new token each; one in 16 opens a block.
        {"name": "plan_chat_step", "kind": "plan", "seqs": 64, "cached": 4096, "new": 1,
         "chunk_share": 0.0, "pad": 0, "lens_seed": 1},
        # Long documents of 32 requests taken in at once, between decode steps, padded rows behind.
        {"name": "plan_ingest", "kind": "plan", "seqs": 64, "cached": 8192, "new": 16384,
         "chunk_share": 0.5, "pad": 1000, "lens_seed": 2},
        # The new tokens of 64 chats: q, k and v of one fused projection, lone cache columns.
        {"name": "rotary_chat_step", "kind": "rotary", **_heads(1), "dtype": "f16", "tokens": 64,
         "run": 1, "rotary_dim": 128, "interleaved": False, "far": 8192, "stretch": 1.0,
         "fused": True},
        # A batch of prompts on the same layer, frequencies stretched for long contexts.
        {"name": "rotary_prompts", "kind": "rotary", **_heads(1), "dtype": "bf16",
         "tokens": 16384, "run": 1365, "rotary_dim": 128, "interleaved": False, "far": 131072,
         "stretch": 8.0, "fused": True},
        # Half of a small head rotated in adjacent pairs, positions of a very long document.
        {"name": "rotary_partial_far", "kind": "rotary", **_heads(0), "dtype": "f16",
         "tokens": 2013, "run": 671, "rotary_dim": 32, "interleaved": True, "far": 1000003,
         "stretch": 1.0, "fused": False},
        # A handful of short chats on a small model with distance biases: latency.
        {"name": "decode_tiny_alibi", "kind": "decode", **_heads(0), "dtype": "f16", "seqs": 4,
         "dist": "uniform", "lo": 1, "hi": 256, "lens_seed": 3, **_score(alibi=True)},
        # The steady state of a server whose model caps its scores.
        {"name": "decode_batch_cap", "kind": "decode", **_heads(1), "dtype": "bf16", "seqs": 64,
         "dist": "uniform", "lo": 512, "hi": 4096, "lens_seed": 4, **_score(cap=50.0)},
        # A layer with a sliding window that keeps the first tokens in sight; ragged contexts.
        {"name": "decode_window_ragged", "kind": "decode", **_heads(1), "dtype": "f16",
         "seqs": 128, "dist": "lognormal", "lo": 1, "hi": 8192, "lens_seed": 5,
         **_score(window=1024, prefix=4)},
        # Few very long contexts on a 70B-like layer: the cache's length has to be split.
        {"name": "decode_long_cap", "kind": "decode", **_heads(2), "dtype": "f16", "seqs": 8,
         "dist": "uniform", "lo": 32768, "hi": 32768, "lens_seed": 6, **_score(cap=30.0)},
        # Mixed instructions whose first part is read in both directions, with distance biases.
        {"name": "prefill_prefix_ragged", "kind": "prefill", **_heads(3), "dtype": "f16",
         "seqs": 24, "dist": "lognormal", "lo": 1, "hi": 2048, "lens_seed": 7, "cached": 0,
         **_score(alibi=True, prefix=200)},
        # A full batch of long prompts with capped scores.
        {"name": "prefill_batch_cap", "kind": "prefill", **_heads(1), "dtype": "bf16", "seqs": 8,
         "dist": "uniform", "lo": 2048, "hi": 2048, "lens_seed": 8, "cached": 0,
         **_score(cap=50.0)},
        # Chunks of long documents on top of what is cached, in a windowed layer.
        {"name": "prefill_chunk_window", "kind": "prefill", **_heads(1), "dtype": "f16",
         "seqs": 4, "dist": "uniform", "lo": 1000, "hi": 1024, "lens_seed": 9, "cached": 7500,
         **_score(window=4096)},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    """An integer in [lo, hi], even over its logarithm; odd as often as even."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _draw_score(rng: random.Random, most: int) -> dict:
    prefix = _log_int(rng, 1, max(1, most)) if rng.random() < 0.35 else 0
    return _score(cap=rng.choice([0.0, 0.0, 15.0, 30.0, 50.0]), alibi=rng.random() < 0.4,
                  window=_log_int(rng, 1, 8192) if rng.random() < 0.4 else 0, prefix=prefix)


def draw(rng: random.Random) -> dict:
    """One more case of the same ranges, bounded by the largest listed ones."""
    kind = rng.choice(["plan", "rotary", "rotary", "decode", "decode", "decode", "prefill",
                       "prefill"])
    seed = rng.randrange(1 << 20)
    if kind == "plan":
        seqs = _log_int(rng, 1, 2048)
        new = _log_int(rng, 1, max(1, 524288 // seqs))
        return {"kind": kind, "seqs": seqs, "cached": _log_int(rng, 1, 32768), "new": new,
                "chunk_share": rng.choice([0.0, 0.1, 0.5, 1.0]), "pad": rng.choice([0, 1, 77]),
                "lens_seed": seed}
    h = rng.randrange(len(HEADS))
    H, Hkv, D = HEADS[h]
    dtype = rng.choice(["f16", "bf16"])
    if kind == "rotary":
        tokens = _log_int(rng, 1, 16384 * 40 // (H + Hkv))
        return {"kind": kind, **_heads(h), "dtype": dtype, "tokens": tokens,
                "run": rng.choice([1, 1, 2, 5]) if rng.random() < 0.4 else _log_int(rng, 6, 4096),
                "rotary_dim": rng.choice([D, D, D // 2, D // 4]),
                "interleaved": rng.random() < 0.4, "far": _log_int(rng, 4096, 1 << 20),
                "stretch": rng.choice([1.0, 4.0, 8.0, 32.0]), "fused": rng.random() < 0.6}
    if kind == "decode":
        seqs = _log_int(rng, 1, 256)
        most = min(32768, (1 << 30) // (seqs * Hkv * D * 4))   # at most 1 GiB of K and V
        hi = _log_int(rng, 1, most)
        dist = rng.choice(["uniform", "uniform", "lognormal"])
        lo = 1 if dist == "lognormal" else max(1, hi // rng.choice([1, 2, 8, 64]))
        return {"kind": kind, **_heads(h), "dtype": dtype, "seqs": seqs, "dist": dist, "lo": lo,
                "hi": hi, "lens_seed": seed, **_draw_score(rng, 300)}
    # at most 2^30 scores in the padded batch of the plain form
    hi = _log_int(rng, 16, 4096)
    cached = _log_int(rng, 1, 16384) if rng.random() < 0.4 else 0
    while H * hi * (hi + cached) > 1 << 30:
        hi, cached = max(16, hi // 2), cached // 2
    seqs = _log_int(rng, 1, max(1, min(48, (1 << 30) // (H * hi * (hi + cached)))))
    dist = rng.choice(["uniform", "lognormal"])
    lo = 1 if dist == "lognormal" else max(1, hi // rng.choice([1, 2, 8]))
    return {"kind": kind, **_heads(h), "dtype": dtype, "seqs": seqs, "dist": dist, "lo": lo,
            "hi": hi, "lens_seed": seed, "cached": cached, **_draw_score(rng, hi)}


def _lens(case: dict) -> list[int]:
    """The new tokens (prefill) or the contexts (decode) of a case's sequences;
    part of its size, not of its data."""
    r = random.Random(case["lens_seed"])
    lo, hi = case["lo"], case["hi"]
    if case["dist"] == "lognormal":
        median = 600.0 if case["kind"] == "decode" else 300.0
        return [min(hi, max(lo, round(math.exp(r.gauss(math.log(median), 1.0)))))
                for _ in range(case["seqs"])]
    return [r.randint(lo, hi) for _ in range(case["seqs"])]


def _cached(case: dict) -> list[int]:
    """Tokens of each prefill sequence that are in the cache before its chunk."""
    r = random.Random(case["lens_seed"] + 1)
    return [r.randint(case["cached"] // 2, case["cached"]) for _ in range(case["seqs"])]


def _prefixes(case: dict) -> list[int]:
    r = random.Random(case["lens_seed"] + 2)
    return [r.randint(0, case["prefix"]) for _ in range(case["seqs"])]


def _plan_lens(case: dict) -> tuple[list[int], list[int]]:
    """(cached, new) tokens of each request: a share takes in a chunk, the others one token."""
    r = random.Random(case["lens_seed"])
    chunks = round(case["chunk_share"] * case["seqs"])
    cached = [r.randint(0, case["cached"]) for _ in range(case["seqs"])]
    new = [r.randint(1, case["new"]) if i < chunks else 1 for i in range(case["seqs"])]
    r.shuffle(new)
    return cached, new


def _blocks(n: int) -> int:
    return (n + BS - 1) // BS


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g: torch.Generator, dtype, *shape, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _tables(g: torch.Generator, need: list[int], spare: float = 1.25):
    """(block tables int32 [S, MB] over a random permutation of the pool, blocks of the pool)."""
    MB, NB = max(max(need), 1), max(1, math.ceil(spare * sum(need)))
    perm = torch.randperm(NB, generator=g, device=DEV).to(I32)
    nb = torch.tensor(need, dtype=I64, device=DEV)
    col = torch.arange(MB, device=DEV)
    first = torch.cumsum(nb, 0) - nb
    bt = torch.where(col < nb[:, None], perm[(first[:, None] + col).clamp_(max=NB - 1)], 0)
    return bt.to(I32).contiguous(), NB


def _inv_freq(case: dict) -> torch.Tensor:
    """Radians a position turns each pair, float64; a stretch divides the slow
    half of the frequencies (wavelengths above the trained context)."""
    half = case["rotary_dim"] // 2
    f = 500000.0 ** (-torch.arange(half, dtype=F64, device=DEV) / half)
    return torch.where(2.0 * math.pi / f > 8192.0, f / case["stretch"], f).contiguous()


def _plan_state(case: dict, seed: int) -> dict:
    g = _gen(seed)
    cached, new = _plan_lens(case)
    have = [_blocks(c) for c in cached]
    need = [_blocks(c + n) - b for c, n, b in zip(cached, new, have)]
    S, T = case["seqs"], sum(new) + case["pad"]
    MB = max(h + n for h, n in zip(have, need)) + 2
    NB = math.ceil(1.25 * (sum(have) + sum(need))) + 1
    perm = torch.randperm(NB, generator=g, device=DEV).to(I32)
    hv = torch.tensor(have, dtype=I64, device=DEV)
    col = torch.arange(MB, device=DEV)
    first = torch.cumsum(hv, 0) - hv
    bt = torch.where(col < hv[:, None], perm[(first[:, None] + col).clamp_(max=NB - 1)], 0)
    free = perm[sum(have):].contiguous()
    return dict(S=S, T=T, MB=MB, NB=NB, F=free.numel(), bt=bt.to(I32).contiguous(), free=free,
                nfree=torch.tensor([free.numel()], dtype=I32, device=DEV),
                cached=torch.tensor(cached, dtype=I32, device=DEV),
                new=torch.tensor(new, dtype=I32, device=DEV))


def _rotary_state(case: dict, seed: int) -> dict:
    """Tokens in runs of `run` positions, each run at a place of its own of a
    document of `far` positions; the pool holds the blocks of the runs."""
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    H, Hkv, D, T, run = (case[k] for k in ("heads", "kv_heads", "head_dim", "tokens", "run"))
    runs = -(-T // run)
    start = torch.randint(0, max(1, case["far"] - run), (runs,), generator=g, device=DEV)
    t = torch.arange(T, device=DEV)
    i = t // run
    pos = start[i] + t % run
    per = _blocks(run) + 1                      # blocks a run can touch
    NB = math.ceil(1.1 * runs * per)
    perm = torch.randperm(NB, generator=g, device=DEV)
    block = perm[i * per + pos // BS - start[i] // BS]
    s = dict(T=T, NB=NB, pos=pos.to(I32), slots=(block * BS + pos % BS).to(I32),
             inv_freq=_inv_freq(case), factor=1.0 + 0.1 * math.log(case["stretch"]))
    if case["fused"]:
        qkv = _normal(g, dt, T, (H + 2 * Hkv) * D)
        s["q"], s["k"], s["v"] = qkv.split([H * D, Hkv * D, Hkv * D], dim=1)
    else:
        s["q"], s["k"], s["v"] = (_normal(g, dt, T, n * D) for n in (H, Hkv, Hkv))
    s["out"] = torch.zeros(T, H, D, dtype=dt, device=DEV)
    s["kc"] = _normal(g, dt, NB, Hkv, D, BS)
    s["vc"] = _normal(g, dt, NB, Hkv, D, BS)
    return s


def _attention_state(case: dict, seed: int) -> dict:
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    H, Hkv, D, S = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    lens = _lens(case)
    d = dict(S=S, H=H, Hkv=Hkv, D=D, scale=1.0 / math.sqrt(D))
    if case["kind"] == "prefill":
        ctx = [c + n for c, n in zip(_cached(case), lens)]
        d["lens"], d["T"] = lens, sum(lens)
        d["qoff"] = torch.tensor([sum(lens[:i]) for i in range(S + 1)], dtype=I32, device=DEV)
    else:
        ctx = lens
    d["ctx_list"] = ctx
    d["bt"], d["NB"] = _tables(g, [_blocks(n) for n in ctx])
    d["MB"] = d["bt"].shape[1]
    d["ctx"] = torch.tensor(ctx, dtype=I32, device=DEV)
    d["kc"] = _normal(g, dt, d["NB"], Hkv, D, BS)
    d["vc"] = _normal(g, dt, d["NB"], Hkv, D, BS)
    # scores of some size, as after training: sigma about 4 before the cap
    d["q"] = _normal(g, dt, S if case["kind"] == "decode" else d["T"], H, D, std=4.0)
    d["slopes"] = d["prefix"] = None
    if case["alibi"]:
        d["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=F32, device=DEV) / H)
    if case["prefix"]:
        d["prefix"] = torch.tensor(_prefixes(case), dtype=I32, device=DEV)
    return d


def prepare(case: dict, seed: int) -> dict:
    if case["kind"] == "plan":
        s = _plan_state(case, seed)
        S, T = s["S"], s["T"]
        empty = lambda n: torch.empty(n, dtype=I32, device=DEV)  # noqa: E731
        s["out"] = {"block_tables": s["bt"], "context_lens": empty(S),
                    "query_offsets": empty(S + 1), "positions": empty(T),
                    "slot_mapping": empty(T), "counts": empty(3)}
    elif case["kind"] == "rotary":
        s = _rotary_state(case, seed)
    else:
        s = _attention_state(case, seed)
        s["out"] = torch.zeros_like(s["q"])
    s["case"] = case
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_plan(s: dict) -> dict:
    T, MB, bt = s["T"], s["MB"], s["bt"]
    cached, new = s["cached"].to(I64), s["new"].to(I64)
    valid = (cached >= 0) & (new >= 0) & (cached + new <= MB * BS)
    have = (cached + BS - 1) // BS
    need = torch.where(valid, (cached + new + BS - 1) // BS - have, 0)
    taken = torch.cumsum(need, 0)
    tokens = torch.cumsum(torch.where(valid, new, 0), 0)
    fits = (valid & ((need == 0) | (taken <= s["nfree"]))
            & ((new == 0) | (tokens <= T)))
    new, need = torch.where(fits, new, 0), torch.where(fits, need, 0)
    end = torch.cumsum(new, 0)
    first = torch.where(need > 0, taken - need, 0)
    col = torch.arange(MB, device=DEV)
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, s["F"] - 1)
    bt.copy_(torch.where(fresh, s["free"][at], bt))
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(end, t, right=True).clamp(max=s["S"] - 1)
    real = t < end[-1]
    pos = torch.where(real, cached[row] + t - (end - new)[row], -1)
    block = bt[row, pos.clamp(min=0) // BS].to(I64)
    known = real & (block >= 0) & (block < s["NB"])
    out = s["out"]
    out["context_lens"].copy_(cached + new)
    out["query_offsets"][:1].zero_()
    out["query_offsets"][1:].copy_(end)
    out["positions"].copy_(pos)
    out["slot_mapping"].copy_(torch.where(known, block * BS + pos % BS, -1))
    out["counts"].copy_(torch.stack([torch.where(need > 0, taken, 0).amax(), end[-1],
                                     (~fits).sum()]))
    return out


def _turn(x, cos, sin, half: int, interleaved: bool):
    """x [T, heads, D] with its first 2 * half values rotated."""
    rot = x[..., :2 * half]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., 2 * half:]], -1)


def _plain_rotary(s: dict) -> dict:
    case = s["case"]
    H, Hkv, D, half = (case["heads"], case["kv_heads"], case["head_dim"], case["rotary_dim"] // 2)
    angle = s["pos"].to(F64)[:, None] * s["inv_freq"]
    cos = (torch.cos(angle) * s["factor"]).to(F32)[:, None]
    sin = (torch.sin(angle) * s["factor"]).to(F32)[:, None]
    q = _turn(s["q"].reshape(-1, H, D).to(F32), cos, sin, half, case["interleaved"])
    k = _turn(s["k"].reshape(-1, Hkv, D).to(F32), cos, sin, half, case["interleaved"])
    s["out"].copy_(q)
    b, o = s["slots"].to(I64) // BS, s["slots"].to(I64) % BS
    s["kc"][b, :, :, o] = k.to(s["kc"].dtype)
    s["vc"][b, :, :, o] = s["v"].reshape(-1, Hkv, D)
    return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}


def _plain_attention(s: dict):
    """The padded batch at once: every sequence's keys gathered to the longest
    table, scores in 32 bits, masked, normalised, times the values."""
    case = s["case"]
    S, H, Hkv, D, MB = s["S"], s["H"], s["Hkv"], s["D"], s["MB"]
    G = H // Hkv
    L = MB * BS
    k = s["kc"][s["bt"].to(I64)].permute(0, 2, 3, 1, 4).reshape(S, Hkv, D, L).to(F32)
    ctx = s["ctx"].to(I64)
    if case["kind"] == "decode":
        n, q = 1, s["q"].to(F32).view(S, 1, H, D)
        pos = (ctx - 1)[:, None]
    else:
        n = max(s["lens"])
        count = (s["qoff"][1:] - s["qoff"][:-1]).to(I64)
        i = torch.arange(n, device=DEV)
        rows = (s["qoff"][:-1].to(I64)[:, None] + i).clamp(max=s["T"] - 1)
        q = s["q"][rows].to(F32)
        pos = (ctx - count)[:, None] + i
    q = q.view(S, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * n, D)
    x = (torch.matmul(q, k) * s["scale"]).view(S, Hkv, G, n, L)
    del k
    key = torch.arange(L, device=DEV)
    slopes = None if s["slopes"] is None else s["slopes"].view(1, Hkv, G, 1, 1)
    prefix = None if s["prefix"] is None else s["prefix"].to(I64).view(S, 1, 1, 1, 1)
    pos = pos.view(S, 1, 1, n, 1)
    if case["cap"] > 0:
        x = case["cap"] * torch.tanh(x / case["cap"])
    if slopes is not None:
        x = x - slopes * (pos - key).abs()
    seen = key <= pos
    if case["window"] > 0:
        seen = seen & (pos - key < case["window"])
    if prefix is not None:
        seen = seen | (key < prefix)
    seen = seen & (key < ctx.view(S, 1, 1, 1, 1))
    x = x.masked_fill(~seen, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    total = x.sum(-1, keepdim=True)
    v = s["vc"][s["bt"].to(I64)].permute(0, 2, 1, 4, 3).reshape(S, Hkv, L, D).to(F32)
    y = torch.matmul(x.view(S, Hkv, G * n, L), v).view(S, Hkv, G, n, D)
    y = torch.where(total > 0, y / total, 0.0)
    y = y.permute(0, 3, 1, 2, 4).reshape(S, n, H, D)
    if case["kind"] == "decode":
        s["out"].copy_(y.view(S, H, D))
    else:
        t = torch.arange(s["T"], device=DEV)
        row = torch.searchsorted(s["qoff"][1:].to(I64), t, right=True)
        s["out"].copy_(y[row, t - s["qoff"].to(I64)[row]])
    return s["out"]


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_run(s: dict):
    from swiftllm_amd import attention_step as step
    case = s["case"]
    if case["kind"] == "plan":
        o = s["out"]
        step.plan_step(_ptr(o["block_tables"]), _ptr(s["cached"]), _ptr(s["new"]), _ptr(s["free"]),
                       _ptr(s["nfree"]), s["F"], s["S"], s["MB"], BS, s["T"],
                       _ptr(o["context_lens"]), _ptr(o["query_offsets"]), _ptr(o["positions"]),
                       _ptr(o["slot_mapping"]), _ptr(o["counts"]), num_blocks=s["NB"])
        return o
    if case["kind"] == "rotary":
        step.rotary_and_cache(_ptr(s["out"]), _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]),
                              _ptr(s["kc"]), _ptr(s["vc"]), _ptr(s["pos"]), _ptr(s["slots"]),
                              _ptr(s["inv_freq"]), s["T"], case["heads"], case["kv_heads"],
                              case["head_dim"], case["rotary_dim"], BS, dtype=case["dtype"],
                              attn_factor=s["factor"], interleaved=case["interleaved"],
                              query_stride=s["q"].stride(0), key_stride=s["k"].stride(0),
                              value_stride=s["v"].stride(0), num_blocks=s["NB"])
        return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}
    score = step.ScoreParams(scale=s["scale"], softcap=case["cap"], window=case["window"],
                             alibi_slopes=_ptr(s["slopes"]), prefix_lens=_ptr(s["prefix"]))
    if case["kind"] == "decode":
        if "ws" not in s:    # kept for the sizes, as a server does
            n = step.scored_decode_workspace_size(s["S"], s["H"], s["Hkv"], s["D"], BS, s["MB"])
            s["ws"] = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)
        step.scored_decode(_ptr(s["out"]), _ptr(s["ws"]), s["ws"].numel(), _ptr(s["q"]),
                           _ptr(s["kc"]), _ptr(s["vc"]), _ptr(s["bt"]), _ptr(s["ctx"]), score,
                           s["S"], s["H"], s["Hkv"], s["D"], BS, s["MB"], dtype=case["dtype"],
                           num_blocks=s["NB"])
    else:
        step.scored_prefill(_ptr(s["out"]), _ptr(s["q"]), _ptr(s["kc"]), _ptr(s["vc"]),
                            _ptr(s["bt"]), _ptr(s["ctx"]), _ptr(s["qoff"]), score, s["T"], s["S"],
                            s["H"], s["Hkv"], s["D"], BS, s["MB"], dtype=case["dtype"],
                            num_blocks=s["NB"])
    return s["out"]


def run(s: dict):
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "plan":
        return _plain_plan(s)
    if kind == "rotary":
        return _plain_rotary(s)
    return _plain_attention(s)


# ---------------------------------------------------------------------------
# What one pass cannot do without
# ---------------------------------------------------------------------------
def _seen(case: dict, pos: int, ctx: int, prefix: int) -> int:
    """Keys the query at position pos sees."""
    low = max(0, pos + 1 - case["window"]) if case["window"] > 0 else 0
    prefix = min(prefix, ctx)
    return pos + 1 - low + min(prefix, low) + max(0, prefix - (pos + 1))


def work(case: dict) -> dict:
    if case["kind"] == "plan":
        cached, new = _plan_lens(case)
        need = sum(_blocks(c + n) - _blocks(c) for c, n in zip(cached, new))
        opened = sum(c % BS != 0 for c in cached)        # ids of blocks that a run begins in
        S, T = case["seqs"], sum(new) + case["pad"]
        return {"bytes": 8 * S + 8 * need + 4 * opened + 8 * S + 8 * T + 20, "flops": 0}
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rotary":
        T = case["tokens"]
        return {"bytes": T * (4 * H * D + 8 * Hkv * D + 8) + 4 * case["rotary_dim"],
                "flops": 3 * T * (H + Hkv) * case["rotary_dim"]}
    lens = _lens(case)
    prefix = _prefixes(case) if case["prefix"] else [0] * case["seqs"]
    rows = case["seqs"] if case["kind"] == "decode" else sum(lens)
    keys = pairs = blocks = 0
    cached = [n - 1 for n in lens] if case["kind"] == "decode" else _cached(case)
    for n, c, p in zip(lens, cached, prefix):
        first, ctx = c, c + (1 if case["kind"] == "decode" else n)
        low = max(0, first + 1 - case["window"]) if case["window"] > 0 else 0
        union = ctx - low + min(min(p, ctx), low)         # keys that some query sees
        keys += union
        blocks += _blocks(union)
        pairs += sum(_seen(case, i, ctx, p) for i in range(first, ctx))
    return {"bytes": 4 * rows * H * D + 4 * keys * Hkv * D + 4 * blocks + 4 * case["seqs"],
            "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotary(case: dict, seed: int) -> dict:
    s = _rotary_state(case, seed)
    H, Hkv, D, R = case["heads"], case["kv_heads"], case["head_dim"], case["rotary_dim"]
    i = torch.arange(R // 2, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2)
    turn = torch.polar(torch.full_like(s["inv_freq"], s["factor"]).expand(s["T"], -1),
                       s["pos"].to(F64)[:, None] * s["inv_freq"])[:, None]

    def rotated(x, heads):
        x = x.reshape(-1, heads, D).to(F64)
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    kc, vc = s["kc"].to(F64), s["vc"].to(F64)
    at = s["slots"].to(I64)
    kc[at // BS, :, :, at % BS] = rotated(s["k"], Hkv)
    vc[at // BS, :, :, at % BS] = s["v"].reshape(-1, Hkv, D).to(F64)
    return {"q": rotated(s["q"], H), "kc": kc, "vc": vc}


def exact(case: dict, seed: int):
    if case["kind"] == "plan":
        return None
    if case["kind"] == "rotary":
        return _exact_rotary(case, seed)
    s = _attention_state(case, seed)
    H, Hkv, D = s["H"], s["Hkv"], s["D"]
    G = H // Hkv
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    lens = s["lens"] if case["kind"] == "prefill" else [1] * s["S"]
    prefix = _prefixes(case) if case["prefix"] else None
    at = 0
    for i, (n, ctx) in enumerate(zip(lens, s["ctx_list"])):
        ids = s["bt"][i, :_blocks(ctx)].to(I64)
        k = s["kc"][ids].permute(1, 2, 0, 3).reshape(Hkv, D, -1)[:, :, :ctx].to(F64)
        v = s["vc"][ids].permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :ctx].to(F64)
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            # how far back each key lies; negative: ahead of the query
            back = (torch.arange(ctx - n + a, ctx - n + b, device=DEV)[:, None]
                    - torch.arange(ctx, device=DEV))
            hidden = (back < 0) | (back >= (case["window"] or ctx + 1))
            if prefix:
                hidden[:, :prefix[i]] = False
            q = s["q"][at + a:at + b].to(F64)
            for h in range(H):
                x = torch.mm(q[:, h].contiguous(), k[h // G].contiguous()).mul_(s["scale"])
                if case["cap"] > 0:
                    e = torch.expm1(x * (2.0 / case["cap"]))     # tanh(y) = (e^2y - 1) / (e^2y + 1)
                    x = case["cap"] * e / (e + 2.0)
                if case["alibi"]:
                    x.addcmul_(s["slopes"][h].to(F64), back.abs().to(F64), value=-1.0)
                p = torch.softmax(x.masked_fill_(hidden, -math.inf), -1)
                out[at + a:at + b, h] = torch.mm(p, v[h // G].contiguous())
        at += n
    return out
