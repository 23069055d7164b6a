"""The measured operators of sequences that come of one another over the paged
cache (beams, parallel samples, chats on one system prompt): a beam search's
selection (swiftllm_amd.beam_search), forking and compacting the cache's pages
(swiftllm_amd.pages), and attention that reads what a group of sequences shares
once (swiftllm_amd.attention_step: plan_shared, shared_decode).

`own` False computes each in elementary torch operations, True calls the
library's kernels. A case fixes every size, the sequence lengths included; a
seed gives the values, the block ids and who goes on.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BS = 16                      # tokens per cache block
DEV = "cuda"
F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}

# (query heads, kv heads, head_dim): a small MHA model, 8B- and 70B-like GQA
# layers, and a wide MHA layer.
HEADS = [(8, 8, 64), (32, 8, 128), (64, 8, 128), (16, 16, 128)]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _heads(i: int) -> dict:
    H, Hkv, D = HEADS[i]
    return {"heads": H, "kv_heads": Hkv, "head_dim": D}


def listed() -> list[dict]:
    return [
        # Two short requests of a small model, searched with four beams: latency.
        {"name": "shared_beams_tiny", "kind": "shared", **_heads(0), "dtype": "f16", "groups": 2,
         "each": 4, "shared_lo": 100, "shared_hi": 250, "own_lo": 1, "own_hi": 40, "idle": 0.0,
         "lens_seed": 1, "cap": 0.0, "alibi": False, "layers": 4},
        # Sixteen requests of an 8B-like model that caps its scores, eight beams each.
        {"name": "shared_beams_cap", "kind": "shared", **_heads(1), "dtype": "bf16", "groups": 16,
         "each": 8, "shared_lo": 1000, "shared_hi": 4000, "own_lo": 1, "own_hi": 200, "idle": 0.0,
         "lens_seed": 2, "cap": 50.0, "alibi": False, "layers": 4},
        # 128 chats on one long system prompt, each with a history of its own.
        {"name": "shared_system_prompt", "kind": "shared", **_heads(1), "dtype": "f16",
         "groups": 1, "each": 128, "shared_lo": 8192, "shared_hi": 8192, "own_lo": 1,
         "own_hi": 1000, "idle": 0.05, "lens_seed": 3, "cap": 0.0, "alibi": False, "layers": 4},
        # Questions on four very long documents, a 70B-like layer with distance biases.
        {"name": "shared_documents_alibi", "kind": "shared", **_heads(2), "dtype": "bf16",
         "groups": 4, "each": 16, "shared_lo": 28000, "shared_hi": 32768, "own_lo": 20,
         "own_hi": 1500, "idle": 0.0, "lens_seed": 4, "cap": 0.0, "alibi": True, "layers": 2},
        # One request's four beams, logits in 32 bits: latency.
        {"name": "select_one", "kind": "select", "dtype": "f32", "requests": 1, "beams": 4,
         "candidates": 8, "vocab": 32000, "pad": 0, "first": False, "banned": 0.0, "eos": True},
        # A server's step: 64 requests of four beams.
        {"name": "select_batch", "kind": "select", "dtype": "bf16", "requests": 64, "beams": 4,
         "candidates": 8, "vocab": 128000, "pad": 0, "first": False, "banned": 0.0, "eos": True},
        # Wide search under a grammar that bans most tokens; rows of a padded vocabulary.
        {"name": "select_wide_banned", "kind": "select", "dtype": "f32", "requests": 9,
         "beams": 32, "candidates": 64, "vocab": 100003, "pad": 29, "first": False,
         "banned": 0.8, "eos": True},
        # One request's beams reordered in a small pool: latency.
        {"name": "fork_one", "kind": "fork", "requests": 1, "beams": 4, "shared": 300, "own": 60,
         "pool": 4096, "lens_seed": 5},
        # Sixteen requests of eight beams in the pool of an 8B-like server.
        {"name": "fork_batch", "kind": "fork", "requests": 16, "beams": 8, "shared": 4000,
         "own": 200, "pool": 65536, "lens_seed": 6},
        # A thousand long beams in a pool that fills the card.
        {"name": "fork_large", "kind": "fork", "requests": 128, "beams": 8, "shared": 16000,
         "own": 500, "pool": 524288, "lens_seed": 7},
        # A few blocks moved between steps, to keep a pool together.
        {"name": "compact_some", "kind": "compact", "seqs": 64, "length": 4000, "used": 0.3,
         "pool": 65536, "moves": 256, "lens_seed": 8},
        # A large pool brought together whole, before half of its memory is given back.
        {"name": "compact_all", "kind": "compact", "seqs": 512, "length": 16000, "used": 0.4,
         "pool": 524288, "moves": 524288, "lens_seed": 9},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    """An integer in [lo, hi], even over its logarithm; odd as often as even."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    """One more case of the same ranges, bounded by the largest listed ones."""
    kind = rng.choice(["shared", "shared", "shared", "select", "select", "fork", "compact"])
    seed = rng.randrange(1 << 20)
    if kind == "shared":
        h = rng.randrange(len(HEADS))
        H, Hkv, D = HEADS[h]
        shared = _log_int(rng, 1, 32768)
        own = _log_int(rng, 1, 2000)
        # sequences: at most 2^26 scores, and 4 GiB of 32-bit keys, in the plain form
        most = max(1, min((1 << 26) // (H * (shared + own)), (1 << 30) // (Hkv * D * (shared + own))))
        each = _log_int(rng, 1, max(1, min(192, most)))
        groups = _log_int(rng, 1, max(1, min(64, most // each)))
        return {"kind": kind, **_heads(h), "dtype": rng.choice(["f16", "bf16"]), "groups": groups,
                "each": each, "shared_lo": max(1, shared // rng.choice([1, 2, 8])),
                "shared_hi": shared, "own_lo": max(1, own // rng.choice([1, 4, 64])),
                "own_hi": own, "idle": rng.choice([0.0, 0.0, 0.2]), "lens_seed": seed,
                "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "alibi": rng.random() < 0.3,
                "layers": rng.choice([1, 2, 3])}
    if kind == "select":
        beams = _log_int(rng, 1, 32)
        vocab = _log_int(rng, 500, 200000)
        requests = _log_int(rng, 1, max(1, min(256, (1 << 25) // (beams * vocab))))
        return {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "requests": requests,
                "beams": beams, "candidates": min(64, beams * rng.choice([1, 2, 2])),
                "vocab": vocab, "pad": rng.choice([0, 0, 1, 64]), "first": rng.random() < 0.2,
                "banned": rng.choice([0.0, 0.0, 0.5, 0.9]), "eos": rng.random() < 0.7}
    pool = _log_int(rng, 1000, 400000)
    if kind == "fork":
        beams = _log_int(rng, 1, 32)
        length = _log_int(rng, 17, 16000)
        own = min(length, _log_int(rng, 1, 500))
        per = _blocks(length) + beams * (_blocks(own) + 4)
        requests = _log_int(rng, 1, max(1, min(256, pool * 2 // 3 // per)))
        return {"kind": kind, "requests": requests, "beams": beams, "shared": length, "own": own,
                "pool": max(pool, 2 * requests * per), "lens_seed": seed}
    return {"kind": kind, "seqs": _log_int(rng, 1, 1024), "length": _log_int(rng, 1, 16000),
            "used": rng.uniform(0.05, 0.95), "pool": pool, "moves": _log_int(rng, 1, pool),
            "lens_seed": seed}


def _blocks(n: int) -> int:
    return (n + BS - 1) // BS


def _group_lens(case: dict) -> tuple[list[int], list[list[int]]]:
    """(shared tokens of each group, own tokens of its sequences, -1 for an idle
    one) of a shared case; part of its size, not of its data."""
    r = random.Random(case["lens_seed"])
    shared = [r.randint(case["shared_lo"], case["shared_hi"]) for _ in range(case["groups"])]
    lens = [[-1 if r.random() < case["idle"] else r.randint(case["own_lo"], case["own_hi"])
             for _ in range(case["each"])] for _ in range(case["groups"])]
    return shared, lens


def _fork_lens(case: dict) -> tuple[list[int], list[int]]:
    """(prompt, context) of each request of a fork case; its beams are as long as each other."""
    r = random.Random(case["lens_seed"])
    prompt = [r.randint(max(1, case["shared"] // 4), case["shared"]) for _ in range(case["requests"])]
    return prompt, [p + r.randint(1, case["own"]) for p in prompt]


def _compact_lens(case: dict) -> list[int]:
    """Contexts of the sequences of a compact case, while the pool has the room."""
    r = random.Random(case["lens_seed"])
    room = int(case["pool"] * case["used"])
    lens = []
    for _ in range(case["seqs"]):
        n = r.randint(1, case["length"])
        n = n if _blocks(n) <= room else 0
        room -= _blocks(n)
        lens.append(n)
    return lens


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g: torch.Generator, dtype, *shape, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=I32, device=DEV)


def _tables(perm: torch.Tensor, common: list[int], need: list[list[int]]) -> torch.Tensor:
    """Tables int32 [rows, most blocks]: the rows of a group begin with the same
    `common` blocks and go on with their own, need[group][row] in all, taken from
    perm in order. Entries behind them name a block too."""
    rows = [n for g in need for n in g]
    group = [i for i, g in enumerate(need) for _ in g]
    owned = [max(n - common[i], 0) for n, i in zip(rows, group)]
    used = sum(common)
    start = []
    for n in owned:
        start.append(used)
        used += n
    lead = torch.tensor([sum(common[:i]) for i in group], dtype=I64, device=DEV)[:, None]
    start = torch.tensor(start, dtype=I64, device=DEV)[:, None]
    have = torch.tensor([common[i] for i in group], dtype=I64, device=DEV)[:, None]
    col = torch.arange(max(max(rows), 1), device=DEV)
    at = torch.where(col < have, lead + col, start + col - have)
    return perm[at.clamp_(max=perm.numel() - 1)].to(I32).contiguous()


def _shared_state(case: dict, seed: int) -> dict:
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    shared, lens = _group_lens(case)
    ctx = [[0 if n < 0 else p + n for n in row] for p, row in zip(shared, lens)]
    # a prompt's last, partly filled block is a sequence's own
    common = [p // BS for p in shared]
    need = [[_blocks(n) for n in row] for row in ctx]
    total = sum(common) + sum(max(n - c, 0) for c, row in zip(common, need) for n in row)
    NB = math.ceil(1.1 * total) + 1
    bt = _tables(torch.randperm(NB, generator=g, device=DEV), common, need)
    flat = [n for row in ctx for n in row]
    S = len(flat)
    s = dict(S=S, MB=bt.shape[1], NB=NB, N=case["groups"], bt=bt, ctx=_ints(flat), ctx_list=flat,
             goff=_ints([i * case["each"] for i in range(case["groups"] + 1)]),
             scale=1.0 / math.sqrt(D), slopes=None)
    if case["alibi"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=F32, device=DEV) / H)
    # scores of some size, as after training: sigma about 4 before a cap
    s["layers"] = [dict(q=_normal(g, dt, S, H, D, std=4.0), kc=_normal(g, dt, NB, Hkv, D, BS),
                        vc=_normal(g, dt, NB, Hkv, D, BS)) for _ in range(case["layers"])]
    return s


def _select_state(case: dict, seed: int) -> dict:
    """Logits of a sharp head over a long tail, in rows of vocab + pad values;
    beams some nats apart, at a request's first step only one of them."""
    g = _gen(seed)
    R, W, V = case["requests"], case["beams"], case["vocab"]
    x = _normal(g, F32, R * W, V + case["pad"], std=2.5)
    top = torch.randint(0, V, (R * W, 24), generator=g, device=DEV)
    x.scatter_add_(1, top, 8.0 * torch.rand(R * W, 24, generator=g, device=DEV))
    if case["banned"]:
        x.masked_fill_(torch.rand(x.shape, generator=g, device=DEV) < case["banned"], -math.inf)
    eos = int(torch.randint(0, V, (1,), generator=g, device=DEV)) if case["eos"] else -1
    if eos >= 0:
        x[::3, eos] = 9.0
    scores = -20.0 * torch.rand(R, W, generator=g, device=DEV)
    if case["first"]:
        scores[:, 1:] = -math.inf
    return dict(x=x.to(DTYPES[case["dtype"]]), scores=scores, eos=eos)


def _fork_state(case: dict, seed: int) -> dict:
    """Beams that share their prompt's whole blocks, and a block that is partly
    filled with nobody. Parents as a search picks them: the better beams more often."""
    g = _gen(seed)
    R, W, NB = case["requests"], case["beams"], case["pool"]
    prompt, ctx = _fork_lens(case)
    bt = _tables(torch.randperm(NB, generator=g, device=DEV), [p // BS for p in prompt],
                 [[_blocks(n)] * W for n in ctx])
    S, MB = bt.shape
    lens = torch.tensor(ctx, dtype=I32, device=DEV).repeat_interleave(W).contiguous()
    nb = (lens.to(I64) + BS - 1) // BS
    used = torch.arange(MB, device=DEV) < nb[:, None]
    refs = torch.zeros(NB, dtype=I64, device=DEV).index_add_(0, bt[used].to(I64),
                                                             torch.ones_like(bt[used], dtype=I64))
    beam = (W * torch.rand(S, generator=g, device=DEV) ** 2).to(I64).clamp_(max=W - 1)
    parents = torch.arange(S, device=DEV) // W * W + beam
    free = torch.nonzero(refs == 0).flatten()
    listing = torch.full((NB,), -1, dtype=I32, device=DEV)
    listing[:free.numel()] = free.to(I32)
    return dict(S=S, MB=MB, NB=NB, parents=parents.to(I32), refs=refs.to(I32), free=listing,
                num_free=_ints([free.numel()]), now=0, tables=[bt, torch.zeros_like(bt)],
                ctx=[lens, torch.zeros_like(lens)],
                pairs=torch.zeros(S, 2, dtype=I64, device=DEV), counts=_ints([0, 0]))


def _compact_state(case: dict, seed: int) -> dict:
    """Sequences of their own blocks, all over the pool."""
    g = _gen(seed)
    NB, lens = case["pool"], _compact_lens(case)
    bt = _tables(torch.randperm(NB, generator=g, device=DEV), [0] * len(lens),
                 [[_blocks(n)] for n in lens])
    ctx = _ints(lens)
    used = torch.arange(bt.shape[1], device=DEV) < ((ctx.to(I64) + BS - 1) // BS)[:, None]
    refs = torch.zeros(NB, dtype=I32, device=DEV)
    refs[bt[used].to(I64)] = 1
    return dict(S=len(lens), MB=bt.shape[1], NB=NB, bt=bt, ctx=ctx, refs=refs,
                moves=min(case["moves"], NB),
                out={"tables": torch.zeros_like(bt), "refs": torch.zeros_like(refs),
                     "free": torch.full((NB,), -1, dtype=I32, device=DEV), "num_free": _ints([0]),
                     "pairs": torch.zeros(min(case["moves"], NB), 2, dtype=I64, device=DEV),
                     "new_ids": torch.zeros_like(refs), "counts": _ints([0, 0])})


def prepare(case: dict, seed: int) -> dict:
    if case["kind"] == "shared":
        s = _shared_state(case, seed)
        s["out"] = [torch.zeros_like(x["q"]) for x in s["layers"]]
        s["shared"] = torch.zeros(s["N"], dtype=I32, device=DEV)
    elif case["kind"] == "select":
        s = _select_state(case, seed)
        R, W, C = case["requests"], case["beams"], case["candidates"]
        s["out"] = {f"{who}_{what}": torch.zeros(R, n, dtype=t, device=DEV)
                    for who, n in (("cand", C), ("next", W))
                    for what, t in (("scores", F32), ("rows", I32), ("tokens", I32))}
    elif case["kind"] == "fork":
        s = _fork_state(case, seed)
    else:
        s = _compact_state(case, seed)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_shared_blocks(s: dict, case: dict):
    """Leading blocks that the sequences of a group with a context all use, and alike."""
    N, each = s["N"], case["each"]
    bt = s["bt"].view(N, each, -1)
    ctx = s["ctx"].to(I64).view(N, each)
    live = ctx > 0
    lead = torch.arange(N, device=DEV), torch.argmax(live.to(I32), 1)
    inside = torch.arange(s["MB"], device=DEV) < ((ctx + BS - 1) // BS)[..., None]
    alike = ((bt == bt[lead][:, None]) & inside) | ~live[..., None]
    n = torch.cumprod(alike.all(1).to(I32), 1).sum(1)
    s["shared"].copy_(torch.where(live.any(1), n, 0))


def _plain_attention(s: dict, x: dict, out: torch.Tensor, case: dict):
    """The padded batch at once, each sequence with all of its own keys."""
    S, MB, H, Hkv, D = s["S"], s["MB"], case["heads"], case["kv_heads"], case["head_dim"]
    G, L = H // Hkv, s["MB"] * BS
    ids = s["bt"].to(I64)
    ctx = s["ctx"].to(I64).view(S, 1, 1, 1)
    k = x["kc"][ids].permute(0, 2, 3, 1, 4).reshape(S, Hkv, D, L).to(F32)
    y = torch.matmul(x["q"].to(F32).view(S, Hkv, G, D), k) * s["scale"]
    del k
    if case["cap"] > 0:
        y = case["cap"] * torch.tanh(y / case["cap"])
    key = torch.arange(L, device=DEV)
    if s["slopes"] is not None:
        y = y - s["slopes"].view(1, Hkv, G, 1) * (ctx - 1 - key)
    y = y.masked_fill(key >= ctx, -math.inf)
    y = torch.exp(y - y.amax(-1, keepdim=True).clamp(min=-3e38))
    total = y.sum(-1, keepdim=True)
    v = x["vc"][ids].permute(0, 2, 1, 4, 3).reshape(S, Hkv, L, D).to(F32)
    y = torch.matmul(y, v)
    out.copy_(torch.where(total > 0, y / total, 0.0).reshape(S, H, D))


def _plain_shared(s: dict) -> dict:
    _plain_shared_blocks(s, s["case"])
    for x, out in zip(s["layers"], s["out"]):
        _plain_attention(s, x, out, s["case"])
    return {"out": s["out"], "shared_blocks": s["shared"]}


def _plain_select(s: dict) -> dict:
    """Every continuation's score in 64 bits, sorted."""
    case = s["case"]
    R, W, V, C = (case[k] for k in ("requests", "beams", "vocab", "candidates"))
    x = s["x"][:, :V].to(F64)
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = (x - lse).view(R, W, V).add_(s["scores"].to(F64)[..., None]).view(R, W * V)
    del x
    score, at = torch.sort(score, dim=1, descending=True, stable=True)
    score, at = score[:, :C], at[:, :C]
    real = score > -math.inf
    rows = torch.where(real, torch.arange(R, device=DEV)[:, None] * W + at // V, -1)
    tokens = torch.where(real, at % V, -1)
    o = s["out"]
    o["cand_scores"].copy_(score)
    o["cand_rows"].copy_(rows)
    o["cand_tokens"].copy_(tokens)
    # the first W that go on keep their order
    on = real & (tokens != s["eos"]) if s["eos"] >= 0 else real
    order = torch.sort((~on).to(I32), dim=1, stable=True).indices
    if C < W:
        raise ValueError("fewer candidates than beams")
    order = order[:, :W]
    on = torch.gather(on, 1, order)
    o["next_scores"].copy_(torch.where(on, torch.gather(score, 1, order), -math.inf))
    o["next_rows"].copy_(torch.where(on, torch.gather(rows, 1, order), -1))
    o["next_tokens"].copy_(torch.where(on, torch.gather(tokens, 1, order), -1))
    return o


def _counted(values: torch.Tensor, used: torch.Tensor, n: int) -> torch.Tensor:
    """How often each id below n stands in the used places."""
    at = torch.where(used, values.to(I64), n).flatten()
    return torch.zeros(n + 1, dtype=I64, device=DEV).index_add_(0, at, torch.ones_like(at))[:n]


def _listed_ids(mask: torch.Tensor, into: torch.Tensor) -> torch.Tensor:
    """The ids where mask holds, ascending, at the front of `into`; how many."""
    n = mask.numel()
    rank = torch.cumsum(mask, 0)
    spill = torch.cat([into, into[:1]])
    spill[torch.where(mask, rank - 1, n)] = torch.arange(n, dtype=into.dtype, device=DEV)
    into.copy_(spill[:n])
    return rank[-1]


def _plain_fork(s: dict) -> dict:
    S, MB, NB = s["S"], s["MB"], s["NB"]
    bt, ctx = s["tables"][s["now"]], s["ctx"][s["now"]].to(I64)
    to, to_ctx = s["tables"][1 - s["now"]], s["ctx"][1 - s["now"]]
    p = s["parents"].to(I64)
    col = torch.arange(MB, device=DEV)
    on = p >= 0
    new = torch.where(on, ctx[p.clamp(min=0)], 0)
    used = col < ((new + BS - 1) // BS)[:, None]
    to.copy_(torch.where(used, bt[p.clamp(min=0)], to))
    refs = (s["refs"].to(I64) + _counted(to, used, NB)
            - _counted(bt, col < ((ctx + BS - 1) // BS)[:, None], NB))
    # who takes a copy of a block that is partly filled
    last = ((new + BS - 1) // BS - 1).clamp(min=0)
    row = torch.arange(S, device=DEV)
    src = to[row, last].to(I64)
    older = ((p[:, None] == p) & (row[:, None] > row)).sum(1)   # children of the same parent before
    copy = (new % BS != 0) & (older < refs[src] - 1)
    k = torch.cumsum(copy, 0) - 1
    spare = torch.full((NB,), -1, dtype=I64, device=DEV)
    F = _listed_ids(refs == 0, spare)
    got = copy & (k < F)
    cut = copy & ~got
    dst = spare[k.clamp(0, NB - 1)]
    to[row, last] = torch.where(got, dst, src).to(I32)
    to_ctx.copy_(torch.where(cut, new // BS * BS, new))
    one = torch.ones_like(src)
    refs.index_add_(0, torch.where(copy, src, 0), torch.where(copy, -one, 0))
    refs.index_add_(0, torch.where(got, dst, 0), torch.where(got, one, 0))
    s["refs"].copy_(refs)
    s["pairs"].fill_(-1)
    at = torch.where(got, k, S)
    pairs = torch.cat([s["pairs"], s["pairs"][:1]])
    pairs[at] = torch.stack([src, dst], 1)
    s["pairs"].copy_(pairs[:S])
    taken = got.sum()
    rest = torch.arange(NB, device=DEV)
    s["free"].copy_(torch.where(rest < F - taken, spare[(rest + taken).clamp(max=NB - 1)], s["free"]))
    s["num_free"].copy_((F - taken).view(1))
    s["counts"].copy_(torch.stack([taken, cut.sum()]))
    return _fork_out(s)


def _fork_out(s: dict) -> dict:
    """The step's state after a pass; the next one goes on from it."""
    s["now"] = 1 - s["now"]
    return {"tables": s["tables"][s["now"]], "ctx": s["ctx"][s["now"]], "refs": s["refs"],
            "free": s["free"], "num_free": s["num_free"], "pairs": s["pairs"], "counts": s["counts"]}


def _plain_compact(s: dict) -> dict:
    NB, M, o = s["NB"], s["moves"], s["out"]
    refs = s["refs"].to(I64)
    live = refs > 0
    up = torch.full((NB,), -1, dtype=I64, device=DEV)
    down = torch.full((NB,), -1, dtype=I64, device=DEV)
    n_free = _listed_ids(~live, up)                       # the lowest free ones first
    n_live = _listed_ids(torch.flip(live, (0,)), down)    # the highest in use first
    k = torch.arange(NB, device=DEV)
    src = NB - 1 - down
    move = (k < n_live) & (k < n_free) & (k < M) & (src > up)
    ids = torch.cat([k, k[:1]])
    ids[torch.where(move, src, NB)] = up
    ids = ids[:NB]
    o["new_ids"].copy_(ids)
    o["pairs"].copy_(torch.where(move[:M, None], torch.stack([src, up], 1)[:M], -1))
    moved = torch.zeros(NB, dtype=I64, device=DEV).index_add_(0, ids, refs)
    o["refs"].copy_(moved)
    used = torch.arange(s["MB"], device=DEV) < ((s["ctx"].to(I64) + BS - 1) // BS)[:, None]
    o["tables"].copy_(torch.where(used, ids[s["bt"].to(I64)], o["tables"]))
    F = _listed_ids(moved == 0, o["free"])
    o["num_free"].copy_(F.view(1))
    o["counts"].copy_(torch.stack([move.sum(), n_live]))
    return o


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _kept(s: dict, name: str, size) -> torch.Tensor:
    """Scratch kept for the sizes, as a server does."""
    if name not in s:
        s[name] = torch.empty(max(size(), 256), dtype=torch.uint8, device=DEV)
    return s[name]


def _own_shared(s: dict) -> dict:
    from swiftllm_amd import attention_step as step
    case = s["case"]
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    sizes = (s["S"], H, Hkv, D, BS, s["MB"])
    plan = _kept(s, "plan", lambda: step.plan_shared_size(*sizes))
    ws = _kept(s, "ws", lambda: step.shared_decode_workspace_size(*sizes))
    step.plan_shared(_ptr(plan), plan.numel(), _ptr(s["shared"]), _ptr(s["bt"]), _ptr(s["ctx"]),
                     _ptr(s["goff"]), s["N"], *sizes)
    score = step.ScoreParams(scale=s["scale"], softcap=case["cap"], alibi_slopes=_ptr(s["slopes"]))
    for x, out in zip(s["layers"], s["out"]):
        step.shared_decode(_ptr(out), _ptr(ws), ws.numel(), _ptr(plan), plan.numel(), _ptr(x["q"]),
                           _ptr(x["kc"]), _ptr(x["vc"]), _ptr(s["bt"]), score, *sizes,
                           dtype=case["dtype"], num_blocks=s["NB"])
    return {"out": s["out"], "shared_blocks": s["shared"]}


def _own_select(s: dict) -> dict:
    from swiftllm_amd import beam_search as bs
    case, o = s["case"], s["out"]
    R, W, V, C = (case[k] for k in ("requests", "beams", "vocab", "candidates"))
    ws = _kept(s, "ws", lambda: bs.beam_select_workspace_size(R, W, V, C))
    bs.beam_select(_ptr(s["x"]), _ptr(s["scores"]), _ptr(o["cand_scores"]), _ptr(o["cand_rows"]),
                   _ptr(o["cand_tokens"]), _ptr(o["next_scores"]), _ptr(o["next_rows"]),
                   _ptr(o["next_tokens"]), _ptr(ws), ws.numel(), R, W, V, C, dtype=case["dtype"],
                   logits_stride=s["x"].stride(0), eos_id=s["eos"])
    return o


def _own_fork(s: dict) -> dict:
    from swiftllm_amd import pages
    now = s["now"]
    ws = _kept(s, "ws", lambda: pages.pages_workspace_size(s["S"], s["NB"]))
    pages.fork_pages(_ptr(s["tables"][1 - now]), _ptr(s["ctx"][1 - now]), _ptr(s["tables"][now]),
                     _ptr(s["ctx"][now]), _ptr(s["parents"]), _ptr(s["refs"]), _ptr(s["free"]),
                     _ptr(s["num_free"]), _ptr(s["pairs"]), _ptr(s["counts"]), _ptr(ws), ws.numel(),
                     s["S"], s["MB"], BS, s["NB"])
    return _fork_out(s)


def _own_compact(s: dict) -> dict:
    from swiftllm_amd import pages
    o = s["out"]
    ws = _kept(s, "ws", lambda: pages.pages_workspace_size(s["S"], s["NB"]))
    pages.compact_pages(_ptr(o["tables"]), _ptr(o["refs"]), _ptr(s["bt"]), _ptr(s["ctx"]),
                        _ptr(s["refs"]), _ptr(o["free"]), _ptr(o["num_free"]), _ptr(o["pairs"]),
                        _ptr(o["new_ids"]), _ptr(o["counts"]), _ptr(ws), ws.numel(), s["S"],
                        s["MB"], BS, s["NB"], s["moves"])
    return o


def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        return {"shared": _own_shared, "select": _own_select, "fork": _own_fork,
                "compact": _own_compact}[kind](s)
    return {"shared": _plain_shared, "select": _plain_select, "fork": _plain_fork,
            "compact": _plain_compact}[kind](s)


# ---------------------------------------------------------------------------
# What one pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    if case["kind"] == "shared":
        H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
        shared, lens = _group_lens(case)
        keys = pairs = entries = rows = 0
        for p, row in zip(shared, lens):
            live = [n for n in row if n >= 0]
            common = p // BS * BS if live else 0
            keys += common + sum(p + n - common for n in live)
            pairs += sum(p + n for n in live)
            entries += sum(_blocks(p + n) for n in live)
            rows += len(row)
        return {"bytes": case["layers"] * (4 * rows * H * D + 4 * keys * Hkv * D) + 4 * entries
                         + 4 * rows, "flops": case["layers"] * 4 * pairs * H * D}
    if case["kind"] == "select":
        R, W, V, C = (case[k] for k in ("requests", "beams", "vocab", "candidates"))
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": R * W * V * size + 4 * R * W + 12 * R * (C + W), "flops": 3 * R * W * V}
    if case["kind"] == "fork":
        _, ctx = _fork_lens(case)
        S, NB = case["requests"] * case["beams"], case["pool"]
        entries = case["beams"] * sum(_blocks(n) for n in ctx)
        return {"bytes": 8 * entries + 8 * NB + 4 * NB + 28 * S, "flops": 0}
    entries = sum(_blocks(n) for n in _compact_lens(case))
    NB = case["pool"]
    moves = min(case["moves"], NB)
    return {"bytes": 8 * entries + 8 * NB + 4 * NB + 4 * (NB - entries) + 16 * moves
                     + 4 * case["seqs"], "flops": 0}


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def _exact_shared(case: dict, seed: int) -> dict:
    s = _shared_state(case, seed)
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    outs = []
    for x in s["layers"]:
        out = torch.zeros(s["S"], H, D, dtype=F64, device=DEV)
        for i, n in enumerate(s["ctx_list"]):
            if n == 0:
                continue
            ids = s["bt"][i, :_blocks(n)].to(I64)
            k = x["kc"][ids].permute(1, 2, 0, 3).reshape(Hkv, D, -1)[:, :, :n].to(F64)
            v = x["vc"][ids].permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :n].to(F64)
            z = torch.bmm(x["q"][i].to(F64).view(Hkv, H // Hkv, D), k.contiguous()).mul_(s["scale"])
            if case["cap"] > 0:
                e = torch.expm1(z * (2.0 / case["cap"]))     # tanh(y) = (e^2y - 1) / (e^2y + 1)
                z = case["cap"] * e / (e + 2.0)
            if case["alibi"]:
                back = torch.arange(n - 1, -1, -1, dtype=F64, device=DEV)
                z = z - s["slopes"].to(F64).view(Hkv, -1, 1) * back
            out[i] = torch.bmm(torch.softmax(z, -1), v.contiguous()).view(H, D)
        outs.append(out)
    return {"out": outs, "shared_blocks": None}


def _exact_select(case: dict, seed: int) -> dict:
    s = _select_state(case, seed)
    R, W, V, C = (case[k] for k in ("requests", "beams", "vocab", "candidates"))
    best, on = [], []
    for r in range(R):
        x = torch.log_softmax(s["x"][r * W:(r + 1) * W, :V].to(F64), 1)
        if s["eos"] >= 0:
            go = x.clone()
            go[:, s["eos"]] = -math.inf
        else:
            go = x
        c = s["scores"][r].to(F64)[:, None]
        best.append(torch.topk((x + c).flatten(), C).values)
        # of those that go on, the ones among the candidates
        on.append(torch.topk((go + c).flatten(), W).values)
    best, on = torch.stack(best), torch.stack(on)
    on = torch.where(on >= best[:, -1:], on, -math.inf)
    return {"cand_scores": best, "cand_rows": None, "cand_tokens": None, "next_scores": on,
            "next_rows": None, "next_tokens": None}


def exact(case: dict, seed: int):
    if case["kind"] == "shared":
        return _exact_shared(case, seed)
    if case["kind"] == "select":
        return _exact_select(case, seed)
    return None
