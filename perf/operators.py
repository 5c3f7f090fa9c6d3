"""The 8-bit paged cache and the attention that reads it, as a serving program calls them once a layer.

Two kinds of case:

  store    the step's keys are rotated and stored with the values, each (token, head) row as 128 e4m3 numbers and one fp32 scale;
           the queries are rotated; the rows are then read back as they are when a request's pages move.  Out: queries, keys, values.
  attend   the step's queries attend to their sequence's stored rows: one token a sequence, a prompt's portion (a query sees
           what is at or before its place), or a tree of drafted tokens at the end of the sequence (a node sees all that was there
           before the draft and the nodes of a 64-bit word).  Out: one row a query.

A stored row of x is s = max(max |x| / 448, 2^-126), c = e4m3(x / s), and stands for c * s.  Heads and lengths are those of the
repository's Llama presets and of its benchmark; the cache's pages have 32 tokens and lie in any order.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE, DIM, TOP = 32, 128, 448.0
TINY = 2.0 ** -126
PLACES = 8192                       # rows of the rotation table
HEADS = [(32, 8), (64, 8), (6, 2), (4, 2), (4, 1), (12, 12), (16, 4)]


# ------------------------------------------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # the next token of one request: nothing but latency
        dict(name="store-one", kind="store", n_q=32, n_kv=8, seqs=1, new_lo=1, new_hi=1, kv_lo=200, kv_hi=200),
        # a busy server's decode step: one row a request, each on a page of its own
        dict(name="store-batch", kind="store", n_q=32, n_kv=8, seqs=96, new_lo=1, new_hi=1, kv_lo=20, kv_hi=2000),
        # a full prefill step of mixed prompts
        dict(name="store-prompts", kind="store", n_q=32, n_kv=8, seqs=6, new_lo=90, new_hi=593, kv_lo=0, kv_hi=0),
        # one short chat with the small model
        dict(name="token-one", kind="attend", n_q=6, n_kv=2, seqs=1, new_lo=1, new_hi=1, kv_lo=17, kv_hi=17, tree=False),
        # the headline batch of 32 decoding requests
        dict(name="tokens-batch", kind="attend", n_q=32, n_kv=8, seqs=32, new_lo=1, new_hi=1, kv_lo=512, kv_hi=640, tree=False),
        # few requests with long contexts, eight query heads a key head
        dict(name="tokens-long", kind="attend", n_q=64, n_kv=8, seqs=7, new_lo=1, new_hi=1, kv_lo=5000, kv_hi=8192, tree=False),
        # eight drafted tokens of one request
        dict(name="tree-one", kind="attend", n_q=32, n_kv=8, seqs=1, new_lo=8, new_hi=8, kv_lo=500, kv_hi=500, tree=True),
        # drafts of a batch, each of its own size
        dict(name="tree-batch", kind="attend", n_q=32, n_kv=8, seqs=16, new_lo=5, new_hi=24, kv_lo=200, kv_hi=1500, tree=True),
        # wide drafts over long contexts
        dict(name="tree-wide", kind="attend", n_q=64, n_kv=8, seqs=4, new_lo=61, new_hi=64, kv_lo=4000, kv_hi=8000, tree=True),
        # many short prompts in one step
        dict(name="prompts-short", kind="attend", n_q=32, n_kv=8, seqs=24, new_lo=9, new_hi=57, kv_lo=0, kv_hi=0, tree=False),
        # a full step of mixed prompts
        dict(name="prompts-mixed", kind="attend", n_q=32, n_kv=8, seqs=6, new_lo=90, new_hi=593, kv_lo=0, kv_hi=0, tree=False),
        # the last portion of a long document
        dict(name="document", kind="attend", n_q=32, n_kv=8, seqs=1, new_lo=1859, new_hi=1859, kv_lo=6144, kv_hi=6144, tree=False),
    ]


def _between(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number, spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    n_q, n_kv = rng.choice(HEADS)
    kind = rng.choice(["store", "store", "token", "token", "tree", "tree", "prompt", "prompt"])
    case = dict(kind="store" if kind == "store" else "attend", n_q=n_q, n_kv=n_kv)
    if kind == "store":
        case["seqs"] = _between(rng, 1, 96)
        case["new_hi"] = 1 if rng.random() < 0.4 else _between(rng, 2, max(2, 2048 // case["seqs"]))
        case["kv_hi"] = _between(rng, 1, 4000)
    elif kind == "token":
        case["seqs"] = _between(rng, 1, 96)
        case["new_hi"] = 1
        case["kv_hi"] = _between(rng, 1, min(8192, 60000 // case["seqs"]))
    elif kind == "tree":
        case["seqs"] = _between(rng, 1, 24)
        case["new_hi"] = _between(rng, 2, min(64, max(2, 320 // case["seqs"])))
        case["kv_hi"] = _between(rng, 1, min(8000, 24000 // case["seqs"]))
    else:
        case["seqs"] = _between(rng, 1, 24)
        case["new_hi"] = _between(rng, 2, max(2, 1800 // case["seqs"]))
        case["kv_hi"] = 0 if rng.random() < 0.5 else _between(rng, 1, 6000 // case["seqs"])
    case["new_lo"] = rng.randint(max(1, case["new_hi"] // 3), case["new_hi"])
    case["kv_lo"] = rng.randint(case["kv_hi"] // 3, case["kv_hi"])
    if case["kind"] == "attend":
        case["tree"] = kind == "tree"
    return case


def _lengths(case: dict, seed: int) -> list[tuple[int, int]]:
    """(new tokens, tokens that were there before them) of every sequence: the former belong to the case, the latter to the seed."""
    sizes, rng = random.Random(" ".join(f"{k}={v}" for k, v in sorted(case.items()) if k != "name")), random.Random(seed * 7919 + 13)
    got = []
    for _ in range(case["seqs"]):
        new, all_ = sizes.randint(case["new_lo"], case["new_hi"]), rng.randint(case["kv_lo"], case["kv_hi"])
        got.append((new, max(0, all_ - 1) if case["new_hi"] == 1 else all_))
    return got


def _mean_lengths(case: dict) -> list[tuple[int, float]]:
    old = (case["kv_lo"] + case["kv_hi"]) / 2
    return [(new, max(0.0, old - 1) if case["new_hi"] == 1 else old) for new, _ in _lengths(case, 0)]


# ------------------------------------------------------------------------------------------------------------ inputs
def _rows(gen, n: int, heads: int) -> torch.Tensor:
    """Projected rows in bf16: a few channels carry large numbers, and tokens differ in size."""
    channel = torch.ones(heads, DIM, device="cuda")
    channel[:, ::37] = 5.0
    token = torch.exp(0.4 * torch.randn(n, 1, 1, device="cuda", generator=gen))
    return (torch.randn(n, heads, DIM, device="cuda", generator=gen) * channel * token).to(torch.bfloat16)


def _table() -> torch.Tensor:
    """cos | sin of every position, rounded as the checkpoint's users do."""
    inv = 1.0 / (500000.0 ** (torch.arange(0, DIM, 2, dtype=torch.float64) / DIM))
    angle = torch.outer(torch.arange(PLACES, dtype=torch.float64), inv)
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(torch.bfloat16).cuda()


def _tree_words(lengths, seed: int) -> list[int]:
    """One word a node: itself and its ancestors among the draft's nodes."""
    rng = random.Random(seed * 31 + 7)
    words = []
    for new, _ in lengths:
        seen: list[int] = []
        for i in range(new):
            parent = max(rng.randint(-1, i - 1), rng.randint(-1, i - 1)) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        words += seen
    return [w - (1 << 64) if w >> 63 else w for w in words]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n_q, n_kv, lengths = case["n_q"], case["n_kv"], _lengths(case, seed)
    rng = random.Random(seed)
    pages = [(new + old + PAGE - 1) // PAGE for new, old in lengths]
    n_pages = sum(pages) + 3
    order = rng.sample(range(n_pages), n_pages)
    table, seqs, slots, places, at, row = [], [], [], [], 0, 0
    for i, (new, old) in enumerate(lengths):
        mine = order[at:at + pages[i]]
        at += pages[i]
        table.append(mine + [0] * (max(pages) - len(mine)))
        seqs.append([row, new, old + new, i])
        slots += [mine[p // PAGE] * PAGE + p % PAGE for p in range(old, old + new)]
        places += range(old, old + new)
        row += new
    dev = dict(device="cuda", dtype=torch.int32)
    st = dict(kind=case["kind"], n_q=n_q, n_kv=n_kv, slots=torch.tensor(slots, **dev), n_pages=n_pages)
    if case["kind"] == "store":
        qkv = torch.cat([_rows(gen, row, n_q), _rows(gen, row, n_kv), _rows(gen, row, n_kv)], dim=1).reshape(row, -1)
        st.update(qkv=qkv, places=torch.tensor(places, **dev), cos_sin=_table())
        # the cache that the rows go to
        codes = torch.zeros(2, n_pages, PAGE, n_kv, DIM, device="cuda").to(torch.float8_e4m3fn)
        st.update(codes=codes, scales=torch.zeros(2, n_pages, PAGE, n_kv, device="cuda"))
        if own:
            from vllm_tgis_adapter_b200.engine.cache8 import Cache8

            st["cache"] = Cache8.empty(n_pages, n_kv)
        return st
    st.update(q=(1.5 * torch.randn(row, n_q * DIM, device="cuda", generator=gen)).to(torch.bfloat16), scale=DIM ** -0.5,
              seqs=torch.tensor(seqs, **dev), table=torch.tensor(table, **dev), max_q=max(new for new, _ in lengths),
              max_kv=max(new + old for new, old in lengths), tree=None)
    if case["tree"]:
        st["tree"] = torch.tensor(_tree_words(lengths, seed), device="cuda", dtype=torch.int64)
    rows = torch.stack([_rows(gen, n_pages * PAGE, n_kv), _rows(gen, n_pages * PAGE, n_kv)])
    codes, scales = _quantise(rows)
    st.update(codes=codes.view(2, n_pages, PAGE, n_kv, DIM), scales=scales.view(2, n_pages, PAGE, n_kv))
    if own:
        # the program has stored these rows step by step
        from vllm_tgis_adapter_b200.engine.cache8 import Cache8

        st["cache"] = Cache8.empty(n_pages, n_kv)
        still = torch.tensor([1.0] * (DIM // 2) + [0.0] * (DIM // 2), device="cuda", dtype=torch.bfloat16).view(1, DIM)
        every = torch.arange(n_pages * PAGE, **dev)
        st["cache"].write(torch.cat([rows[0], rows[1]], dim=1).reshape(n_pages * PAGE, -1), torch.zeros_like(every), every, still)
        st["out"] = torch.empty_like(st["q"])
    return st


# --------------------------------------------------------------------------------------------------------- plain form
def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    x = x.float()
    s = (x.abs().amax(dim=-1) / TOP).clamp(min=TINY)
    return (x / s[..., None]).to(torch.float8_e4m3fn), s


def _turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    a, b = x[..., : DIM // 2], x[..., DIM // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_store(st: dict):
    n_q, n_kv, slots = st["n_q"], st["n_kv"], st["slots"].long()
    x = st["qkv"].view(len(slots), n_q + 2 * n_kv, DIM).float()
    turn = st["cos_sin"][st["places"].long()].float()[:, None]
    x[:, : n_q + n_kv] = _turn(x[:, : n_q + n_kv], turn[..., : DIM // 2], turn[..., DIM // 2:])
    codes, scales = _quantise(x[:, n_q:].reshape(len(slots), 2, n_kv, DIM).transpose(0, 1))
    st["codes"].view(2, -1, n_kv, DIM)[:, slots] = codes
    st["scales"].view(2, -1, n_kv)[:, slots] = scales
    back = st["codes"].view(2, -1, n_kv, DIM)[:, slots].float() * st["scales"].view(2, -1, n_kv)[:, slots][..., None]
    back = back.to(torch.bfloat16).reshape(2, len(slots), n_kv * DIM)
    return dict(q=x[:, :n_q].reshape(len(slots), n_q * DIM).to(torch.bfloat16), k=back[0], v=back[1])


def _plain_attend(st: dict):
    n_q, n_kv, (start, new, all_, row) = st["n_q"], st["n_kv"], st["seqs"].long().unbind(dim=1)
    group, most_q, table = n_q // n_kv, st["max_q"], st["table"].long()[row]
    k, v = (st["codes"][i][table].float() * st["scales"][i][table][..., None] for i in range(2))
    k, v = k.flatten(1, 2).permute(0, 2, 3, 1), v.flatten(1, 2).permute(0, 2, 1, 3)        # [seq, head, dim, key], [seq, head, key, dim]
    i, j = torch.arange(most_q, device="cuda"), torch.arange(k.shape[-1], device="cuda")
    is_row = i < new[:, None]
    rows = (start[:, None] + i).clamp(max=len(st["q"]) - 1)
    q = st["q"][rows].float().view(len(start), most_q, n_kv, group, DIM).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s = (q * st["scale"]) @ k                                                               # [seq, head, query x group, key]
    old = (all_ - new)[:, None, None]
    sees = j <= old + i[:, None]
    if st["tree"] is not None:
        bit = (j - old).clamp(0, 63)
        sees = (j < old) | (st["tree"][rows][..., None] >> bit & 1).bool()
    sees = sees & (j < all_[:, None, None])
    s.view(len(start), n_kv, most_q, group, -1).masked_fill_(~sees[:, None, :, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(top).exp_()
    o = (p @ v) / p.sum(dim=-1, keepdim=True)
    o = o.view(len(start), n_kv, most_q, group, DIM).permute(0, 2, 1, 3, 4).reshape(len(start), most_q, n_q * DIM)
    return o[is_row].to(torch.bfloat16)


def run(st: dict):
    if not own:
        return _plain_store(st) if st["kind"] == "store" else _plain_attend(st)
    cache = st["cache"]
    if st["kind"] == "store":
        q = cache.write(st["qkv"], st["places"], st["slots"], st["cos_sin"])
        k, v = cache.read(st["slots"])
        return dict(q=q, k=k, v=v)
    return cache.attend(st["q"], st["seqs"], st["table"], st["scale"], st["max_q"], st["max_kv"], out=st["out"], tree=st["tree"])


# --------------------------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    n_q, n_kv, lengths = case["n_q"], case["n_kv"], _mean_lengths(case)
    tokens, stored = sum(new for new, _ in lengths), 2 * n_kv * (DIM + 4)
    if case["kind"] == "store":
        bytes_ = tokens * (2 * DIM * (n_q + 2 * n_kv) + 2 * DIM + 8) + tokens * (2 * DIM * n_q + 2 * stored + 2 * DIM * 2 * n_kv)
        return dict(bytes=bytes_, flops=tokens * DIM * (3 * (n_q + n_kv) + 6 * n_kv))
    keys = sum(new + old for new, old in lengths)
    # a tree's node sees about as many nodes as the draft is deep: counted as the logarithm of its size
    pairs = sum(new * old + (new * (1 + math.log2(max(new, 1))) if case["tree"] else new * (new + 1) / 2) for new, old in lengths)
    return dict(bytes=keys * stored + 2 * tokens * n_q * DIM * 2, flops=4 * pairs * n_q * DIM)


# ------------------------------------------------------------------------------------------------------ in 64 bits
def _to_e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest number with three bits behind the first, none below 2^-6 with steps smaller than 2^-9; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def exact(case: dict, seed: int):
    global own
    keep, own = own, False
    st = prepare(case, seed)
    own = keep
    n_q, n_kv = case["n_q"], case["n_kv"]
    if case["kind"] == "store":
        t = len(st["slots"])
        heads = st["qkv"].double().view(t, n_q + 2 * n_kv, 2, DIM // 2)
        cs = st["cos_sin"].double()[st["places"].long()].view(t, 1, 2, DIM // 2)
        turned = torch.stack([heads[:, :, 0] * cs[:, :, 0] - heads[:, :, 1] * cs[:, :, 1],
                              heads[:, :, 0] * cs[:, :, 1] + heads[:, :, 1] * cs[:, :, 0]], dim=2)
        q = turned[:, :n_q].reshape(t, -1)
        out = []
        for x in (turned[:, n_q:n_q + n_kv], heads[:, n_q + n_kv:]):
            x = x.reshape(t, n_kv, DIM)
            # the scale is a stored number of 32 bits
            s = (x.abs().amax(-1).float() / TOP).clamp(min=TINY).double()[..., None]
            out.append((_to_e4m3(x / s) * s).reshape(t, -1))
        return dict(q=q, k=out[0], v=out[1])
    group, out = n_q // n_kv, torch.empty(len(st["q"]), n_kv, n_q // n_kv, DIM, device="cuda", dtype=torch.float64)
    for n, (start, new, all_, row) in enumerate(st["seqs"].tolist()):
        mine = st["table"][row, : (all_ + PAGE - 1) // PAGE].long()
        k, v = (st["codes"][i][mine].double().mul_(st["scales"][i][mine].double()[..., None]).reshape(-1, n_kv, DIM)[:all_] for i in range(2))
        hidden = torch.ones(new, all_, dtype=torch.bool, device="cuda").triu(all_ - new + 1)
        if case["tree"]:
            words = st["tree"][start:start + new].tolist()
            hidden[:, all_ - new:] = torch.tensor([[not w >> b & 1 for b in range(new)] for w in words], device="cuda")
        q = st["q"][start:start + new].double().view(new, n_kv, group, DIM)
        for h in range(n_kv):
            s = torch.einsum("qgd,kd->gqk", q[:, h], k[:, h]) * st["scale"]
            out[start:start + new, h] = torch.einsum("gqk,kd->qgd", torch.softmax(s.masked_fill_(hidden, -math.inf), dim=-1), v[:, h])
    return out.view(len(st["q"]), n_q * DIM)
