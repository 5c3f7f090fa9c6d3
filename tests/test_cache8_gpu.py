"""The 8-bit paged cache and attention over it (csrc/cache8.cu, csrc/attention8.cu) against 64-bit arithmetic.

Tolerances.  Stored rows: x / s is rounded to 3 bits behind the first: half a step, 2^-4 relative, or 2^-10 s below the normal range (2^-6 s);
the code of an fp32 rotation may be that of the neighbouring step where the 64-bit one lies on the border.  Attention reads exact
operands (codes times scales).  A probability times its value row's scale s is one f16 number (half a step: 2^-11); with more than 16 rows a
sequence and kv head (max_q * group) the value, code times s in f16, is another (s and the product 2^-11 each); the result is rounded to bf16 (half
a step: 2^-8): |out - exact| <= (2^-8 + 2^-9) * sum p |v| elementwise, 2^-11 of which cover fp32 sums, exponentials and scores.
f16's smallest step adds: a weight is held times 2^7 / r, r at most 2 max s, so that half of 2^-24 is 2^-31 max s, and what a number c s of
the sum is off by |c| times that; values that are held in f16 lose as much at most: 2^-30 max s * sum |c| in all (p <= 1 and the sum of p that all
is divided by is 1 at least, against the row's largest score; the reference lies up to 2^8 below it, which only raises both).
Keys of calls with more than 16 rows are held in f16 too: each number is off by 2^-11 of itself, a score by d = 2^-11 |scale| sum |q k| at most, a
weight by a factor between exp(-2 d) and exp(2 d) for the largest d of the row.
"""
import math
import random
import subprocess
import sys

import pytest
import torch

from vllm_tgis_adapter_b200.engine.cache8 import PAGE_BYTES, Cache8

pytestmark = pytest.mark.gpu
D, PAGE, TINY = 128, 32, 2.0 ** -126
TOL = 2.0 ** -8 + 2.0 ** -9


def to_e4m3(y: torch.Tensor) -> torch.Tensor:
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def table(n=300):
    angle = torch.outer(torch.arange(n, dtype=torch.float64), 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)))
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(torch.bfloat16).cuda()


def still():
    return torch.tensor([1.0] * 64 + [0.0] * 64, device="cuda", dtype=torch.bfloat16).view(1, D)


def ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def pages_natural(cache: Cache8):
    """Values of every slot by the documented layout, in 64 bits: keys and values [slots, n_kv, 128]."""
    raw = cache.pages.view(cache.n_pages * cache.n_kv, PAGE_BYTES)
    n = raw.shape[0]
    t, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(D, device="cuda")[None]
    k_at = t * D + (((d >> 4) ^ (t & 7)) << 4) + (d & 15)
    h = t & 15
    v_at = 4096 + (t >> 4) * 2048 + d * 16 + ((h >> 1 & 3) << 2 | (h >> 3 & 1) << 1 | (h & 1))
    out = []
    for at, scale_at in ((k_at, 8192), (v_at, 8320)):
        codes = raw[:, at.reshape(-1)].view(torch.float8_e4m3fn).double().view(n, PAGE, D)
        scale = raw[:, scale_at:scale_at + 128].contiguous().view(torch.float32).double()
        out.append((codes * scale[..., None]).view(cache.n_pages, cache.n_kv, PAGE, D).transpose(1, 2).reshape(-1, cache.n_kv, D))
    return out


def scales_natural(cache: Cache8, i: int):
    """fp32 scales of every slot's key (0) or value (1) row, in 64 bits [slots, n_kv]."""
    raw = cache.pages.view(cache.n_pages * cache.n_kv, PAGE_BYTES)[:, 8192 + 128 * i:8320 + 128 * i].contiguous()
    return raw.view(torch.float32).double().view(cache.n_pages, cache.n_kv, PAGE).transpose(1, 2).reshape(-1, cache.n_kv)


def filled(n_pages, n_kv, seed, spread=0.5):
    g = gen(seed)
    cache = Cache8.empty(n_pages, n_kv)
    n = n_pages * PAGE
    x = torch.randn(n, 2 * n_kv * D, device="cuda", generator=g) * torch.exp(spread * torch.randn(n, 1, device="cuda", generator=g))
    cache.write(x.to(torch.bfloat16), torch.zeros(n, device="cuda", dtype=torch.int32), torch.arange(n, device="cuda", dtype=torch.int32), still())
    return cache


def reference(cache, q, seqs, bt, scale, tree=None):
    """(out, sum p |v|, largest |scale| sum |q k|) in 64 bits; rows that see nothing are zeros, rows without a sequence NaN."""
    k, v = pages_natural(cache)
    T, n_q = q.shape[0], q.shape[1] // D
    G = n_q // cache.n_kv
    out = torch.full((T, n_q, D), math.nan, dtype=torch.float64, device="cuda")
    size, most = out.clone(), torch.zeros(T, n_q, 1, dtype=torch.float64, device="cuda")
    for start, new, all_, row in seqs:
        for i in range(new):
            old = all_ - new
            toks = list(range(old + i + 1)) if tree is None else list(range(old)) + [old + j for j in range(new) if tree[start + i] >> j & 1]
            if not toks:
                out[start + i], size[start + i] = 0, 0
                continue
            tt = torch.tensor(toks, device="cuda")
            slot = torch.tensor(bt[row], device="cuda")[tt // PAGE] * PAGE + tt % PAGE
            kk, vv = k[slot], v[slot]
            qq = q[start + i].double().view(cache.n_kv, G, D)
            p = torch.softmax(torch.einsum("hgd,khd->hgk", qq, kk) * scale, dim=-1)
            out[start + i] = torch.einsum("hgk,khd->hgd", p, vv).reshape(n_q, D)
            size[start + i] = torch.einsum("hgk,khd->hgd", p, vv.abs()).reshape(n_q, D)
            most[start + i] = (torch.einsum("hgd,khd->hgk", qq.abs(), kk.abs()).amax(-1) * abs(scale)).reshape(n_q, 1)
    return out.view(T, -1), size.view(T, -1), most.expand(T, n_q, D).reshape(T, -1)


def floor_of(cache, seqs, bt, T, n_q):
    """2^-30 max s * sum |c| over the tokens of a row's sequence."""
    s, v = scales_natural(cache, 1), pages_natural(cache)[1]
    low = torch.zeros(T, cache.n_kv, D, dtype=torch.float64, device="cuda")
    for start, new, all_, row in seqs:
        if new:
            t = torch.arange(all_, device="cuda")
            slot = torch.tensor(bt[row], device="cuda")[t // PAGE] * PAGE + t % PAGE
            low[start:start + new] = (2.0 ** -30 * s[slot].amax(0)[:, None] * (v[slot] / s[slot][..., None]).abs().sum(0))[None]
    return low.repeat_interleave(n_q // cache.n_kv, dim=1).view(T, -1)


def batch(lengths, seed, extra_rows=0, extra_pages=2, gap=0):
    """Records, table and sizes of sequences of (new, old) tokens; pages in any order, unused table entries -1, `gap` rows between sequences."""
    rng = random.Random(seed)
    need = [(n + o + PAGE - 1) // PAGE for n, o in lengths]
    n_pages = sum(need) + extra_pages
    order, at, row = rng.sample(range(n_pages), n_pages), 0, 0
    width = max(max(need), 1)
    bt, seqs = [], []
    for i, (n, o) in enumerate(lengths):
        bt.append(order[at:at + need[i]] + [-1] * (width - need[i]))
        seqs.append([row, n, n + o, i])
        at += need[i]
        row += n + gap
    return seqs, bt, n_pages, row + extra_rows


def attend_case(lengths, n_q, n_kv, seed, tree=None, scale=D ** -0.5, q_size=1.0, gap=0, extra_rows=0, max_more=0, cache=None):
    seqs, bt, n_pages, T = batch(lengths, seed, extra_rows, gap=gap)
    cache = cache or filled(n_pages, n_kv, seed)
    q = (q_size * torch.randn(T, n_q * D, device="cuda", generator=gen(seed + 1))).to(torch.bfloat16)
    words = tree(seqs, T, seed) if tree else None
    t = torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], device="cuda", dtype=torch.int64) if tree else None
    out = torch.full_like(q, 7.0)
    max_q, max_kv = max(s[1] for s in seqs) + (0 if tree else max_more), max(s[2] for s in seqs) + max_more
    got = cache.attend(q, ints(seqs), ints(bt), scale, max_q, max_kv, out=out, tree=t)
    cache.check()
    want, size, most = reference(cache, q, seqs, bt, scale, words)
    keys = torch.expm1(2 * 2.0 ** -11 * most) if max_q * (n_q // n_kv) > 16 else torch.zeros_like(most)
    named = ~want.isnan().all(dim=1)
    assert bool((got[~named] == 7.0).all()), "rows that no sequence names were touched"
    off = (got[named].double() - want[named]).abs()
    # (2^-133: half a step of the smallest bf16 numbers)
    may = (TOL + keys[named]) * size[named] + floor_of(cache, seqs, bt, T, n_q)[named] + 2.0 ** -133
    assert bool((off <= may).all()), f"off by {(off / may).max().item():.4g} of what it may"
    return cache, q, seqs, bt, got


# ------------------------------------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("T,n_q,n_kv", [(1, 4, 1), (3, 32, 8), (17, 6, 2), (96, 12, 12), (33, 0, 3), (130, 64, 8)])
def test_rows_are_rotated_quantised_and_read_back(T, n_q, n_kv):
    n_pages = 9
    cache = Cache8.empty(n_pages, n_kv)
    g = gen(T)
    qkv = (torch.randn(T, (n_q + 2 * n_kv) * D + 64, device="cuda", generator=g) * 3).to(torch.bfloat16)[:, 8:8 + (n_q + 2 * n_kv) * D]   # (strided rows)
    rng = random.Random(T)
    slots = rng.sample(range(n_pages * PAGE), T)
    places = [rng.randrange(300) for _ in range(T)]
    cs = table()
    q = cache.write(qkv, ints(places), ints(slots), cs)
    k, v = cache.read(ints(slots))
    cache.check()
    x = qkv.double().reshape(T, n_q + 2 * n_kv, 2, 64)
    c = cs.double()[ints(places).long()].view(T, 1, 2, 64)
    turned = torch.stack([x[:, :, 0] * c[:, :, 0] - x[:, :, 1] * c[:, :, 1], x[:, :, 1] * c[:, :, 0] + x[:, :, 0] * c[:, :, 1]], dim=2).reshape(T, -1, D)
    # (a bf16 rotation: fp32 products and one sum, 3 * 2^-24 of |a c| + |b s| at most, then half a step of bf16)
    if n_q:
        want = turned[:, :n_q].reshape(T, -1)
        big = torch.stack([x.abs()[:, :, 0] + x.abs()[:, :, 1]] * 2, dim=2).reshape(T, -1, D)[:, :n_q].reshape(T, -1)
        assert bool(((q.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * big).all())
    else:
        assert q is None
    nat = pages_natural(cache)
    at = ints(slots).long()
    for i, (got, stored, rows) in enumerate(((k, nat[0][at], turned[:, n_q:n_q + n_kv]), (v, nat[1][at], x.reshape(T, -1, D)[:, n_q + n_kv:]))):
        s = scales_natural(cache, i)[at][..., None]
        assert bool((s / (rows.abs().amax(-1, keepdim=True) / 448.0).clamp(min=TINY) - 1).abs().max() < 2.0 ** -21)
        # half a step of the code; 2^-15 of that and 2^-22 of the largest number for the fp32 rotation, scale and quotient
        assert bool(((stored - rows).abs() <= torch.maximum(rows.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -15) + 448 * s * 2.0 ** -22).all())
        near = to_e4m3(rows / s) * s
        assert ((stored - near).abs() > 2.0 ** -20 * 448 * s).double().mean().item() < 1e-3   # (codes next to a border)
        assert bool(((got.double().view(T, n_kv, D) - stored).abs() <= 2.0 ** -8 * stored.abs()).all())
    # nothing else was written
    other = torch.ones(n_pages * PAGE, dtype=torch.bool, device="cuda")
    other[at] = False
    assert bool((nat[0][other] == 0).all()) and bool((nat[1][other] == 0).all())


def test_codes_of_values_are_those_of_torch():
    """No rotation: the quotient, the rounding and the scale are IEEE operations, so every code is that of the plain form."""
    g = gen(5)
    x = (torch.randn(64, 2 * D, device="cuda", generator=g) * torch.exp(4 * torch.randn(64, 1, device="cuda", generator=g))).to(torch.bfloat16)
    x[3] = 0
    x[4] = x[4] * 1e-38
    cache = Cache8.empty(2, 1)
    cache.write(x, ints([0] * 64), ints(list(range(64))), still())
    rows = x.float().view(64, 2, D)
    s = (rows.abs().amax(-1) * torch.tensor(1.0 / 448.0, device="cuda")).clamp(min=TINY)
    want = (rows / s[..., None]).to(torch.float8_e4m3fn).double() * s.double()[..., None]
    k, v = pages_natural(cache)
    assert torch.equal(k[:, 0], want[:, 0]) and torch.equal(v[:, 0], want[:, 1])


def test_rotation_in_place_and_without_queries():
    g = gen(6)
    qkv = torch.randn(5, 8 * D, device="cuda", generator=g).to(torch.bfloat16)
    cs, places, slots = table(), ints([0, 5, 9, 200, 299]), ints([3, 4, 40, 41, 2])
    one, two, three = Cache8.empty(2, 2), Cache8.empty(2, 2), Cache8.empty(2, 2)
    q = one.write(qkv, places, slots, cs)
    assert two.write(qkv, places, slots, cs, want_q=False) is None
    same = qkv.clone()
    in_place = three.write(same, places, slots, cs, q_out=same[:, : 4 * D])
    assert in_place.data_ptr() == same.data_ptr() and torch.equal(same[:, : 4 * D], q) and torch.equal(same[:, 4 * D:], qkv[:, 4 * D:])
    assert torch.equal(one.pages, two.pages) and torch.equal(one.pages, three.pages)


def test_rows_that_are_not_finite_are_nan_as_a_whole():
    x = torch.ones(4, 4 * D, device="cuda", dtype=torch.bfloat16)
    x[0, 5], x[1, D + 3], x[2, 2 * D + 7] = math.nan, math.inf, -math.inf
    cache = Cache8.empty(1, 2)
    cache.write(x, ints([0] * 4), ints([0, 1, 2, 3]), still())
    k, v = cache.read(ints([0, 1, 2, 3]))
    bad_k, bad_v = k.view(4, 2, D).isnan(), v.view(4, 2, D).isnan()
    want = torch.zeros(4, 2, dtype=torch.bool, device="cuda")
    want[0, 0] = want[1, 1] = True
    assert torch.equal(bad_k.all(-1), want) and torch.equal(bad_k.any(-1), want)
    want = torch.zeros(4, 2, dtype=torch.bool, device="cuda")
    want[2, 0] = True
    assert torch.equal(bad_v.all(-1), want) and torch.equal(bad_v.any(-1), want)


def test_slots_and_positions_out_of_range_are_left_out_and_reported():
    x = torch.ones(4, 3 * D, device="cuda", dtype=torch.bfloat16)
    cache = Cache8.empty(2, 1)
    cache.write(x, ints([0] * 4), ints([-1, 64, 2 ** 31 - 1, 5]), still())
    with pytest.raises(RuntimeError, match="slot"):
        cache.check()
    cache.check()
    k, _ = pages_natural(cache)
    assert k[:, 0, 0].nonzero().flatten().tolist() == [5]
    k, v = cache.read(ints([5, -3, 64]))
    assert bool((k[0] == 1).all()) and bool((k[1:] == 0).all()) and bool((v[1:] == 0).all())
    with pytest.raises(RuntimeError, match="slot"):
        cache.check()
    cache.write(x, ints([0, 1, -1, 0]), ints([1, 2, 3, 4]), still())
    with pytest.raises(RuntimeError, match="position"):
        cache.check()


# ---------------------------------------------------------------------------------------------------------- attention
HEADS = [(4, 1), (6, 2), (32, 8), (16, 2), (3, 3), (10, 2), (24, 2)]


@pytest.mark.parametrize("n_q,n_kv", HEADS)
def test_single_tokens(n_q, n_kv):
    attend_case([(1, n) for n in (0, 1, 15, 16, 30, 31, 32, 33, 126, 127, 128, 300, 700)], n_q, n_kv, n_q)


@pytest.mark.parametrize("n_q,n_kv", HEADS)
def test_portions_of_prompts(n_q, n_kv):
    attend_case([(2, 0), (7, 3), (33, 0), (31, 1), (64, 64), (5, 300), (1, 40), (130, 0), (70, 131)], n_q, n_kv, n_q + 1, gap=2, extra_rows=3)


@pytest.mark.parametrize("n_q,n_kv", [(64, 1), (40, 1), (128, 1), (150, 1), (34, 2)])
def test_wide_groups(n_q, n_kv):
    """More query heads than a tile of rows, than half an accumulator, than one."""
    attend_case([(1, 0), (1, 90), (3, 200), (1, 300), (9, 0)], n_q, n_kv, n_q)
    attend_case([(1, 0), (1, 90), (1, 700)], n_q, n_kv, n_q + 1)
    attend_case([(3, 40), (7, 200)], n_q, n_kv, n_q + 2, tree=branches)


def test_many_sequences():
    """More sequences than a CTA has threads, most of them empty or bad; pages shared by many."""
    cache, rng = filled(40, 2, 77), random.Random(5)
    for most_q, n in ((1, 3000), (40, 1500)):
        seqs, bt, row = [], [], 0
        for i in range(n):
            new = rng.randint(1, most_q) if i % 3 else 0
            old = rng.randint(0, 150)
            seqs.append([row, new, new + old, i])
            row += new
            bt.append([rng.randrange(40) for _ in range(6)])
        q = torch.randn(row, 4 * D, device="cuda", generator=gen(n)).to(torch.bfloat16)
        out = torch.full_like(q, 7.0)
        cache.attend(q, ints(seqs), ints(bt), D ** -0.5, most_q, 190, out=out)
        cache.check()
        some = rng.sample([s for s in seqs if s[1]], 40) + [s for s in seqs if s[1]][-3:]
        want, size, most = reference(cache, q, some, bt, D ** -0.5)
        named = ~want.isnan().all(dim=1)
        may = (TOL + torch.expm1(2 * 2.0 ** -11 * most[named])) * size[named] + 1e-6
        assert int(named.sum()) > 40 and bool(((out[named].double() - want[named]).abs() <= may).all())


def test_a_step_captured_before_any_call_and_replayed_on_two_streams(tmp_path):
    """A process whose first calls are captured; two graphs with workspaces of their own at the same time."""
    code = f"""
import sys; sys.path[:0] = {sys.path[:2]!r}
import torch
from vllm_tgis_adapter_b200.engine.cache8 import Cache8
cache = Cache8.empty(64, 2)
still = torch.tensor([1.0] * 64 + [0.0] * 64, device="cuda").bfloat16().view(1, 128)
n = 64 * 32
rows = torch.randn(n, 512, device="cuda").bfloat16()
zero, every = torch.zeros(n, device="cuda", dtype=torch.int32), torch.arange(n, device="cuda", dtype=torch.int32)
bt = torch.arange(64, device="cuda", dtype=torch.int32).view(1, 64)
jobs = []
for new in (1, 90):
    q = torch.randn(new, 512, device="cuda").bfloat16()
    seqs = torch.tensor([[0, new, 2000, 0]], device="cuda", dtype=torch.int32)
    jobs.append((q, seqs, new, torch.zeros_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()))
first = torch.cuda.CUDAGraph()
with torch.cuda.graph(first):
    cache.write(rows, zero, every, still)
for q, seqs, new, out, stream, graph in jobs:
    with torch.cuda.graph(graph, stream=stream):
        cache.attend(q, seqs, bt, 0.1, new, 2048, out=out)
first.replay()
torch.cuda.synchronize()
for _ in range(50):
    for q, seqs, new, out, stream, graph in jobs:
        with torch.cuda.stream(stream):
            graph.replay()
torch.cuda.synchronize()
for q, seqs, new, out, stream, graph in jobs:
    assert torch.equal(out, cache.attend(q, seqs, bt, 0.1, new, 2048)) and bool(out.isfinite().all()) and bool((out != 0).any())
cache.check()
print("right")
"""
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "right" in got.stdout, got.stderr[-2000:]


def chains(seqs, T, seed):
    words = [0] * T
    for start, new, _, _ in seqs:
        for i in range(new):
            words[start + i] = (2 << i) - 1
    return words


def branches(seqs, T, seed):
    rng = random.Random(seed)
    words = [0] * T
    for start, new, _, _ in seqs:
        for i in range(new):
            parent = rng.randint(-1, i - 1)
            words[start + i] = (words[start + parent] if parent >= 0 else 0) | 1 << i
    return words


def any_words(seqs, T, seed):
    """Any bits, those behind the draft and empty words among them."""
    rng = random.Random(seed)
    return [rng.getrandbits(64) if rng.random() < 0.8 else 0 for _ in range(T)]


@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("tree", [chains, branches, any_words])
def test_trees(n_q, n_kv, tree):
    attend_case([(1, 0), (2, 0), (8, 24), (8, 25), (24, 200), (64, 0), (64, 31), (63, 300), (5, 127), (3, 128)], n_q, n_kv, n_q + 2, tree=tree, gap=1, extra_rows=2)


def test_a_chain_is_the_causal_mask():
    lengths = [(9, 100), (16, 0), (4, 300)]
    _, q, seqs, bt, a = attend_case(lengths, 8, 2, 3)
    cache, q2, _, _, b = attend_case(lengths, 8, 2, 3, tree=chains)
    assert torch.equal(q, q2) and torch.equal(a, b)


@pytest.mark.parametrize("tree", [None, chains])
def test_large_scores_small_and_negative_scales(tree):
    for scale, size in ((1.0, 4.0), (-0.2, 1.0), (0.0, 1.0), (0.1, 1e-30), (1e-30, 1e30), (1e-3, 3.0)):
        attend_case([(6, 40), (1, 200), (20, 0)], 4, 2, 9, tree=tree, scale=scale, q_size=size)


@pytest.mark.parametrize("spread", [0.0, 6.0, 20.0])
def test_rows_of_very_different_sizes(spread):
    seqs, bt, n_pages, T = batch([(1, 500), (6, 300), (40, 60)], 11)
    cache = filled(n_pages, 2, 12, spread)
    attend_case([(1, 500), (6, 300), (40, 60)], 4, 2, 11, cache=cache, scale=1e-3 if spread < 10 else 1e-9)


def test_rows_whose_mask_leaves_nothing_are_zeros():
    seqs, bt, n_pages, T = batch([(4, 0), (3, 50)], 2)
    cache = filled(n_pages, 1, 2)
    q = torch.randn(T, 2 * D, device="cuda", generator=gen(3)).to(torch.bfloat16)
    out = cache.attend(q, ints(seqs), ints(bt), 0.1, 4, 53, tree=torch.tensor([0, 2, 1 << 10, 8, 0, 0, 0], device="cuda"))
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all()) and bool((out[1] != 0).any()) and bool((out[4:] != 0).any(dim=1).all())


def test_numbers_that_are_not_finite_stay_with_the_rows_that_see_them():
    lengths = [(6, 90), (1, 63), (40, 8)]
    seqs, bt, n_pages, T = batch(lengths, 4)
    plain = filled(n_pages, 2, 4)
    bad = Cache8(plain.pages.clone())
    slot = lambda s, t: bt[s][t // PAGE] * PAGE + t % PAGE  # noqa: E731
    x = torch.ones(3, 4 * D, device="cuda", dtype=torch.bfloat16)
    x[0, 3 * D], x[1, 0], x[2, 3 * D + 5] = math.nan, math.inf, -math.inf
    # a value of node 3 of the first sequence, a key of its node 4, a value of the third's token 30
    places = [slot(0, 93), slot(0, 94), slot(2, 30)]
    bad.write(x, ints([0] * 3), ints(places), still())
    plain.write(torch.ones_like(x), ints([0] * 3), ints(places), still())
    q = torch.randn(T, 4 * D, device="cuda", generator=gen(5)).to(torch.bfloat16)
    words = torch.tensor(branches(seqs, T, 8), device="cuda", dtype=torch.int64)
    for tree in (None, words):
        a = plain.attend(q, ints(seqs), ints(bt), 0.1, 40, 96, tree=tree)
        b = bad.attend(q, ints(seqs), ints(bt), 0.1, 40, 96, tree=tree)
        sees = lambda s, i, node: i >= node if tree is None else bool(int(words[seqs[s][0] + i]) >> node & 1)  # noqa: E731
        for s, (start, new, all_, _) in enumerate(seqs):
            for i in range(new):
                nan_heads = set()
                if s == 0 and sees(0, i, 3):
                    nan_heads |= {2, 3}       # values of kv head 1
                if s == 0 and sees(0, i, 4):
                    nan_heads |= {0, 1}       # keys of kv head 0
                if s == 2 and sees(2, i, 22):
                    nan_heads |= {2, 3}
                row_a, row_b = a[start + i].view(4, D), b[start + i].view(4, D)
                for h in range(4):
                    if h in nan_heads:
                        assert bool(row_b[h].isnan().all()), (s, i, h)
                    else:
                        # the row's own arithmetic, but for the scale that values are held in: a power of two
                        assert bool(row_b[h].isfinite().all()) and torch.allclose(row_a[h].float(), row_b[h].float(), rtol=2 * TOL, atol=1e-2), (s, i, h)


def test_queries_that_are_not_finite():
    lengths = [(1, 100), (5, 20)]
    seqs, bt, n_pages, T = batch(lengths, 6)
    cache = filled(n_pages, 1, 6)
    q = torch.randn(T, 2 * D, device="cuda", generator=gen(7)).to(torch.bfloat16)
    a = cache.attend(q, ints(seqs), ints(bt), 0.1, 5, 101)
    q[0, 3], q[3, D + 4], q[4, 0] = math.nan, math.inf, -math.inf
    b = cache.attend(q, ints(seqs), ints(bt), 0.1, 5, 101).view(T, 2, D)
    a = a.view(T, 2, D)
    for t in range(T):
        for h in range(2):
            if (t, h) in ((0, 0), (3, 1), (4, 0)):
                assert bool(b[t, h].isnan().all())
            else:
                assert torch.equal(a[t, h], b[t, h])


def test_bounds_may_be_larger_than_the_lengths():
    """Larger bounds may choose other kernels and splits: each is right."""
    for more in (0, 1, 40, 200, 1000, 9000):
        attend_case([(1, 70), (3, 200), (1, 0)], 8, 2, 21, max_more=more)


def test_bad_records_and_pages_are_left_out_and_reported():
    lengths = [(2, 60), (3, 100), (1, 40)]
    seqs, bt, n_pages, T = batch(lengths, 13)
    cache = filled(n_pages, 2, 13)
    q = torch.randn(T, 4 * D, device="cuda", generator=gen(14)).to(torch.bfloat16)
    good = cache.attend(q, ints(seqs), ints(bt), 0.1, 3, 103)
    for at, value in ((0, -1), (0, T), (0, 2 ** 31 - 1), (1, -2), (1, 4), (2, 2), (2, 104), (2, -5), (3, -1), (3, 3), (1, 2 ** 31 - 1), (2, -2 ** 31)):
        wrong = [list(s) for s in seqs]
        wrong[1][at] = value
        out = torch.full_like(q, 7.0)
        cache.attend(q, ints(wrong), ints(bt), 0.1, 3, 103, out=out)
        with pytest.raises(RuntimeError, match="record"):
            cache.check()
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[5:], good[5:]) and bool((out[2:5] == 7).all()), (at, value)
    # a page outside: its keys are left out
    for page in (-1, n_pages, 2 ** 31 - 1, -2 ** 31):
        wrong = [list(r) for r in bt]
        wrong[1][1] = page
        out = cache.attend(q, ints(seqs), ints(wrong), 0.1, 3, 103)
        with pytest.raises(RuntimeError, match="page"):
            cache.check()
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[5:], good[5:]) and bool(out[2:5].isfinite().all()) and not torch.equal(out[2:5], good[2:5])
    # no page at all
    out = cache.attend(q, ints(seqs), ints([[-1] * len(bt[0])] * 3), 0.1, 3, 103)
    assert bool((out == 0).all())
    with pytest.raises(RuntimeError, match="page"):
        cache.check()


def test_nothing_to_do():
    cache = filled(2, 1, 1)
    q = torch.zeros(3, 2 * D, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 5.0)
    cache.attend(q, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), ints([[0]]), 1.0, 1, 1, out=out)
    cache.attend(q, ints([[0, 0, 0, 0], [2, 0, 9, 0]]), ints([[0]]), 1.0, 1, 9, out=out)
    assert bool((out == 5).all())
    cache.check()
    assert cache.read(torch.zeros(0, dtype=torch.int32, device="cuda"))[0].shape == (0, D)
    assert cache.write(torch.zeros(0, 3 * D, device="cuda", dtype=torch.bfloat16), ints([]), ints([]), still()).shape == (0, D)


def test_strided_rows_workspace_and_repeat():
    lengths = [(4, 500), (1, 900), (1, 10)]
    cache, q, seqs, bt, got = attend_case(lengths, 8, 2, 31)
    wide = torch.zeros(q.shape[0], q.shape[1] + 264, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:8 + q.shape[1]] = q
    out = torch.full_like(wide, 3.0)
    need = cache.workspace_bytes(q.shape[0], 3, 8, 4, 901)
    for _ in range(3):
        ws = torch.randint(0, 255, (need + 16,), device="cuda", dtype=torch.uint8)
        o = cache.attend(wide[:, 8:8 + q.shape[1]], ints(seqs), ints(bt), D ** -0.5, 4, 901, out=out[:, 16:16 + q.shape[1]], workspace=ws)
        assert torch.equal(o, got)
    assert bool((out[:, :16] == 3).all()) and bool((out[:, 16 + q.shape[1]:] == 3).all())
    if need:
        with pytest.raises(ValueError, match="workspace"):
            cache.attend(q, ints(seqs), ints(bt), 1.0, 4, 901, workspace=torch.zeros(need - 1, device="cuda", dtype=torch.uint8))


def test_replayed_step_on_another_stream():
    """Write, attend and read captured once; lengths, pages, slots and rows change between replays."""
    n_q, n_kv, n = 8, 2, 3
    cache, check = Cache8.empty(40, n_kv), Cache8.empty(40, n_kv)
    g, cs = gen(8), table(1200)
    qkv = torch.zeros(n, (n_q + 2 * n_kv) * D, device="cuda", dtype=torch.bfloat16)
    places, slots = ints([0] * n), ints([-1] * n)
    bt = ints([[i * 12 + j for j in range(12)] for i in range(n)])
    seqs = ints([[i, 1, 1, i] for i in range(n)])
    out, stream = torch.zeros(n, n_q * D, device="cuda", dtype=torch.bfloat16), torch.cuda.Stream()

    def step(c, to):
        q = c.write(qkv, places, slots, cs)
        c.attend(q, seqs, bt, D ** -0.5, 1, 384, out=to)
        return c.read(slots)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(cache, out)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        k, v = step(cache, out)
    for s in range(150):
        lens = [s + 1, 2 * s + 1, s % 7 + 1]
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g).to(torch.bfloat16))
        places.copy_(ints([x - 1 for x in lens]))
        slots.copy_(ints([int(bt[i, (x - 1) // PAGE]) * PAGE + (x - 1) % PAGE for i, x in enumerate(lens)]))
        seqs.copy_(ints([[i, 1, x, i] for i, x in enumerate(lens)]))
        graph.replay()
        if s % 37 == 0 or s == 149:
            want = torch.zeros_like(out)
            check.pages.copy_(cache.pages)
            k2, v2 = step(check, want)
            assert torch.equal(out, want) and torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(check.pages, cache.pages)
    cache.check()


def test_a_conversation_over_the_cache():
    """A prompt in two portions, then drafts of which a path is accepted: the same rows as one causal pass over the accepted tokens."""
    n_q, n_kv, total = 8, 2, 150
    g, cs = gen(17), table()
    qkv = torch.randn(total, (n_q + 2 * n_kv) * D, device="cuda", generator=g).to(torch.bfloat16)
    scale = D ** -0.5
    whole, steps = Cache8.empty(6, n_kv), Cache8.empty(6, n_kv)
    bt = ints([[3, 1, 4, 0, 5]])
    slot = lambda t: [3, 1, 4, 0, 5][t // PAGE] * PAGE + t % PAGE  # noqa: E731
    q = whole.write(qkv, ints(list(range(total))), ints([slot(t) for t in range(total)]), cs)
    want = whole.attend(q, ints([[0, total, total, 0]]), bt, scale, total, total)
    got = torch.zeros_like(want)
    at = 0
    for n in (90, 37):
        q = steps.write(qkv[at:at + n], ints(list(range(at, at + n))), ints([slot(t) for t in range(at, at + n)]), cs)
        got[at:at + n] = steps.attend(q, ints([[0, n, at + n, 0]]), bt, scale, n, at + n)
        at += n
    while at < total:
        # nodes 0, 2, 4 are the tokens to come (a path); 1, 3 are drafts that are not taken
        n = min(3, total - at)
        nodes = [0, None, 1, None, 2][: 2 * n - 1]
        rows = torch.stack([qkv[at + i] if i is not None else -qkv[at] for i in nodes])
        depth = [0, 0, 1, 1, 2][: len(nodes)]
        words = [0b1, 0b10, 0b101, 0b1010, 0b10101][: len(nodes)]
        m = len(nodes)
        # (a draft may reach behind the last page: it is cut there)
        m = min(m, 5 * PAGE - at)
        q = steps.write(rows[:m], ints([at + d for d in depth[:m]]), ints([slot(at + j) for j in range(m)]), cs)
        out = steps.attend(q, ints([[0, m, at + m, 0]]), bt, scale, m, at + m, tree=torch.tensor(words[:m], device="cuda"))
        taken = [j for j in range(m) if nodes[j] is not None]
        for j in taken:
            got[at + nodes[j]] = out[j]
        # the accepted rows move to their places: written again, as the path's tokens
        steps.write(torch.stack([rows[j] for j in taken]), ints([at + nodes[j] for j in taken]), ints([slot(at + nodes[j]) for j in taken]), cs, want_q=False)
        at += len(taken)
    whole.check(), steps.check()
    assert torch.equal(whole.pages.view(6, n_kv, -1)[[3, 1, 4, 0]], steps.pages.view(6, n_kv, -1)[[3, 1, 4, 0]])
    # other splits and orders of the same sums: each within TOL of exact
    _, size, most = reference(whole, q_all(whole, qkv, cs, total), [[0, total, total, 0]], bt.tolist(), scale)
    assert bool(((got.double() - want.double()).abs() <= 2 * (TOL + torch.expm1(2 * 2.0 ** -11 * most)) * size + 1e-6).all())


def q_all(cache, qkv, cs, total):
    return Cache8.empty(6, cache.n_kv).write(qkv, ints(list(range(total))), ints([-1] * total), cs)


# ------------------------------------------------------- the kernel of long prompts on short sequences (bounds choose between the two)
@pytest.mark.parametrize("n_q,n_kv", HEADS)
def test_portions_in_bounds_of_long_prompts(n_q, n_kv):
    attend_case([(2, 0), (7, 3), (33, 0), (31, 1), (64, 64), (5, 300), (1, 40), (130, 0), (70, 131), (1, 0), (1, 127), (1, 128)], n_q, n_kv, n_q + 1, gap=2, extra_rows=3, max_more=2000)


@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("tree", [chains, branches, any_words])
def test_trees_in_bounds_of_long_contexts(n_q, n_kv, tree):
    attend_case([(1, 0), (2, 0), (8, 24), (24, 200), (64, 0), (63, 300), (5, 127), (3, 128), (64, 64)], n_q, n_kv, n_q + 2, tree=tree, gap=1, extra_rows=2, max_more=2000)


@pytest.mark.parametrize("tree", [None, chains])
def test_large_scores_in_bounds_of_long_prompts(tree):
    for scale, size in ((1.0, 4.0), (-0.2, 1.0), (0.0, 1.0), (0.1, 1e-30), (1e-30, 1e30), (1e-3, 3.0)):
        attend_case([(6, 40), (1, 200), (20, 0), (64, 9)], 4, 2, 9, tree=tree, scale=scale, q_size=size, max_more=2000)


@pytest.mark.parametrize("spread", [0.0, 6.0, 20.0])
def test_rows_of_very_different_sizes_in_bounds_of_long_prompts(spread):
    seqs, bt, n_pages, T = batch([(1, 500), (6, 300), (40, 60)], 11)
    cache = filled(n_pages, 2, 12, spread)
    attend_case([(1, 500), (6, 300), (40, 60)], 4, 2, 11, cache=cache, scale=1e-3 if spread < 10 else 1e-9, max_more=2000)


@pytest.mark.parametrize("case", [test_rows_whose_mask_leaves_nothing_are_zeros, test_numbers_that_are_not_finite_stay_with_the_rows_that_see_them,
                                  test_queries_that_are_not_finite])
def test_empty_rows_and_no_numbers_in_bounds_of_long_prompts(case, monkeypatch):
    attend = Cache8.attend
    monkeypatch.setattr(Cache8, "attend", lambda self, q, seqs, bt, scale, max_q, max_kv, **more: attend(self, q, seqs, bt, scale, max(max_q, 64), max(max_kv, 2000), **more))
    case()


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (32, 8), (3, 3)])
def test_a_few_queries_behind_long_contexts(n_q, n_kv):
    """17 to 48 rows a sequence and splits: several chunks of rows, each joined over its splits."""
    most = 48 // (n_q // n_kv)
    attend_case([(most, 1500), (most - 3, 900), (1, 2100), (2, 0), (5, 770)], n_q, n_kv, 31)
    attend_case([(most, 1100), (most - 3, 900), (1, 40)], n_q, n_kv, 32, tree=branches)
