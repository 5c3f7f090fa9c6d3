"""What the tests of the 8-bit cache's attention hold its two kernels to (a helper, no tests of its own).

`check` computes every row in 64 bits from the stored codes and scales of the tokens that it sees, and none other, and allows

  both:      half a step of the result in bf16 (2^-8 of it); 2^-133, half a step of the smallest bf16 numbers;
  "rows"     (csrc/attention8.cu): 2^-11 of sum p |v| for a weight (probability times its value's scale) as one f16 number, and 2^-11 for
             sums, exponentials and factors in fp32.  Keys are exact: a score is off by fp32 sums alone, eight MMAs of sixteen products,
             each off by 2^-22 of what it adds up at most: 2^-19 |scale| sum |q k|.  Weights are held times 2^7 / r, r at most twice the row's
             largest weight: half of f16's smallest step is 2^-25, so each is off by 2^-31 of that, times |c|.
  "prompt"   (csrc/attention8_prompt.cu): 2^-9 of sum p |v| (a probability, a value's scale and their code's product in f16, 2^-11
             each, and fp32).  A key's number is off by 2^-11 of itself (2^-16 of it for the two f16 numbers of its scale and the
             fp32 sum) and (but for zeros) by half of f16's smallest step of the tile's unit, 2^-25 * 2^13 / 16 = 2^-16 of its scale.  Values: 2^-25 * 2^13 / 64 =
             2^-18 of the scale; probabilities: 2^-31 of what the row's largest one stands for, whose unit may be 2^12 above its own scale.

A query's number is held in f16 where the largest of its row is 2^14 at least.  It is exact there from 2^-17 on (bf16 has 8 bits, f16's smallest step is
2^-24), which 2^-31 of the largest is; a smaller one, if it is not zero, is off by half a step, 2^-25, which is 2^-39 of the largest.  A score is off by that times |scale| sum |k|
over such numbers, in both.

A score off by d changes a weight by exp(d) and the sum that all is divided by as well: two tokens' d together, those of the two largest among tokens
whose p is not below 2^-40 (a lone one's does not matter, and one far below them stays there).
"""
import math
import random

import torch

from vllm_tgis_adapter_b200.engine.cache8 import PAGE_BYTES, Cache8

D, PAGE = 128, 32


def ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def still():
    return torch.tensor([1.0] * 64 + [0.0] * 64, device="cuda", dtype=torch.bfloat16).view(1, D)


def cache_of(n_pages, n_kv, k, v):
    """A cache whose slots hold the rows k, v [n_pages * 32, n_kv, 128]."""
    cache, n = Cache8.empty(n_pages, n_kv), n_pages * PAGE
    every = torch.arange(n, device="cuda", dtype=torch.int32)
    cache.write(torch.cat([k, v], dim=1).to(torch.bfloat16).reshape(n, -1), torch.zeros_like(every), every, still())
    return cache


def stored(cache):
    """(codes, scales) of keys and of values of every slot: [slots, n_kv, 128] and [slots, n_kv, 1] in 64 bits."""
    raw = cache.pages.view(cache.n_pages * cache.n_kv, PAGE_BYTES)
    t, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(D, device="cuda")[None]
    k_at = t * D + (((d >> 4) ^ (t & 7)) << 4) + (d & 15)
    h = t & 15
    v_at = 4096 + (t >> 4) * 2048 + d * 16 + ((h >> 1 & 3) << 2 | (h >> 3 & 1) << 1 | (h & 1))
    out = []
    for at, scale_at in ((k_at, 8192), (v_at, 8320)):
        codes = raw[:, at.reshape(-1)].view(torch.float8_e4m3fn).double()
        scale = raw[:, scale_at:scale_at + 128].contiguous().view(torch.float32).double()
        natural = lambda x, w: x.view(cache.n_pages, cache.n_kv, PAGE, w).transpose(1, 2).reshape(-1, cache.n_kv, w)  # noqa: E731
        out.append((natural(codes, D), natural(scale, 1)))
    return out


def layout(lengths, seed, spare=2):
    """Records, tables (pages in any order) and sizes of sequences of (new, old) tokens."""
    rng = random.Random(seed)
    need = [(n + o + PAGE - 1) // PAGE for n, o in lengths]
    n_pages = sum(need) + spare
    order, bt, seqs, at, row = rng.sample(range(n_pages), n_pages), [], [], 0, 0
    for i, (n, o) in enumerate(lengths):
        bt.append(order[at:at + need[i]] + [-1] * (max(need) - need[i]))
        seqs.append([row, n, n + o, i])
        at, row = at + need[i], row + n
    return seqs, bt, n_pages, row


def slot_of(bt, row, token):
    return bt[row][token // PAGE] * PAGE + token % PAGE


def branches(seqs, T, seed):
    rng, words = random.Random(seed), [0] * T
    for start, new, _, _ in seqs:
        for i in range(new):
            parent = rng.randint(-1, i - 1)
            words[start + i] = (words[start + parent] if parent >= 0 else 0) | 1 << i
    return words


def visible(seq, i, words):
    start, new, all_, _ = seq
    old = all_ - new
    return list(range(old + i + 1)) if words is None else list(range(old)) + [old + j for j in range(new) if words[start + i] >> j & 1]


def attend(cache, q, seqs, bt, scale, kernel, words=None):
    """By the kernel that is named: bounds choose it."""
    group = q.shape[1] // D // cache.n_kv
    max_q, max_kv = max(s[1] for s in seqs), max(s[2] for s in seqs)
    if kernel == "prompt":
        max_q, max_kv = max(max_q, 64), max(max_kv, 2000)
    else:
        assert max_q * group <= 48 or (max_kv <= 1024 and len(seqs) * cache.n_kv * ((max_q * group + 15) // 16) <= 296)
    tree = None if words is None else torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], device="cuda", dtype=torch.int64)
    return cache.attend(q, ints(seqs), ints(bt), scale, max_q, max_kv, out=torch.full_like(q, 7.0), tree=tree)


def check(cache, q, seqs, bt, scale, kernel, words=None, got=None, only=None):
    """`only`: {(sequence, query)}, where not all are to be looked at"""
    if got is None:
        got = attend(cache, q, seqs, bt, scale, kernel, words)
        cache.check()
    (kc, ks), (vc, vs) = stored(cache)
    n_q, worst = q.shape[1] // D, 0.0
    G = n_q // cache.n_kv
    for n, seq in enumerate(seqs):
        for i in range(seq[1]):
            if only is not None and (n, i) not in only:
                continue
            toks = visible(seq, i, words)
            row = got[seq[0] + i].double().view(cache.n_kv, G, D)
            if not toks:
                assert bool((row == 0).all())
                continue
            slots = torch.tensor([slot_of(bt, seq[3], t) for t in toks], device="cuda")
            c, s, codes, vscale = kc[slots], ks[slots], vc[slots], vs[slots]
            k, v = c * s, codes * vscale
            qq = q[seq[0] + i].double().view(cache.n_kv, G, D)
            p = torch.softmax(torch.einsum("hgd,khd->hgk", qq, k) * scale, dim=-1)
            want = torch.einsum("hgk,khd->hgd", p, v)
            size = torch.einsum("hgk,khd->hgd", p, v.abs())
            most = torch.einsum("hgd,khd->hgk", qq.abs(), k.abs()) * abs(scale)
            weight = p * vscale[..., 0].t()[:, None]
            low = weight.amax(-1, keepdim=True) * codes.abs().sum(0)[:, None]
            if kernel == "rows":
                d, plain, floor = 2.0 ** -19 * most, 2.0 ** -10, 2.0 ** -31 * low
            else:
                d = (2.0 ** -11 + 2.0 ** -16) * most + 2.0 ** -16 * abs(scale) * torch.einsum("hgd,khd->hgk", qq.abs(), (c != 0).double()) * s[..., 0].t()[:, None]
                plain, floor = 2.0 ** -9, 2.0 ** -19 * low + 2.0 ** -18 * weight.sum(-1, keepdim=True)
            top = qq.abs().amax(-1, keepdim=True)
            d = d + 2.0 ** -39 * abs(scale) * top * torch.einsum("hgd,khd->hgk", ((qq.abs() < 2.0 ** -31 * top) & (qq != 0)).double(), k.abs())
            d = torch.where(p > 2.0 ** -40, d, 0.0)
            two = d.topk(min(2, d.shape[-1]), dim=-1).values.sum(-1, keepdim=True)
            two = torch.where((p > 2.0 ** -40).sum(-1, keepdim=True) > 1, two, 0.0)
            assert float(two.max()) < 0.05, "scores too large for a check that says something"
            may = (2.0 ** -8 * want.abs() + (plain + torch.expm1(two)) * size + floor) * (1 + 2.0 ** -8) + 2.0 ** -133
            off = (row - want).abs()
            assert bool((off <= may).all()), f"sequence {seq}, query {i}: off by {(off / may).nan_to_num(nan=math.inf).max().item():.4g} of what it may"
            worst = max(worst, (off / may).max().item())
    return worst
