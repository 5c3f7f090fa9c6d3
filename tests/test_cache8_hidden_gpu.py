"""Attention over the 8-bit cache: a row's result is that of the tokens that it sees, whatever finite numbers the others hold; and of tokens
that it sees those count whose probability does, whatever the others' size."""
import pytest
import torch

from cache8_checks import D, PAGE, attend, branches, cache_of, check, layout, slot_of, visible

pytestmark = pytest.mark.gpu
N_Q, N_KV = 8, 2
DRAFTS = [("rows", [(12, 300), (5, 60), (1, 40), (12, 0)]), ("prompt", [(12, 300), (5, 60), (1, 40), (12, 0)]), ("prompt", [(64, 100), (40, 0), (61, 3), (64, 300)])]
CASES = [c + (t,) for c in DRAFTS for t in (None, branches)] + [("prompt", [(300, 0), (129, 171), (200, 0)], None)]


def rows(n_pages, seed, q_rows):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = torch.randn(2, n_pages * PAGE, N_KV, D, device="cuda", generator=g)
    return k, v, torch.randn(q_rows, N_Q * D, device="cuda", generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("kernel,lengths,tree", CASES)
@pytest.mark.parametrize("power", [-60, 10, 21, 40, 100])
@pytest.mark.parametrize("what", ["keys", "values", "both"])
def test_large_and_small_rows_behind_the_mask(kernel, lengths, tree, power, what):
    """One token of the new ones, and those behind a sequence's end, hold 2^power times what the others do."""
    seqs, bt, n_pages, T = layout(lengths, 11)
    k, v, q = rows(n_pages, 12, T)
    words, blind = tree(seqs, T, 13) if tree else None, set()
    for n, (start, new, all_, row) in enumerate(seqs):
        odd = all_ - new + (2 * new) // 3
        for t in (odd, *range(all_, (all_ + PAGE - 1) // PAGE * PAGE)):
            at = slot_of(bt, row, t)
            if what != "values":
                k[at] *= 2.0 ** power
            if what != "keys":
                v[at] *= 2.0 ** power
        blind |= {(n, i) for i in range(new) if odd not in visible(seqs[n], i, words)}
    assert len(blind) > len(seqs)
    cache = cache_of(n_pages, N_KV, k, v)
    got = attend(cache, q, seqs, bt, D ** -0.5, kernel, words)
    cache.check()
    assert bool(got.isfinite().all())
    check(cache, q, seqs, bt, D ** -0.5, kernel, words, got=got, only=blind)


@pytest.mark.parametrize("kernel,lengths,tree", CASES)
@pytest.mark.parametrize("first", [True, False])
def test_large_values_without_weight(kernel, lengths, tree, first):
    """Tokens with values of 2^40 whose probability is below 2^-60 count for less than the others' rounding."""
    seqs, bt, n_pages, T = layout(lengths, 21)
    k, v, q = rows(n_pages, 22, T)
    q = q.view(T, N_Q, D).clone()
    q[:, :, 0] = 8.0
    q = q.view(T, -1)
    for start, new, all_, row in seqs:
        old = all_ - new
        for t in (range(0, old // 2) if first else range(old // 2, old)):
            at = slot_of(bt, row, t)
            k[at, :, 0] = -64.0                    # scale * 8 * -64 = -45
            v[at] *= 2.0 ** 40
    check(cache_of(n_pages, N_KV, k, v), q, seqs, bt, D ** -0.5, kernel, tree(seqs, T, 23) if tree else None)


@pytest.mark.parametrize("kernel,lengths,tree", CASES)
@pytest.mark.parametrize("k_spread,v_spread", [(0.0, 3.0), (0.0, 8.0), (3.0, 0.0), (8.0, 0.0), (6.0, 6.0), (0.0, 0.0)])
def test_rows_of_very_different_sizes(kernel, lengths, tree, k_spread, v_spread):
    """Sizes spread over many octaves; the scale is chosen for the largest sum |scale q k| to be 20."""
    seqs, bt, n_pages, T = layout(lengths, 31)
    k, v, q = rows(n_pages, 32, T)
    g = torch.Generator(device="cuda").manual_seed(33)
    size = lambda s: torch.exp(s * torch.randn(n_pages * PAGE, N_KV, 1, device="cuda", generator=g))  # noqa: E731
    k, v = k * size(k_spread), v * size(v_spread)
    largest = (k.abs().amax(0).sum(-1).amax() * q.abs().amax()).item()
    check(cache_of(n_pages, N_KV, k, v), q, seqs, bt, 20.0 / largest, kernel, tree(seqs, T, 34) if tree else None)
