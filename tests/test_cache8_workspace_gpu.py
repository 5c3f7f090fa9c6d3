"""One workspace, sized for the widest drafts over the longest contexts, under every smaller call; nothing is written behind it."""
import pytest
import torch

from cache8_checks import D, PAGE, cache_of, check, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_q,n_kv,most_seqs,longest", [(32, 8, 128, 8100), (8, 2, 300, 3000)])
def test_one_workspace_for_all_calls(n_q, n_kv, most_seqs, longest):
    n_pages = (longest + PAGE - 1) // PAGE
    g = torch.Generator(device="cuda").manual_seed(51)
    k, v = torch.randn(2, n_pages * PAGE, n_kv, D, device="cuda", generator=g)
    cache = cache_of(n_pages, n_kv, k, v)
    size = cache.workspace_bytes(most_seqs * 64, most_seqs, n_q, 64, longest)
    room = torch.full((size + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    for n, new in ((1, 1), (most_seqs, 1), (1, 8), (most_seqs, 8), (most_seqs, 12), (most_seqs // 3, 12), (2, 13), (most_seqs, 2), (1, 64)):
        # (sequences share the pages, each has its own length)
        lengths = [longest - (31 * i) % (longest // 2) for i in range(n)]
        seqs, bt = [[i * new, new, kv, 0] for i, kv in enumerate(lengths)], [list(range(n_pages))]
        q = torch.randn(n * new, n_q * D, device="cuda", generator=g).to(torch.bfloat16)
        max_kv = max(lengths)
        assert cache.workspace_bytes(n * new, n, n_q, new, max_kv) <= size
        got = cache.attend(q, ints(seqs), ints(bt), 0.5 * D ** -0.5, new, max_kv, workspace=room[:size])
        assert torch.equal(got, cache.attend(q, ints(seqs), ints(bt), 0.5 * D ** -0.5, new, max_kv))
        cache.check()
        some = {(s, i) for s in {0, n // 2, n - 1} for i in {0, new - 1}}
        check(cache, q, seqs, bt, 0.5 * D ** -0.5, "rows" if new * n_q // n_kv <= 48 else "prompt", got=got, only=some)
        assert bool((room[size:] == 0x5a).all())


def test_bounds_are_not_cut_to_32_bits():
    cache = cache_of(1, 1, *torch.ones(2, PAGE, 1, D, device="cuda"))
    q, seqs, bt = torch.ones(1, D, device="cuda", dtype=torch.bfloat16), ints([[0, 1, 1, 0]]), ints([[0]])
    ws = torch.zeros(64, dtype=torch.uint8, device="cuda")
    for max_q, max_kv in ((1 << 32 | 1, 1), (1, 1 << 32 | 1), (1, 1 << 31), (-1, 1)):
        for workspace in (None, ws):
            with pytest.raises(ValueError, match="31 bits"):
                cache.attend(q, seqs, bt, 1.0, max_q, max_kv, workspace=workspace)
