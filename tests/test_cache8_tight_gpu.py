"""The two attention kernels of the 8-bit cache, each held to its own rounding (cache8_checks): what reads exact keys gets no allowance for rounded ones."""
import pytest
import torch

from cache8_checks import D, PAGE, branches, cache_of, check, layout
from vllm_tgis_adapter_b200.engine.cache8 import Cache8

pytestmark = pytest.mark.gpu


def ordinary(lengths, n_q, n_kv, seed):
    seqs, bt, n_pages, T = layout(lengths, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = torch.randn(2, n_pages * PAGE, n_kv, D, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(2, n_pages * PAGE, n_kv, 1, device="cuda", generator=g))
    return cache_of(n_pages, n_kv, k, v), torch.randn(T, n_q * D, device="cuda", generator=g).to(torch.bfloat16), seqs, bt, T


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (32, 8), (6, 2), (3, 3), (16, 2)])
@pytest.mark.parametrize("tree", [None, branches])
def test_17_to_48_rows_read_exact_keys(n_q, n_kv, tree):
    most = 48 // (n_q // n_kv)
    for lengths in ([(most, 500), (most - 1, 0), (1, 40), (most // 2 + 1, 130)], [(most, 1500), (most - 2, 900), (1, 1200)]):
        cache, q, seqs, bt, T = ordinary(lengths, n_q, n_kv, 41)
        check(cache, q, seqs, bt, 0.4 * D ** -0.5, "rows", tree(seqs, T, 42) if tree else None)


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (32, 8), (3, 3)])
def test_short_prompts_that_run_at_once_read_exact_keys(n_q, n_kv):
    cache, q, seqs, bt, _ = ordinary([(64, 0), (40, 20)], n_q, n_kv, 43)
    check(cache, q, seqs, bt, 0.4 * D ** -0.5, "rows")


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (32, 8), (6, 2), (64, 8), (3, 3)])
@pytest.mark.parametrize("tree", [None, branches])
def test_prompts_and_wide_drafts(n_q, n_kv, tree):
    cache, q, seqs, bt, T = ordinary([(64, 500), (33, 0), (1, 127), (50, 130)], n_q, n_kv, 44)
    check(cache, q, seqs, bt, 0.1 * D ** -0.5, "prompt", tree(seqs, T, 45) if tree else None)


@pytest.mark.parametrize("kernel,lengths", [("rows", [(6, 300), (1, 77), (6, 0)]), ("prompt", [(64, 300), (50, 0), (1, 77)])])
def test_heads_on_two_ranks(kernel, lengths):
    """Half of the heads each, as tensor-parallel ranks hold them: the same stored bytes, and each half right."""
    n_q, n_kv = 16, 4
    cache, q, seqs, bt, T = ordinary(lengths, n_q, n_kv, 46)
    check(cache, q, seqs, bt, 0.03, kernel)
    for r in range(2):
        part = Cache8(cache.pages[:, 2 * r:2 * r + 2].contiguous())
        check(part, q.view(T, n_q, D)[:, 8 * r:8 * r + 8].reshape(T, -1).contiguous(), seqs, bt, 0.03, kernel)


def test_ranks_store_what_one_does():
    n_q, n_kv, T = 8, 4, 90
    g = torch.Generator(device="cuda").manual_seed(47)
    qkv = torch.randn(T, (n_q + 2 * n_kv) * D, device="cuda", generator=g).to(torch.bfloat16)
    cs = torch.randn(100, D, device="cuda", generator=g).to(torch.bfloat16)
    at = torch.arange(T, device="cuda", dtype=torch.int32)
    whole = Cache8.empty(3, n_kv)
    q = whole.write(qkv, at, at, cs).view(T, n_q, D)
    heads = qkv.view(T, -1, D)
    for r in range(2):
        part = Cache8.empty(3, 2)
        mine = torch.cat([heads[:, 4 * r:4 * r + 4], heads[:, n_q + 2 * r:n_q + 2 * r + 2], heads[:, n_q + n_kv + 2 * r:n_q + n_kv + 2 * r + 2]], dim=1)
        assert torch.equal(part.write(mine.reshape(T, -1).contiguous(), at, at, cs).view(T, 4, D), q[:, 4 * r:4 * r + 4])
        assert torch.equal(part.pages, whole.pages[:, 2 * r:2 * r + 2])
