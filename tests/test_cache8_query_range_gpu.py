"""Attention over the 8-bit cache: numbers of a query far below the largest of its row count where the keys have nothing for that one."""
import pytest
import torch

from cache8_checks import D, PAGE, branches, cache_of, check, layout

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,lengths", [("rows", [(12, 300), (1, 40), (12, 0)]), ("prompt", [(64, 100), (40, 0), (1, 77)])])
@pytest.mark.parametrize("tree", [None, branches])
@pytest.mark.parametrize("power", [0, 20, 28, 30])
def test_small_numbers_of_a_query(kernel, lengths, tree, power):
    n_q, n_kv = 8, 2
    seqs, bt, n_pages, T = layout(lengths, 61)
    g = torch.Generator(device="cuda").manual_seed(62)
    k, v = torch.randn(2, n_pages * PAGE, n_kv, D, device="cuda", generator=g)
    q = torch.randn(T, n_q, D, device="cuda", generator=g)
    k[..., 5] = 0
    q[..., 5] = 2.0 ** power
    check(cache_of(n_pages, n_kv, k, v), q.to(torch.bfloat16).view(T, -1), seqs, bt, D ** -0.5, kernel, tree(seqs, T, 63) if tree else None)


@pytest.mark.parametrize("kernel,lengths", [("rows", [(12, 300), (1, 40), (12, 0)]), ("prompt", [(64, 100), (40, 0), (1, 77)])])
@pytest.mark.parametrize("power", [60, 100, 120])
def test_large_queries_and_keys_that_have_nothing_in_common(kernel, lengths, power):
    """Every score is zero, though the units of queries and keys together pass fp32's largest number."""
    n_q, n_kv = 8, 2
    seqs, bt, n_pages, T = layout(lengths, 64)
    g = torch.Generator(device="cuda").manual_seed(65)
    v = torch.randn(n_pages * PAGE, n_kv, D, device="cuda", generator=g)
    k, q = torch.zeros_like(v), torch.zeros(T, n_q, D, device="cuda")
    k[..., 6] = 2.0 ** power
    q[..., 5] = 2.0 ** power
    check(cache_of(n_pages, n_kv, k, v), q.to(torch.bfloat16).view(T, -1), seqs, bt, D ** -0.5, kernel)
