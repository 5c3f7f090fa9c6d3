"""Attention over the 8-bit cache where scores are zeros: queries, keys or both so small that units of the products pass fp32's smallest number.

Every probability of a row is then the same to 2^-40, so the answer is the mean of the values that it sees, in both kernels, under every mask.
"""
import numpy as np
import pytest
import torch

from cache8_checks import D, PAGE, branches, cache_of, check, layout

pytestmark = pytest.mark.gpu

SHORT = [(1, 0), (2, 0), (7, 26), (12, 300), (1, 127), (3, 128), (12, 116)]
LONG = [(1, 0), (33, 0), (64, 31), (64, 64), (63, 237), (1, 299), (64, 128), (5, 124)]


@pytest.mark.parametrize("kernel,lengths", [("rows", SHORT), ("prompt", SHORT), ("prompt", LONG), ("prompt", [(300, 0), (129, 171)])])
@pytest.mark.parametrize("tree", [None, branches])
@pytest.mark.parametrize("q_size,k_size", [(0.0, 0.0), (0.0, 1e-4), (1e-6, 0.0), (1e-30, 0.0), (0.0, 1.0), (1.0, 0.0), (1e-38, 1e-36)])
def test_scores_of_nothing(kernel, lengths, tree, q_size, k_size):
    if tree and max(n for n, _ in lengths) > 64:
        pytest.skip("a draft has 64 nodes at most")
    n_q, n_kv = 8, 2
    seqs, bt, n_pages, T = layout(lengths, 3)
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = torch.randn(2, n_pages * PAGE, n_kv, D, device="cuda", generator=g)
    q = (torch.randn(T, n_q * D, device="cuda", generator=g) * q_size).to(torch.bfloat16)
    cache = cache_of(n_pages, n_kv, k * k_size, v)
    for scale in (D ** -0.5, 0.0, -1e-3):
        check(cache, q, seqs, bt, scale, kernel, tree(seqs, T, 5) if tree else None)


def test_a_prompt_with_a_run_of_tokens_without_an_embedding():
    """300 tokens whose embedding is zero (queries, keys and values of nothing), others before and behind them."""
    from oracle.llama_oracle import CONFIGS, synthetic_weights
    from test_cache8_engine_gpu import WIDER, Oracle8, engine

    cfg = CONFIGS["tiny"]
    weights = synthetic_weights(cfg, seed=1)
    weights["model.embed_tokens.weight"][7] = 0
    rng = np.random.RandomState(3)
    prompts = [[7] * 300 + rng.randint(8, cfg.vocab, size=40).tolist(), rng.randint(8, cfg.vocab, size=9).tolist() + [7] * 300 + [11, 12]]
    eng = engine("tiny", weights)
    for i, p in enumerate(prompts):
        rows = [5, len(p) - 3, len(p) - 1]
        got = eng.trace_step([(f"p{i}", p, rows)], end=[f"p{i}"])
        ora = Oracle8(cfg, weights)
        want = ora.step([(ora.new_seq(), p)], want_all_logits=True)[rows].numpy()
        spread = max(float(np.abs(want).std()), 1.0)
        assert np.isfinite(got).all() and np.abs(got - want).max() < 2e-2 * WIDER * spread
    eng.close()
