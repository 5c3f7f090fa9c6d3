"""The engine over 8-bit weights and the 8-bit cache together, against the oracle that quantises rows, weights, keys and values.

Tolerances: those of test_linear8_engine_gpu.py (eight times the 16-bit engine's envelope, for four projections a layer that read rows in 8 bits), times the square
root of 6 / 4 for two more such tensors, keys and values: ten times, 9.8.
"""
import numpy as np
import pytest
import torch

from oracle.llama_oracle import CONFIGS, synthetic_weights
from test_cache8_engine_gpu import Oracle8
from test_linear8_engine_gpu import OracleW8, engine, generate

pytestmark = pytest.mark.gpu
WIDER = 10.0


class OracleBoth(OracleW8, Oracle8):
    """Steps of the former, rotation and rows of the latter."""


@pytest.mark.parametrize("cfg_name,chunk,graphs", [("tiny", 2048, True), ("tiny", 48, False), ("small", 256, True)])
def test_greedy_generation(cfg_name, chunk, graphs):
    cfg = CONFIGS[cfg_name]
    weights = synthetic_weights(cfg, seed=1)
    rng = np.random.RandomState(0)
    prompts = [rng.randint(3, cfg.vocab, size=n).tolist() for n in (5, 33, 64, 100, 17, 250)]
    n_new, flips, diffs, ora = 24, 0, [], OracleBoth(cfg, weights)
    outs, st = generate(cfg_name, weights, prompts, n_new, max_batched_tokens=chunk, use_cuda_graphs=graphs, kv_cache_dtype="fp8")
    assert (st.graph_launches > 0) == graphs
    for p, recs in zip(prompts, outs):
        assert len(recs) == n_new
        state = ora.new_seq()
        logits = ora.step([(state, p)])[0]
        for r in recs:
            lp, top2 = torch.log_softmax(logits, -1), torch.topk(logits, 2).values
            diffs.append(abs(r.logprob - float(lp[r.new_token])))
            if r.new_token != int(torch.argmax(logits)):
                assert float(top2[0] - top2[1]) < 0.02 * WIDER
                flips += 1
            logits = ora.step([(state, [r.new_token])])[0]
    diffs = np.array(diffs)
    assert flips <= WIDER * len(diffs) / 25
    assert diffs.mean() < 2e-3 * WIDER and np.percentile(diffs, 95) < 5e-3 * WIDER and diffs.max() < 1e-2 * WIDER, (diffs.mean(), np.percentile(diffs, 95), diffs.max())


def test_prompts_in_portions():
    cfg = CONFIGS["small"]
    weights = synthetic_weights(cfg, seed=3)
    rng = np.random.RandomState(4)
    a, b = rng.randint(3, cfg.vocab, size=300).tolist(), rng.randint(3, cfg.vocab, size=77).tolist()
    eng = engine("small", weights, kv_cache_dtype="fp8")
    whole = eng.trace_step([("w", a, [150, 299])], end=["w"])
    eng.trace_step([("p", a[:37], []), ("q", b[:76], [])])
    mixed = [eng.trace_step([("p", a[37:151], [113]), ("q", b[76:], [0])])[0]]
    eng.trace_step([("p", a[151:299], [])])
    mixed.append(eng.trace_step([("p", a[299:], [0])], end=["p", "q"])[0])
    eng.close()
    ora = OracleBoth(cfg, weights)
    want = ora.step([(ora.new_seq(), a)], want_all_logits=True)[[150, 299]].numpy()
    spread = max(float(np.abs(want).std()), 1)
    for got in (whole, np.stack(mixed)):
        assert np.abs(got - want).mean() < 2e-3 * WIDER * spread and np.abs(got - want).max() < 2e-2 * WIDER * spread
