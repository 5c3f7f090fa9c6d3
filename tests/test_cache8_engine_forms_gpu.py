"""The engine over the 8-bit cache in the forms that the first tests leave out: contexts whose single tokens are split and joined inside a captured
step, and adapters.  Tolerances: those of test_cache8_engine_gpu (WIDER times the 16-bit envelope); with adapters WIDER times that of test_lora_gpu."""
import numpy as np
import pytest
import torch

from oracle.llama_oracle import CONFIGS, synthetic_weights
from test_cache8_engine_gpu import WIDER, Oracle8, engine, generate

pytestmark = pytest.mark.gpu


def follow(ora, prompt, records, near, lora=None):
    """Differences of log-probabilities and flips at near-ties, the oracle following the engine's tokens."""
    diffs, flips, state = [], 0, ora.new_seq()
    logits = ora.step([(state, prompt)], lora=[lora])[0]
    for token, logprob in records:
        lp, top2 = torch.log_softmax(logits, -1), torch.topk(logits, 2).values
        diffs.append(abs(logprob - float(lp[token])))
        if token != int(torch.argmax(logits)):
            assert float(top2[0] - top2[1]) < near
            flips += 1
        logits = ora.step([(state, [token])], lora=[lora])[0]
    return diffs, flips


@pytest.mark.parametrize("lengths", [(900, 10, 760, 801), (950,)])
def test_contexts_that_are_split(lengths):
    cfg = CONFIGS["small"]
    weights = synthetic_weights(cfg, seed=1)
    rng = np.random.RandomState(11)
    prompts = [rng.randint(3, cfg.vocab, size=n).tolist() for n in lengths]
    outs, st = generate("small", weights, prompts, 24, max_batched_tokens=512)
    assert st.graph_launches > 0
    ora, diffs, flips = Oracle8(cfg, weights), [], 0
    for p, recs in zip(prompts, outs):
        d, f = follow(ora, p, [(r.new_token, r.logprob) for r in recs], 0.02 * WIDER)
        diffs += d
        flips += f
    diffs = np.array(diffs)
    assert flips <= WIDER * len(diffs) / 25
    assert diffs.mean() < 2e-3 * WIDER and np.percentile(diffs, 95) < 5e-3 * WIDER and diffs.max() < 1e-2 * WIDER, (diffs.mean(), np.percentile(diffs, 95), diffs.max())


def test_adapters(tmp_path):
    from test_lora_gpu import _peft_for, _run

    from vllm_tgis_adapter_b200.engine.lora import read_adapter

    cfg = CONFIGS["tiny"]
    weights = synthetic_weights(cfg, seed=1)
    adapters = {}
    for slot, kw in ((1, dict(r=8, alpha=16, seed=1)), (2, dict(r=16, alpha=16, seed=2, modules=("q_proj", "v_proj", "down_proj")))):
        adapters[slot] = read_adapter(str(_peft_for(cfg, tmp_path, f"a{slot}", **kw)), n_layers=cfg.n_layers, max_rank=16)[1]
    rng = np.random.RandomState(7)
    prompts, slots, n_new = [rng.randint(3, cfg.vocab, size=n).tolist() for n in (5, 33, 64, 100, 17)], [1, 1, 2, 0, 0], 16
    eng = engine("tiny", weights, max_loras=2, max_lora_rank=16, max_batched_tokens=128)
    for slot, adapter in adapters.items():
        eng.load_adapter(slot, adapter)
    outs = _run(eng, prompts, slots, n_new)
    plain = _run(eng, prompts, [0] * len(prompts), n_new)
    assert eng.status().errored == 0
    eng.close()
    assert outs[0] != plain[0] and outs[2] != plain[2]
    ora, diffs, flips = Oracle8(cfg, weights), [], 0
    for p, recs, slot in zip(prompts, outs, slots):
        d, f = follow(ora, p, recs, 0.03 * WIDER, adapters.get(slot))
        diffs += d
        flips += f
    assert flips <= WIDER * len(diffs) / 25 and np.mean(diffs) < 6e-3 * WIDER and np.max(diffs) < 4e-2 * WIDER, (flips, np.mean(diffs), np.max(diffs))
