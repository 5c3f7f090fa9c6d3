"""The engine over the 8-bit cache (kv_cache_dtype="fp8"): against the oracle with quantised rows, against itself in other portions and
batches, its capacity.

Tolerances: the envelope of the 16-bit engine against the oracle (mean 2e-3, 95 % 5e-3, largest 1e-2 of a log-probability) comes from
activations that round to the other side in bf16, 2^-8 of a value.  Where such a value is stored, a code is off by its step, 2^-3, with
a probability of 2^-8 / 2^-3: its root mean square grows by the square root of 2^5, 5.7.  So six times that envelope, and near-ties of
six times the margin (0.02) may flip.
"""
import dataclasses

import numpy as np
import pytest
import torch

from oracle.llama_oracle import CONFIGS, LlamaOracle, rope_table, synthetic_weights

pytestmark = pytest.mark.gpu
WIDER = 6.0


class Oracle8(LlamaOracle):
    """Rotation in fp32; keys and values as e4m3 codes times the row's scale."""

    def _rope(self, x, pos):
        half = self.cfg.head_dim // 2
        cs = self.cos_sin[pos].float()
        cos, sin = cs[:, None, :half], cs[:, None, half:]
        x1, x2 = x[..., :half].float(), x[..., half:].float()
        return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)

    def _attend(self, q, k, v, first_pos):
        def rows(x):
            x = x.float()
            s = (x.abs().amax(-1, keepdim=True) * torch.tensor(1.0 / 448.0)).clamp(min=2.0 ** -126)
            return (x / s).to(torch.float8_e4m3fn).float() * s

        return super()._attend(q.to(self.dtype), rows(k), rows(v), first_pos)


def engine(cfg_name, weights, **kw):
    from vllm_tgis_adapter_b200.engine.core import ModelConfig, NativeEngine

    cfg = CONFIGS[cfg_name]
    names = {f.name for f in dataclasses.fields(ModelConfig)}
    mc = ModelConfig(**{f.name: getattr(cfg, f.name) for f in dataclasses.fields(cfg) if f.name in names})
    kw = {"max_num_seqs": 8, "max_batched_tokens": 2048, "kv_cache_bytes": 64 << 20, "kv_cache_dtype": "fp8", **kw}
    eng = NativeEngine(mc, **kw)
    eng.load_weights(weights)
    eng.load_weight("tgis.rope_cos_sin", rope_table(cfg))
    return eng


def generate(cfg_name, weights, prompts, n_new, **kw):
    from vllm_tgis_adapter_b200.engine.core import make_sampling_params

    eng = engine(cfg_name, weights, **kw)
    sp = make_sampling_params(greedy=True, max_tokens=n_new, min_tokens=n_new, num_logprobs=1, eos_token_id=2)
    outs = eng.generate_sync(prompts, sp)
    st = eng.status()
    eng.close()
    assert st.errored == 0
    return [[r for r in recs if r.new_token is not None] for recs in outs], st


@pytest.mark.parametrize("cfg_name,chunk,graphs", [("tiny", 2048, True), ("tiny", 48, False), ("small", 256, True)])
def test_greedy_generation_matches_the_oracle_with_quantised_rows(cfg_name, chunk, graphs):
    cfg = CONFIGS[cfg_name]
    weights = synthetic_weights(cfg, seed=1)
    rng = np.random.RandomState(0)
    prompts = [rng.randint(3, cfg.vocab, size=n).tolist() for n in (5, 33, 64, 100, 17, 250)]
    n_new, flips, diffs, ora = 24, 0, [], Oracle8(cfg, weights)
    outs, st = generate(cfg_name, weights, prompts, n_new, max_batched_tokens=chunk, use_cuda_graphs=graphs)
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


def test_prompts_in_portions_and_alone():
    """The logits of given tokens: whole, in portions, among others, beside single tokens."""
    cfg = CONFIGS["small"]
    weights = synthetic_weights(cfg, seed=3)
    rng = np.random.RandomState(4)
    a, b = rng.randint(3, cfg.vocab, size=300).tolist(), rng.randint(3, cfg.vocab, size=77).tolist()
    eng = engine("small", weights)
    whole = eng.trace_step([("w", a, [150, 299])], end=["w"])
    eng.trace_step([("p", a[:37], []), ("q", b[:76], [])])
    mixed = [eng.trace_step([("p", a[37:151], [113]), ("q", b[76:], [0])])[0]]   # a portion beside a single token
    eng.trace_step([("p", a[151:152], [])])
    eng.trace_step([("p", a[152:299], [])])
    mixed.append(eng.trace_step([("p", a[299:], [0])], end=["p", "q"])[0])
    alone = eng.trace_step([("b", b, [76])], end=["b"])
    eng.close()
    ora = Oracle8(cfg, weights)
    want = ora.step([(ora.new_seq(), a)], want_all_logits=True)[[150, 299]].numpy()
    spread = float(np.abs(want).std())
    for got in (whole, np.stack(mixed)):
        assert np.abs(got - want).mean() < 2e-3 * WIDER * max(spread, 1) and np.abs(got - want).max() < 2e-2 * WIDER * max(spread, 1)
    want_b = ora.step([(ora.new_seq(), b)])[0].numpy()
    assert np.abs(alone[0] - want_b).max() < 2e-2 * WIDER * max(spread, 1)


def test_capacity_and_difference_from_the_16_bit_cache():
    cfg = CONFIGS["tiny"]
    weights = synthetic_weights(cfg, seed=1)
    prompts = [np.random.RandomState(2).randint(3, cfg.vocab, size=n).tolist() for n in (40, 90)]
    bytes_ = 40 * 2 * cfg.n_layers * cfg.n_kv_heads * 32 * 128 * 2   # forty blocks of the 16-bit cache
    eight, st8 = generate("tiny", weights, prompts, 8, kv_cache_bytes=bytes_)
    sixteen, st16 = generate("tiny", weights, prompts, 8, kv_cache_bytes=bytes_, kv_cache_dtype="auto")
    assert st16.total_blocks == 40 and st8.total_blocks == 40 * 16384 // 8448
    first = [(a[0].logprob, b[0].logprob) for a, b in zip(eight, sixteen)]
    assert any(x != y for x, y in first) and all(abs(x - y) < 0.3 for x, y in first)


def test_cache_pressure_preempts_and_recovers():
    """More sequences than the cache holds: what is evicted is computed again, and the results are those of a roomy cache."""
    cfg = CONFIGS["tiny"]
    weights = synthetic_weights(cfg, seed=1)
    prompts = [np.random.RandomState(5 + i).randint(3, cfg.vocab, size=60).tolist() for i in range(6)]
    block = cfg.n_layers * cfg.n_kv_heads * 8448
    roomy, _ = generate("tiny", weights, prompts, 40, max_num_seqs=6)
    tight, st = generate("tiny", weights, prompts, 40, max_num_seqs=6, kv_cache_bytes=18 * block)
    assert st.preemptions > 0
    same = sum(a.new_token == b.new_token for x, y in zip(roomy, tight) for a, b in zip(x, y))
    assert same >= 0.9 * 6 * 40   # (sums in another order may flip a near-tie, and what follows it)
