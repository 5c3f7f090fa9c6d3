"""The engine over 8-bit weights (quantization="fp8"): against the oracle with rows and weights quantised, against itself in other portions and
batches, over the 8-bit cache, its memory and refusals.

Tolerances: the envelope of the 16-bit engine against the oracle (mean 2e-3, 95 % 5e-3, largest 1e-2 of a log-probability) comes from activations
that round to the other side in bf16, 2^-8 of a value.  Where such a value becomes a code, the code is off by its step, 2^-3, with a probability of
2^-8 / 2^-3: its root mean square grows by the square root of 2^5, 5.7; four projections a layer read such rows where the 8-bit cache has
two such tensors, so the sum of their squares is twice that one's: eight times the envelope, and near-ties of eight times the margin (0.02) may flip.
"""
import dataclasses

import numpy as np
import pytest
import torch

from oracle.llama_oracle import CONFIGS, LlamaOracle, rope_table, synthetic_weights

pytestmark = pytest.mark.gpu
WIDER = 8.0


def quantised(v, rows):
    """fp32 -> what its groups of `rows` x 128 stand for, and the scales"""
    r, k = v.shape
    p = torch.nn.functional.pad(v, (0, -k % 128, 0, -r % rows))
    p = p.view(p.shape[0] // rows, rows, -1, 128)
    s = (p.abs().amax(dim=(1, 3), keepdim=True) * torch.tensor(1.0 / 448.0)).clamp(min=2.0 ** -126)
    return ((p / s).to(torch.float8_e4m3fn).float() * s).reshape(p.shape[0] * rows, -1)[:r, :k]


class OracleW8(LlamaOracle):
    def __init__(self, cfg, weights):
        super().__init__(cfg, weights)
        for layer in self.layers:
            for name in ("qkv", "o", "gu", "d"):   # (heads and feed-forward sizes are multiples of 128: blocks do not cross)
                layer[name] = quantised(layer[name].float(), 128)

    def _norm_rows(self, r, w):
        f = r.float()
        return quantised(f * w.float(), 1) * torch.rsqrt(f.square().mean(-1, keepdim=True) + self.cfg.rms_eps)

    @torch.no_grad()
    def step(self, work, want_all_logits=False):
        cfg = self.cfg
        toks = torch.tensor([t for _, ts in work for t in ts])
        pos = torch.tensor([st.n + j for st, ts in work for j in range(len(ts))])
        resid, x, T = self.embed[toks], None, len(toks)
        for li, L in enumerate(self.layers):
            resid = resid if li == 0 else x + resid
            qkv = (self._norm_rows(resid, L["ln1"]) @ L["qkv"].t()).to(self.dtype)
            q, k, v = (y.reshape(T, -1, cfg.head_dim) for y in qkv.split([cfg.q_dim, cfg.kv_dim, cfg.kv_dim], dim=1))
            q, k = self._rope(q, pos), self._rope(k, pos)
            outs, off = [], 0
            for st, ts in work:
                st.k[li], st.v[li] = torch.cat([st.k[li], k[off:off + len(ts)]]), torch.cat([st.v[li], v[off:off + len(ts)]])
                outs.append(self._attend(q[off:off + len(ts)], st.k[li], st.v[li], st.n))
                off += len(ts)
            x = (quantised(torch.cat(outs).reshape(T, cfg.q_dim).float(), 1) @ L["o"].t()).to(self.dtype)
            resid = x + resid
            g, u = (self._norm_rows(resid, L["ln2"]) @ L["gu"].t()).split(cfg.ffn, dim=1)
            x = (quantised(g / (1 + torch.exp(-g)) * u, 1) @ L["d"].t()).to(self.dtype)
        xn = self._rms(x + resid, self.norm)
        for st, ts in work:
            st.n += len(ts)
        if not want_all_logits:
            xn = xn[torch.tensor([len(ts) for _, ts in work]).cumsum(0) - 1]
        return self.head(xn, normed=True)


def engine(cfg_name, weights, **kw):
    from vllm_tgis_adapter_b200.engine.core import ModelConfig, NativeEngine

    cfg = CONFIGS[cfg_name]
    names = {f.name for f in dataclasses.fields(ModelConfig)}
    mc = ModelConfig(**{f.name: getattr(cfg, f.name) for f in dataclasses.fields(cfg) if f.name in names})
    kw = {"max_num_seqs": 8, "max_batched_tokens": 2048, "kv_cache_bytes": 64 << 20, "quantization": "fp8", **kw}
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
def test_greedy_generation_matches_the_quantised_oracle(cfg_name, chunk, graphs):
    cfg = CONFIGS[cfg_name]
    weights = synthetic_weights(cfg, seed=1)
    rng = np.random.RandomState(0)
    prompts = [rng.randint(3, cfg.vocab, size=n).tolist() for n in (5, 33, 64, 100, 17, 250)]
    n_new, flips, diffs, ora = 24, 0, [], OracleW8(cfg, weights)
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


@pytest.mark.parametrize("cache", ["auto", "fp8"])
def test_prompts_in_portions_and_alone(cache):
    """The logits of given tokens: whole (on the prompts' kernel), in portions, among others, beside single tokens."""
    cfg = CONFIGS["small"]
    weights = synthetic_weights(cfg, seed=3)
    rng = np.random.RandomState(4)
    a, b = rng.randint(3, cfg.vocab, size=300).tolist(), rng.randint(3, cfg.vocab, size=77).tolist()
    eng = engine("small", weights, kv_cache_dtype=cache)
    whole = eng.trace_step([("w", a, [150, 299])], end=["w"])
    eng.trace_step([("p", a[:37], []), ("q", b[:76], [])])
    mixed = [eng.trace_step([("p", a[37:151], [113]), ("q", b[76:], [0])])[0]]
    eng.trace_step([("p", a[151:152], [])])
    eng.trace_step([("p", a[152:299], [])])
    mixed.append(eng.trace_step([("p", a[299:], [0])], end=["p", "q"])[0])
    alone = eng.trace_step([("b", b, [76])], end=["b"])
    eng.close()
    ora = OracleW8(cfg, weights)
    wider = WIDER * (1.5 if cache == "fp8" else 1)   # (two more tensors of codes a layer: the square root of 6 / 4, and the cache's own rounding, not the oracle's)
    want = ora.step([(ora.new_seq(), a)], want_all_logits=True)[[150, 299]].numpy()
    spread = max(float(np.abs(want).std()), 1)
    if cache == "auto":
        for got in (whole, np.stack(mixed)):
            assert np.abs(got - want).mean() < 2e-3 * wider * spread and np.abs(got - want).max() < 2e-2 * wider * spread
        want_b = ora.step([(ora.new_seq(), b)])[0].numpy()
        assert np.abs(alone[0] - want_b).max() < 2e-2 * wider * spread
    assert np.abs(whole - np.stack(mixed)).mean() < 2e-3 * wider * spread and np.abs(whole - np.stack(mixed)).max() < 2e-2 * wider * spread


def test_weights_take_half_the_memory_and_the_results_differ():
    cfg = CONFIGS["small"]
    weights = synthetic_weights(cfg, seed=1)
    prompts = [np.random.RandomState(2).randint(3, cfg.vocab, size=n).tolist() for n in (40, 90)]
    eight, _ = generate("small", weights, prompts, 8)
    sixteen, _ = generate("small", weights, prompts, 8, quantization=None)
    first = [(a[0].logprob, b[0].logprob) for a, b in zip(eight, sixteen)]
    assert any(x != y for x, y in first) and all(abs(x - y) < 0.5 for x, y in first)
    big = dataclasses.replace(CONFIGS["llama3-8b"], n_layers=4, vocab=1024)
    used = {}
    for quantization in (None, "fp8"):
        from vllm_tgis_adapter_b200.engine.core import ModelConfig, NativeEngine

        names = {f.name for f in dataclasses.fields(ModelConfig)}
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        eng = NativeEngine(ModelConfig(**{f.name: getattr(big, f.name) for f in dataclasses.fields(big) if f.name in names}), max_num_seqs=4, max_batched_tokens=256,
                           kv_cache_bytes=256 << 20, quantization=quantization)
        used[quantization] = before - torch.cuda.mem_get_info()[0]
        eng.close()
    per_layer = 4096 * (6144 + 4096 + 3 * 14336)
    assert used[None] - used["fp8"] > 4 * per_layer * 0.8   # (2 - 1 byte a number, less a tensor's place on its way and the rows)


def test_scores_of_prompts_and_sampling_run():
    """Prompt log-probabilities and sampled requests over 8-bit weights."""
    from vllm_tgis_adapter_b200.engine.core import make_sampling_params

    cfg = CONFIGS["tiny"]
    weights = synthetic_weights(cfg, seed=1)
    prompt = np.random.RandomState(3).randint(3, cfg.vocab, size=60).tolist()
    eng = engine("tiny", weights)
    recs = eng.generate_sync([prompt], make_sampling_params(greedy=True, max_tokens=2, num_logprobs=1, prompt_logprobs=1, eos_token_id=2))[0]
    scored = [r for r in recs if r.new_token is None]
    ora = OracleW8(cfg, weights)
    want = torch.log_softmax(ora.step([(ora.new_seq(), prompt)], want_all_logits=True), -1)
    assert len(scored) == 59
    diffs = np.array([abs(r.logprob - float(want[r.prompt_pos - 1, prompt[r.prompt_pos]])) for r in scored])
    assert diffs.mean() < 2e-3 * WIDER and diffs.max() < 1e-2 * WIDER
    sampled = eng.generate_sync([prompt], make_sampling_params(greedy=False, temperature=0.9, top_k=20, seed=7, max_tokens=12, min_tokens=12))[0]
    assert len([r for r in sampled if r.new_token is not None]) == 12
    assert eng.status().errored == 0
    eng.close()


def test_profiling_counts_the_products():
    """Four a layer and the head's, as over 16-bit weights, and of the projections' bytes about half."""
    from vllm_tgis_adapter_b200.engine.core import make_sampling_params

    cfg = CONFIGS["small"]
    weights = synthetic_weights(cfg, seed=1)
    prompt = np.random.RandomState(5).randint(3, cfg.vocab, size=40).tolist()
    calls, moved = {}, {}
    for quantization in (None, "fp8"):
        eng = engine("small", weights, quantization=quantization)
        eng.set_profiling(1)
        eng.generate_sync([prompt], make_sampling_params(greedy=True, max_tokens=6, min_tokens=6, eos_token_id=2))
        eng.set_profiling(False)
        st = eng.status()
        calls[quantization], moved[quantization] = st.gemm_calls / st.steps, st.gemm_bytes
        assert st.errored == 0 and st.gemm_ms > 0
        eng.close()
    assert calls["fp8"] == calls[None] == 4 * cfg.n_layers + 1
    assert moved["fp8"] < moved[None]
