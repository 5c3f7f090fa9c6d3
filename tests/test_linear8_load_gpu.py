"""Weights on their way into 8 bits: which device they are made on, and the place that they pass through."""
import dataclasses
import threading

import numpy as np
import pytest
import torch

from oracle.llama_oracle import CONFIGS, rope_table, synthetic_weights
from test_linear8_engine_gpu import WIDER, OracleW8, engine

pytestmark = pytest.mark.gpu
NAME = "model.layers.0.mlp.down_proj.weight"


def config_of(eng):
    """The engine's own record, which it begins with."""
    from vllm_tgis_adapter_b200.engine import _lib

    cfg = _lib.TgisConfig.from_address(eng._h.value)
    assert cfg.abi_version == _lib.ABI_VERSION and (cfg.hidden, cfg.device) == (eng.model.hidden, 0)
    return cfg


@pytest.mark.parametrize("quantization", [None, "fp8"])
def test_weights_are_loaded_on_the_engines_device(quantization):
    """An engine whose device is not the thread's current one: here one that there is not, which has to be noticed before anything is launched."""
    from vllm_tgis_adapter_b200.engine.core import EngineError

    weights = synthetic_weights(CONFIGS["tiny"], seed=1)
    eng = engine("tiny", weights, quantization=quantization)
    cfg = config_of(eng)
    cfg.device = torch.cuda.device_count()
    try:
        with pytest.raises(EngineError, match="device"):
            eng.load_weight(NAME, weights[NAME])
    finally:
        cfg.device = 0
    assert torch.cuda.current_device() == 0
    eng.load_weight(NAME, weights[NAME])
    assert len(eng.trace_step([("a", [5, 6, 7], [2])], end=["a"])) == 1
    eng.close()


def test_weights_of_a_layer_list_are_loaded_on_the_engines_device():
    from vllm_tgis_adapter_b200.engine import ponenex
    from vllm_tgis_adapter_b200.engine.core import EngineError, NativeEngine, cache_block_bytes

    mc = ponenex.PRESETS["ponenex-tiny"]
    weights = ponenex.synthetic_weights(mc, seed=5)
    eng = NativeEngine(mc, max_num_seqs=2, max_batched_tokens=64, kv_cache_bytes=cache_block_bytes(mc) * 8)
    eng.load_weights(weights)
    cfg = config_of(eng)
    cfg.device = torch.cuda.device_count()
    try:
        with pytest.raises(EngineError, match="device"):
            eng.load_weight("head", weights["head"])
    finally:
        cfg.device = 0
    eng.load_weight("head", weights["head"])
    eng.close()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two GPUs")
def test_another_thread_loads_for_an_engine_on_another_device():
    weights = synthetic_weights(CONFIGS["tiny"], seed=1)
    got = []
    for device in (0, 1):
        torch.cuda.set_device(0)
        eng = engine("tiny", {}, device=device)
        seen = []

        def load():
            torch.cuda.set_device(0)
            eng.load_weights(weights)
            eng.load_weight("tgis.rope_cos_sin", rope_table(CONFIGS["tiny"]))
            seen.append(torch.cuda.current_device())

        thread = threading.Thread(target=load)
        thread.start()
        thread.join()
        assert seen == [0]
        torch.cuda.set_device(device)
        got.append(eng.trace_step([("a", [5, 6, 7], [2])], end=["a"]))
        eng.close()
    torch.cuda.set_device(0)
    assert np.array_equal(*got)


def test_tensors_that_come_in_pieces():
    """Matrices of more numbers than are on their way at a time: rows of 2 048 and of 11 264 numbers."""
    cfg = dataclasses.replace(CONFIGS["small"], hidden=2048, n_q_heads=16, n_kv_heads=4, ffn=11264, n_layers=1)
    assert cfg.hidden * cfg.ffn > 2 * (8 << 20)
    CONFIGS["pieces"] = cfg
    try:
        weights = synthetic_weights(cfg, seed=2)
        eng = engine("pieces", weights)
    finally:
        del CONFIGS["pieces"]
    tokens = np.random.RandomState(1).randint(3, cfg.vocab, size=40).tolist()
    got = eng.trace_step([("a", tokens, [10, 39])], end=["a"])
    eng.close()
    ora = OracleW8(cfg, weights)
    want = ora.step([(ora.new_seq(), tokens)], want_all_logits=True)[[10, 39]].numpy()
    spread = max(float(np.abs(want).std()), 1)
    assert np.abs(got - want).mean() < 2e-3 * WIDER * spread and np.abs(got - want).max() < 2e-2 * WIDER * spread


def test_nothing_is_held_that_only_loading_needs():
    """What an engine takes, when it is made and once it runs, beside the same one with 16-bit weights."""
    from vllm_tgis_adapter_b200.engine.core import ModelConfig, NativeEngine, make_sampling_params

    cfg = dataclasses.replace(CONFIGS["llama3-8b"], n_layers=2, vocab=1024)
    names = {f.name for f in dataclasses.fields(ModelConfig)}
    mc = ModelConfig(**{f.name: getattr(cfg, f.name) for f in dataclasses.fields(cfg) if f.name in names})
    H, F, kv, T = cfg.hidden, cfg.ffn, cfg.n_kv_heads * cfg.head_dim, 256
    shapes = {"self_attn.q_proj": (H, H), "self_attn.k_proj": (kv, H), "self_attn.v_proj": (kv, H), "self_attn.o_proj": (H, H), "mlp.gate_proj": (F, H), "mlp.up_proj": (F, H),
              "mlp.down_proj": (H, F)}
    zeros = torch.zeros(H * F, dtype=torch.bfloat16)

    def free():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]

    made, running = {}, {}
    for quantization in (None, "fp8", None, "fp8"):   # (the first two load the kernels)
        before = free()
        eng = NativeEngine(mc, max_num_seqs=4, max_batched_tokens=T, kv_cache_bytes=256 << 20, quantization=quantization, use_cuda_graphs=False)
        made[quantization] = before - free()
        for layer in range(cfg.n_layers):
            for name, (n, k) in shapes.items():
                eng.load_weight(f"model.layers.{layer}.{name}.weight", zeros[: n * k].view(n, k))
            for name in ("input_layernorm", "post_attention_layernorm"):
                eng.load_weight(f"model.layers.{layer}.{name}.weight", torch.ones(H))
        eng.load_weight("model.embed_tokens.weight", zeros[: cfg.vocab * H].view(cfg.vocab, H))
        eng.load_weight("model.norm.weight", torch.ones(H))
        eng.load_weight("tgis.rope_cos_sin", rope_table(cfg))
        eng.generate_sync([[5, 6, 7]], make_sampling_params(greedy=True, max_tokens=3, min_tokens=3))
        running[quantization] = before - free()
        eng.close()
    numbers = cfg.n_layers * sum(n * k for n, k in shapes.values())
    rows = T * (H + F) * (1 + 4 / 128)
    saved = numbers * (2 - 1 - 4 / 128 ** 2) - rows
    room = 24 << 20   # (allocations are rounded up; a tensor on its way would be 117 MB)
    assert abs(made[None] - made["fp8"] - saved) < room, (made, saved)
    assert abs(running[None] - running["fp8"] - saved) < room, (running, saved)
