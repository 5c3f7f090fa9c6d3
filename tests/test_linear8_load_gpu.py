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
