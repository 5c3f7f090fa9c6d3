"""A wait that runs out in a product over 8-bit weights makes the engine's step fail.  The word that such a product raises is raised on the host, at a chosen launch."""
import numpy as np
import pytest

from oracle.llama_oracle import CONFIGS, synthetic_weights
from test_linear8_engine_gpu import engine

pytestmark = pytest.mark.gpu


@pytest.fixture
def lib():
    from vllm_tgis_adapter_b200.engine._lib import load_library

    lib = load_library()
    lib.tgis_k_pair_fault(0)
    yield lib
    lib.tgis_k_pair_fault(0)


@pytest.mark.parametrize("tokens", [3, 200])
@pytest.mark.parametrize("nth", [1, 5, 8])
def test_a_step_fails(lib, nth, tokens):
    from vllm_tgis_adapter_b200.engine.core import EngineError

    weights = synthetic_weights(CONFIGS["tiny"], seed=1)
    eng, work = engine("tiny", weights), [("a", list(range(5, 5 + tokens)), [tokens - 1])]
    lib.tgis_k_pair_fault(0)
    good = eng.trace_step(work, end=["a"])
    assert lib.tgis_k_pair_fault(nth) >= 4 * CONFIGS["tiny"].n_layers   # every product of the layers is one of them
    with pytest.raises(EngineError, match="wait ran out"):
        eng.trace_step(work, end=["a"])
    eng.close()
    lib.tgis_k_pair_fault(0)
    eng = engine("tiny", weights)
    assert np.array_equal(eng.trace_step(work, end=["a"]), good)
    eng.close()


def test_a_request_ends_with_an_error(lib):
    from vllm_tgis_adapter_b200.engine.core import EngineError, make_sampling_params

    eng = engine("tiny", synthetic_weights(CONFIGS["tiny"], seed=1))
    lib.tgis_k_pair_fault(3)
    with pytest.raises(EngineError, match="wait ran out"):
        eng.generate_sync([[5, 6, 7]], make_sampling_params(greedy=True, max_tokens=4))
    assert eng.status().errored == 1
    eng.close()
