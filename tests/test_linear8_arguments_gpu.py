"""Arguments of the binding of 8-bit weights that are not what they have to be: a ValueError, as for every other one."""
import pytest
import torch

import linear8_checks as checks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from vllm_tgis_adapter_b200.engine import linear8

    return linear8


def layers(lib):
    one, other = (lib.Linear8.from_weight(checks.case(1, 128, 128, seed)[1]) for seed in (1, 2))
    return one, other, lib.FeedForward8(one, other, one)


def test_what_is_not_rows_in_8_bits_is_refused(lib):
    one, _, block = layers(lib)
    for x in (torch.zeros(2, 128, device="cuda"), torch.zeros(2, 128, device="cuda", dtype=torch.bfloat16), None):
        with pytest.raises(ValueError, match="x:"):
            one(x)
        with pytest.raises(ValueError, match="x:"):
            block(x)
        with pytest.raises(ValueError, match="x:"):
            block.hidden(x)


def test_what_is_not_a_place_for_rows_or_a_matrix_is_refused(lib):
    one, other, block = layers(lib)
    x = torch.zeros(2, 128, device="cuda")
    rows = lib.quantise(x)
    for out in (torch.empty(2, 128, device="cuda"), torch.empty(2, 128, device="cuda").to(torch.float8_e4m3fn)):
        with pytest.raises(ValueError, match="out:"):
            lib.quantise(x, out=out)
        with pytest.raises(ValueError, match="out:"):
            block.hidden(rows, out=out)
    for some in ((x, other, one), (one, x, one), (one, other, x)):
        with pytest.raises(ValueError, match="gate, up, down"):
            lib.FeedForward8(*some)
