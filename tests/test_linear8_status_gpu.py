"""What a layer's check() says where a wait has run out: the word is raised by the host in the kernels' place."""
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


def raised(layer) -> bool:
    try:
        layer.check()
    except RuntimeError as e:
        assert "ran out" in str(e)
        return True
    return False


def test_every_layer_is_told_once(lib):
    some = layers(lib)
    assert not any(map(raised, some))
    for order in ((0, 1, 2), (2, 0, 1), (1, 0, 2)):
        some[0]._on.status.fill_(1)
        assert [raised(some[i]) for i in order] == [True, True, True]
        assert not any(map(raised, some))


def test_a_layer_is_not_told_of_what_was_before_it(lib):
    some = layers(lib)
    some[0]._on.status.fill_(1)
    assert raised(some[0])
    later = layers(lib)
    assert not any(map(raised, later)) and raised(some[1]) and raised(some[2])


def test_a_stall_between_two_checks_is_another(lib):
    some = layers(lib)
    some[1]._on.status.fill_(1)
    assert raised(some[0]) and not raised(some[0])
    some[1]._on.status.fill_(1)
    assert raised(some[0]) and raised(some[1]) and not raised(some[1])
