"""Storing rows in the 8-bit cache with the queries rotated where they lie, one row (a single request's step) and two."""
import pytest
import torch

from cache8_checks import D
from vllm_tgis_adapter_b200.engine.cache8 import Cache8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2])
def test_rotation_in_place_of_few_rows(T):
    g = torch.Generator(device="cuda").manual_seed(48)
    qkv = torch.randn(T, 8 * D, device="cuda", generator=g).to(torch.bfloat16)
    cs = torch.randn(100, D, device="cuda", generator=g).to(torch.bfloat16)
    at = torch.arange(5, 5 + T, device="cuda", dtype=torch.int32)
    one, two = Cache8.empty(1, 2), Cache8.empty(1, 2)
    want = one.write(qkv, at, at, cs)
    same = qkv.clone()
    got = two.write(same, at, at, cs, q_out=same[:, :4 * D])
    assert got.data_ptr() == same.data_ptr() and torch.equal(got, want) and torch.equal(same[:, 4 * D:], qkv[:, 4 * D:]) and torch.equal(one.pages, two.pages)
