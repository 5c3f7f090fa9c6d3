"""A bounded wait that runs out in some lanes of a warp has run out for all of them (the barrier in question is one that nothing arrives at)."""
import ctypes as C

import pytest

from vllm_tgis_adapter_b200.engine import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("arrived", [0xffffffff, 0, 1, 0x80000000, 0xfffffffe, 0x7fffffff, 0x0000ffff, 0x55555555])
def test_all_lanes_or_none(arrived):
    lib, told = _lib.load_library(), C.c_uint32(0x12345678)
    assert lib.tgis_k_warp_wait(arrived, 200_000, C.byref(told)) == 0
    assert told.value == (0xffffffff if arrived == 0xffffffff else 0)
