"""The products' wait where it runs out (the barrier in question is one that nothing arrives at): the warp stays together, and the report gets to where it is read."""
import ctypes as C

import pytest

from vllm_tgis_adapter_b200.engine import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("words", [0, 1, 2, 3])
@pytest.mark.parametrize("arrived", [0xffffffff, 0, 1, 0x80000000, 0xfffffffe, 0x7fffffff, 0x0000ffff, 0x55555555])
def test_a_wait_that_runs_out_is_reported(arrived, words):
    lib, told, status, stalled = _lib.load_library(), C.c_uint32(0x12345678), C.c_int32(-7), C.c_int32(-7)
    assert lib.tgis_k_await8(arrived, 200_000, words, C.byref(told), C.byref(status), C.byref(stalled)) == 0
    out = arrived != 0xffffffff
    assert told.value == arrived
    assert status.value == (1 if out and words & 1 else 0)   # TGIS_W8_STALLED
    assert stalled.value == (1 if out and words & 2 else 0)


def test_hook_refuses():
    lib, told, word = _lib.load_library(), C.c_uint32(), C.c_int32()
    assert lib.tgis_k_await8(0, 200_000, 3, None, C.byref(word), C.byref(word)) == -1
    assert lib.tgis_k_await8(0, 0, 3, C.byref(told), C.byref(word), C.byref(word)) == -1
    assert lib.tgis_k_await8(0, 1 << 40, 3, C.byref(told), C.byref(word), C.byref(word)) == -1
    assert lib.tgis_k_await8(0, 200_000, 4, C.byref(told), C.byref(word), C.byref(word)) == -1
