"""What the 8-bit cache's C ABI takes and asks for at its bounds, without a GPU (every call here is refused before a launch)."""
import pytest
from test_cache8_cpu import AT, WRITE

from vllm_tgis_adapter_b200.engine import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


@pytest.mark.parametrize("T,says", [(1, "positions"), (2, "in place")])
def test_one_row_in_place_has_no_pitch(lib, T, says):
    """A tensor of one row has any pitch: its queries rotated in place keep their row whatever ldq is.  (Refused for the next argument.)"""
    args = {**WRITE, "qkv": AT, "q_out": AT, "ld": 1024, "ldq": 512, "T": T, "positions": None}
    assert lib.tgis_kv8_write(*args.values()) == -1
    assert says in lib.tgis_kv8_last_error().decode()
