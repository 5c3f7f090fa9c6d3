"""Bounded waits of the 8-bit cache's attention: what a warp does next is one thing for all its lanes."""
import ctypes as C
import re
from pathlib import Path

import pytest

from vllm_tgis_adapter_b200.engine import _lib

CSRC = Path(_lib.__file__).resolve().parent.parent / "csrc"


@pytest.mark.parametrize("source", ["attention8.cu", "attention8_prompt.cu"])
def test_every_wait_is_the_whole_warps(source):
    """Lanes time out one by one; what goes on by a wait's result uses instructions of the whole warp."""
    text = re.sub(r"//.*", "", (CSRC / source).read_text())
    waits = [s for s in re.split(r"[;{}]", text) if re.search(r"\bbounded_wait\(", s)]
    assert all(re.search(r"__all_sync\(0xffffffffu, (bounded_wait\([^;]*)+\)", s) for s in waits)
    assert waits or "warp_wait(" in text


def test_hook_refuses():
    lib, told = _lib.load_library(), C.c_uint32()
    assert lib.tgis_k_warp_wait(0, 1, None) == -1 and lib.tgis_k_warp_wait(0, -1, C.byref(told)) == -1 and lib.tgis_k_warp_wait(0, 1 << 40, C.byref(told)) == -1
