"""How products with 8-bit weights are cut, by how many clusters run at once: sizes that do not fit at all are passed over."""
import ctypes as C

import pytest

from vllm_tgis_adapter_b200.engine import _lib

B200 = (148, 74, 33, 15)   # clusters of 1, 2, 4 and 8 CTAs, one to an SM


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def pieces(lib, tiles, groups, ctas, at_once):
    return lib.tgis_k_w8_pieces(tiles, groups, ctas, (C.c_int32 * 4)(*at_once))


def pair_plan(lib, n, x_tiles, groups, gated, at_once):
    got = lib.tgis_k_w8_pair_plan(n, x_tiles, groups, gated, (C.c_int32 * 4)(*at_once))
    return divmod(got, 16) if got > 0 else got


def test_few_tokens(lib):
    """32 tokens of 4096 x 14336: by eight on a whole device, by what is left where GPCs are smaller."""
    assert pieces(lib, 32, 112, 2, B200) == 8
    assert pieces(lib, 32, 112, 2, (148, 74, 33, 0)) == 4
    assert pieces(lib, 32, 112, 2, (148, 74, 0, 0)) == 2
    assert pieces(lib, 32, 112, 2, (148, 0, 0, 0)) == 1
    assert pieces(lib, 32, 112, 2, (148, 0, 33, 0)) == 4
    assert pieces(lib, 32, 112, 2, (0, 0, 0, 0)) == -1 and "fits" in lib.tgis_k_last_error().decode()


def test_few_numbers_a_row_are_not_cut(lib):
    assert [pieces(lib, 1, g, 2, B200) for g in (1, 2, 3, 4, 8, 16)] == [1, 1, 1, 2, 4, 8]
    assert pieces(lib, 1, 1, 1, (0, 74, 33, 15)) == -1


@pytest.mark.parametrize("n,x_tiles,groups,gated,want", [(4096, 1, 32, 0, (2, 2)), (6144, 2, 32, 0, (3, 1)), (2128, 2, 88, 0, (4, 2)), (512, 4, 64, 0, (4, 4)), (8192, 8, 64, 0, (4, 1)),
                                                         (512, 1, 12, 0, (2, 1)), (1536, 1, 4, 1, (4, 1)), (14336, 8, 32, 1, (4, 1)), (512, 1, 1, 0, (2, 1))])
def test_pairs(lib, n, x_tiles, groups, gated, want):
    assert pair_plan(lib, n, x_tiles, groups, gated, B200) == want
    for fit in ((148, 74, 33, 0), (148, 74, 0, 0), (0, 10, 0, 0)):
        chunks, s = pair_plan(lib, n, x_tiles, groups, gated, fit)
        assert fit[s.bit_length()] > 0 and (chunks, s) in [(4, 4), (4, 2), (2, 2), (4, 1), (3, 1), (2, 1)] and (not gated or chunks == 4)
    assert pair_plan(lib, n, x_tiles, groups, gated, (0, 0, 0, 0)) == -1



def test_hooks_refuse(lib):
    fit = (C.c_int32 * 4)(*B200)
    assert lib.tgis_k_w8_pieces(1, 1, 1, None) == -1 and lib.tgis_k_w8_pair_plan(1, 1, 1, 0, None) == -1
    assert [lib.tgis_k_w8_pieces(*a, fit) for a in ((0, 1, 1), (1, 0, 1), (1, 1, 0))] == [-1] * 3
    assert [lib.tgis_k_w8_pair_plan(*a, 0, fit) for a in ((0, 1, 1), (1, 0, 1), (1, 1, 0))] == [-1] * 3
