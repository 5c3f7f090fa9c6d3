"""What the 8-bit cache's C ABI takes and asks for at its bounds, without a GPU (every call here is refused before a launch)."""
import pytest
from test_cache8_cpu import AT, WRITE

from vllm_tgis_adapter_b200.engine import _lib, cache8


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


@pytest.mark.parametrize("T,says", [(1, "positions"), (2, "in place")])
def test_one_row_in_place_has_no_pitch(lib, T, says):
    """A tensor of one row has any pitch: its queries rotated in place keep their row whatever ldq is.  (Refused for the next argument.)"""
    args = {**WRITE, "qkv": AT, "q_out": AT, "ld": 1024, "ldq": 512, "T": T, "positions": None}
    assert lib.tgis_kv8_write(*args.values()) == -1
    assert says in lib.tgis_kv8_last_error().decode()


@pytest.mark.parametrize("n_q,n_kv", [(32, 8), (64, 8), (6, 2), (4, 1), (12, 12), (150, 1)])
def test_workspace_of_the_largest_call_serves_every_smaller_one(lib, n_q, n_kv):
    """Fewer sequences, fewer queries of each or shorter ones ask for no more, whichever kernel takes them; and nothing asks for more than a
    unit of sums twice for each of 160 CTAs."""
    ask = lambda n, q, kv: lib.tgis_kv8_attention_workspace(n * q, n, n_q, n_kv, q, kv)  # noqa: E731
    counts, queries, lengths = (1, 2, 7, 40, 256, 1024, 4096), (1, 2, 3, 4, 6, 8, 11, 12, 13, 16, 24, 48, 49, 64), (1, 500, 768, 769, 1024, 1025, 2048, 5000, 8192, 60000)
    size = {(n, q, kv): ask(n, q, kv) for n in counts for q in queries for kv in lengths}
    for (n, q, kv), here in size.items():
        assert 0 <= here <= 160 * (2 * 256 * 130 * 4 + 32)
        for smaller in ((counts[max(counts.index(n) - 1, 0)], q, kv), (n, queries[max(queries.index(q) - 1, 0)], kv), (n, q, lengths[max(lengths.index(kv) - 1, 0)])):
            assert size[smaller] <= here, (smaller, (n, q, kv))


@pytest.mark.parametrize("max_q,max_kv,says", [(1 << 32 | 5, 100, "31 bits"), (5, 1 << 32 | 100, "31 bits"), (5, 1 << 31, "31 bits"), (-1, 100, "31 bits"), (5, (1 << 31) - 1, "max_kv")])
def test_bounds_are_not_cut_to_32_bits(lib, max_q, max_kv, says):
    cache = object.__new__(cache8.Cache8)   # (as far as sizes go: one with pages needs a device)
    cache._lib, cache._workspace, cache.n_kv = lib, lib.tgis_kv8_attention_workspace, 2
    with pytest.raises(ValueError, match=says):
        cache.workspace_bytes(5, 1, 4, max_q, max_kv)
